"""Operators of a serving step that drafts over caches held in 8 bits and in pages, and what each costs:

* store: rows of K and V become codes of 8 bits with a scale for each block of sixteen tokens and head; load: what they stand for comes back;
* attn: attention of a step's tokens - one per conversation, or a tree of drafted ones - over such caches;
* pages: sequences take pages, share them, copy a shared one before it is written and give them back; kept slots move together;
* verify: drafted tokens are accepted or rejected by the target's and the draft's distributions and given random numbers, and the next token is drawn.

`run` computes the plain form, or where `own` is true makes the calls of this framework.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16                  # tokens that share a scale
IO = {"float32": torch.float32, "bfloat16": torch.bfloat16}
# heads, kv heads, head size, layers that the framework's models bring
SHAPES = {"qwen2-0.5b": (14, 2, 64, 24), "llama-3.2-1b": (32, 8, 64, 16), "llama-3.1-8b": (32, 8, 128, 32)}
# the records of the framework's calls
SEQ = np.dtype([("table", "u8"), ("hidden", "u8"), ("n_kv", "i4"), ("n_tok", "i4"), ("n_table", "i4"), ("reserved", "i4")])
EDIT = np.dtype([("table", "u8"), ("from", "u8"), ("n_old", "i4"), ("n_new", "i4"), ("n_table", "i4"), ("reserved", "i4")])
MOVE = np.dtype([("table", "u8"), ("keep", "u8"), ("n_keep_dev", "u8"), ("first", "i4"), ("n_kv", "i4"), ("n_keep", "i4"), ("n_table", "i4")])


def listed():
    return [
        # the smallest step: four short chats of a small model, one token each
        {"name": "attn_chats_4", "op": "attn", "shape": "qwen2-0.5b", "io": "float32", "page": 16, "seqs": 4, "tok": 1, "past": 290, "ragged": True, "tree": False, "hidden": False},
        # a server's step: 64 conversations of all lengths
        {"name": "attn_sessions_64", "op": "attn", "shape": "llama-3.1-8b", "io": "float32", "page": 64, "seqs": 64, "tok": 1, "past": 2040, "ragged": True, "tree": False, "hidden": False},
        # trees of different depths over caches with hidden slots
        {"name": "attn_trees_bf16", "op": "attn", "shape": "llama-3.2-1b", "io": "bfloat16", "page": 32, "seqs": 8, "tok": 20, "past": 8100, "ragged": True, "tree": True, "hidden": True},
        # the widest tree of the speculative decoder over two long documents
        {"name": "attn_tree_32_long", "op": "attn", "shape": "llama-3.1-8b", "io": "float32", "page": 128, "seqs": 2, "tok": 32, "past": 32700, "ragged": False, "tree": True, "hidden": False},
        # one layer of a server's step: a token of each conversation
        {"name": "store_step", "op": "store", "shape": "llama-3.1-8b", "io": "float32", "page": 64, "seqs": 64, "tok": 1, "past": 2040, "ragged": True},
        # portions of prompts, of different lengths and beginnings
        {"name": "store_prompts", "op": "store", "shape": "llama-3.1-8b", "io": "bfloat16", "page": 128, "seqs": 5, "tok": 2041, "past": 6000, "ragged": True},
        # room for a drafted tree is taken and given back
        {"name": "pages_room", "op": "room", "shape": "llama-3.2-1b", "page": 16, "seqs": 64, "tok": 12, "past": 500, "spare": 900},
        # eight answers to each of eight prompts: the last step's are dropped, new ones begin with the prompt's pages, whose last one is copied
        {"name": "pages_fork", "op": "fork", "shape": "llama-3.1-8b", "page": 64, "seqs": 8, "answers": 8, "past": 489, "spare": 8},
        # the accepted tokens of drafted trees move together, in all layers
        {"name": "compact_step", "op": "compact", "shape": "llama-3.2-1b", "page": 16, "layers": 16, "seqs": 64, "past": 250, "behind": 12, "keep": 5},
        # caches that were longer than their budget, in four layers
        {"name": "compact_prompt", "op": "compact", "shape": "llama-3.1-8b", "page": 64, "layers": 4, "seqs": 4, "past": 4, "behind": 8186, "keep": 2043},
        # a drafted tree of the speculative decoder's default size, tokens of its own choice
        {"name": "verify_tree_12", "op": "verify", "seqs": 1, "nodes": 12, "fan": 3, "vocab": 151936, "kind": "chat", "draft": False},
        # a server's step: four drafted tokens of each conversation, drawn from the draft's rows, every request with its own settings
        {"name": "verify_sessions_64", "op": "verify", "seqs": 64, "nodes": 5, "fan": 1, "vocab": 128256, "kind": "mixed", "draft": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "store", "room", "fork", "compact", "verify"])
    if op == "verify":
        seqs = _log(rng, 1, 40)
        nodes = _log(rng, 1, max(2, min(24, 240 // seqs)))
        return {"op": op, "seqs": seqs, "nodes": nodes, "fan": rng.choice([1, 1, 2, 3]), "vocab": _log(rng, 2000, 128256), "kind": rng.choice(["chat", "nucleus", "plain", "mixed"]), "draft": rng.random() < 0.6}
    shape, page = rng.choice(sorted(SHAPES)), rng.choice([16, 32, 64, 128])
    if op == "store":
        seqs = _log(rng, 1, 64)
        return {"op": op, "shape": shape, "io": rng.choice(["float32", "bfloat16"]), "page": page, "seqs": seqs, "tok": _log(rng, 1, max(1, 8000 // seqs)), "past": _log(rng, 1, 16000 // seqs + 50), "ragged": rng.random() < 0.6}
    if op == "room":
        return {"op": op, "shape": shape, "page": page, "seqs": _log(rng, 1, 64), "tok": _log(rng, 1, 300), "past": _log(rng, 1, 500), "spare": rng.choice([5, 60, 1500])}
    if op == "fork":
        return {"op": op, "shape": shape, "page": page, "seqs": _log(rng, 1, 8), "answers": _log(rng, 1, 8), "past": _log(rng, 1, 500), "spare": rng.choice([0, 3, 40])}
    if op == "compact":
        behind = _log(rng, 1, 4000)
        return {"op": op, "shape": shape, "page": page, "layers": rng.choice([1, 4, 8]), "seqs": _log(rng, 1, max(1, min(40, 12000 // (behind + 100)))), "past": _log(rng, 1, 300), "behind": behind, "keep": max(1, int(behind * rng.uniform(0.1, 1.0)))}
    seqs = _log(rng, 1, 64)
    tree = rng.random() < 0.5
    tok = _log(rng, 2, 32) if tree else rng.choice([1, 1, 1, _log(rng, 2, 32)])
    past = _log(rng, 1, max(32, min(32700, 65400 // seqs)))
    tok = max(1, min(tok, 2097152 // (seqs * (past + 32))))     # no dearer than the largest listed one
    return {"op": op, "shape": shape, "io": rng.choice(["float32", "float32", "bfloat16"]), "page": page, "seqs": seqs, "tok": tok, "past": past, "ragged": rng.random() < 0.6, "tree": tree, "hidden": rng.random() < 0.4}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(most, count, ragged, least):
    if not ragged:
        return np.full(count, most, np.int64)
    r = np.random.Generator(np.random.SFC64([most, count]))     # a case's sizes are its own, whatever the seed
    n = np.exp(r.uniform(math.log(max(least, most // 8, 1)), math.log(most + 0.5), count)).astype(np.int64).clip(least, most)
    n[0] = most
    return n


def _tokens(case):
    return _lengths(case["tok"], case["seqs"], case["ragged"] and case["tok"] > 1, 1)


def _tree(n, r):
    """mask [n][n] of a drafted tree: a node sees its ancestors and itself"""
    m = np.zeros((n, n), np.uint8)
    for i in range(n):
        if i:
            m[i] = m[int(r.integers(max(0, i - 4), i))]
        m[i, i] = 1
    return m


def _up(n, page):
    return -(-n // page)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _cache(case, layers, counts, spare, g):
    """codes and scales of `layers` layers, and a table of pages, in no order, for every sequence: counts[s] pages of them are its own"""
    _, G, D, _ = SHAPES[case["shape"]]
    P, most, n_pages = case["page"], int(max(counts)), int(sum(counts)) + spare
    codes = torch.randint(-127, 128, (layers, n_pages, G, 2, P * D), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(layers, n_pages, G, 2, P // BLOCK, generator=g, device="cuda") * 0.02 + 0.005
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.as_tensor(counts, device="cuda")
    at = (torch.cumsum(counts, 0) - counts)[:, None] + torch.arange(most, device="cuda")
    table = torch.where(torch.arange(most, device="cuda") < counts[:, None], order[at.clamp(max=n_pages - 1)], -1)
    return {"case": case, "codes": codes, "scales": scales, "table": table.contiguous()}


def _records(kind, count, fields):
    t = np.zeros(count, kind)
    for name, v in fields.items():
        t[name] = [x.data_ptr() for x in v] if isinstance(v, torch.Tensor) else v
    return t


def _prepare_attn(case, seed):
    H, G, D, _ = SHAPES[case["shape"]]
    S, g, r = case["seqs"], _gen(seed), np.random.Generator(np.random.SFC64([int(seed) & 0x7FFFFFFF, 11]))
    past, tok = _lengths(case["past"], S, case["ragged"], 0), _tokens(case)
    n_kv = past + tok
    st = _cache(case, 1, _up(n_kv, case["page"]), 3, g)
    q = (torch.randn(int(tok.sum()), H * D, generator=g, device="cuda") * 1.5).to(IO[case["io"]])
    most = st["table"].shape[1] * case["page"]
    hidden = None
    if case["hidden"]:
        hidden = torch.rand(S, most, generator=g, device="cuda") < 0.03
        hidden &= torch.arange(most, device="cuda")[None] < torch.as_tensor(past, device="cuda")[:, None]
        hidden = hidden.to(torch.uint8)
    mask = torch.from_numpy(np.concatenate([_tree(int(t), r).reshape(-1) for t in tok])).cuda() if case["tree"] else None
    fields = {"table": st["table"], "n_kv": n_kv, "n_tok": tok, "n_table": st["table"].shape[1]} | ({"hidden": hidden} if hidden is not None else {})
    return st | {"q": q, "out": torch.zeros_like(q), "hidden": hidden, "mask": mask, "seqs": _records(SEQ, S, fields), "n_kv": torch.as_tensor(n_kv, device="cuda"),
                 "n_tok": torch.as_tensor(tok, device="cuda"), "scale": 1.0 / math.sqrt(D)}


def _prepare_store(case, seed):
    _, G, D, _ = SHAPES[case["shape"]]
    S, g = case["seqs"], _gen(seed)
    past, tok = _lengths(case["past"], S, case["ragged"], 0), _tokens(case)
    n_kv = past + tok
    st = _cache(case, 1, _up(n_kv, case["page"]), 1, g)
    k = torch.randn(int(tok.sum()), G * D, generator=g, device="cuda")
    k[:, 0::D] += 3.0               # keys share a direction, as cached ones do
    v = torch.randn(int(tok.sum()), G * D, generator=g, device="cuda")
    k, v = k.to(IO[case["io"]]), v.to(IO[case["io"]])
    return st | {"k": k, "v": v, "k_held": torch.zeros_like(k), "v_held": torch.zeros_like(v), "n_kv": torch.as_tensor(n_kv, device="cuda"), "n_tok": torch.as_tensor(tok, device="cuda"),
                 "seqs": _records(SEQ, S, {"table": st["table"], "n_kv": n_kv, "n_tok": tok, "n_table": st["table"].shape[1]})}


def _refs(st, tables, counts):
    """holders of every page"""
    held = torch.arange(tables.shape[1], device="cuda") < counts[:, None]
    st["refs"] = torch.zeros(st["codes"].shape[1], dtype=torch.int32, device="cuda").index_add_(0, tables[held].long(), torch.ones(int(held.sum()), dtype=torch.int32, device="cuda"))


def _prepare_room(case, seed):
    S, P, g = case["seqs"], case["page"], _gen(seed)
    n = _lengths(case["past"], S, True, 0)
    st = _cache(case, SHAPES[case["shape"]][3], np.maximum(_up(n, P), 1), S * (_up(case["tok"], P) + 1) + case["spare"], g)
    room = torch.full((S, _up(case["past"] + case["tok"], P) + 1), -1, dtype=torch.int32, device="cuda")
    room[:, :st["table"].shape[1]] = st["table"]
    n_dev, m_dev = torch.as_tensor(n, device="cuda"), torch.as_tensor(n + case["tok"], device="cuda")
    _refs(st, room, _up(n_dev, P))
    edit = {"table": room, "n_table": room.shape[1]}
    return st | {"table": room, "held": torch.zeros(2, S, dtype=torch.int32, device="cuda"),
                 "edits": [(_records(EDIT, S, edit | {"n_old": a, "n_new": b}), room, None, c, d) for a, b, c, d in ((n, n + case["tok"], n_dev, m_dev), (n + case["tok"], n, m_dev, n_dev))]}


def _prepare_fork(case, seed):
    S, P, A, g = case["seqs"], case["page"], case["answers"], _gen(seed)
    n = _lengths(case["past"], S, True, 1)
    st = _cache(case, SHAPES[case["shape"]][3], _up(n, P), 2 * S * A + case["spare"], g)
    wide = st["table"].shape[1] + 1
    prompts = torch.full((S, wide), -1, dtype=torch.int32, device="cuda")
    prompts[:, :wide - 1] = st["table"]
    two = torch.full((2, S * A, wide), -1, dtype=torch.int32, device="cuda")
    start = np.repeat(n, A)
    old, new = torch.as_tensor(start, device="cuda"), torch.as_tensor(start + 1, device="cuda")
    none = torch.zeros_like(old)
    _refs(st, prompts, _up(torch.as_tensor(n, device="cuda"), P))
    begun = prompts.repeat_interleave(A, 0)
    turns = []
    for a, b in ((0, 1), (1, 0)):       # one set of answers is dropped, another one begins
        gone = _records(EDIT, S * A, {"table": two[a], "n_table": wide, "n_old": start + 1, "n_new": 0})
        come = _records(EDIT, S * A, {"table": two[b], "from": [x.data_ptr() for x in prompts for _ in range(A)], "n_table": wide, "n_old": start, "n_new": start + 1})
        every = torch.cat([two[a], two[b]])
        turns.append((np.concatenate([gone, come]), (two[a], two[b]), begun, torch.cat([new, old]), torch.cat([none, new]), every.shape[0]))
    st |= {"prompts": prompts, "two": two, "turns": turns, "turn": 0, "held": torch.zeros(2 * S * A, dtype=torch.int32, device="cuda")}
    # the answers of the step before: pages as the plain form gives them
    _share(st["refs"], two[0], begun, old, P)
    copies = _grow(st["refs"], two[0], old, new, torch.ones_like(old).bool(), P)[1]
    _copy(st, *copies)
    return st


def _prepare_compact(case, seed):
    S, P, g = case["seqs"], case["page"], _gen(seed)
    past = _lengths(case["past"], S, True, 0)
    behind, keep = case["behind"], case["keep"]
    st = _cache(case, case["layers"], _up(past + behind, P), 1, g)
    order = torch.rand(S, behind, generator=g, device="cuda").argsort(1)[:, :keep].sort(1).values.to(torch.int32)
    order[:, 0] = 0                     # (the first of a drafted tree's tokens is always kept)
    order = order.contiguous()
    n_keep = torch.randint(max(1, keep // 2), keep + 1, (S,), generator=g, device="cuda", dtype=torch.int32)
    moves = _records(MOVE, S, {"table": st["table"], "keep": order, "n_keep_dev": n_keep, "first": past, "n_kv": past + behind, "n_keep": keep, "n_table": st["table"].shape[1]})
    return st | {"keep": order, "n_keep": n_keep, "first": torch.as_tensor(past, device="cuda"), "moves": moves}


def _settings(kind, n, r):
    """rows of [temperature, top-k, top-p, min-p]"""
    p = np.zeros((n, 4))
    p[:, 0], p[:, 2] = 1.0, 1.0
    if kind == "chat":
        p[:] = [0.8, 40, 0.95, 0.0]
    elif kind == "nucleus":
        p[:] = [1.0, 0, 0.9, 0.02]
    elif kind == "mixed":
        every = np.array([[0.8, 40, 0.95, 0.0], [1.0, 0, 0.9, 0.0], [1.3, 0, 1.0, 0.05], [0.0, 0, 1.0, 0.0], [1.0, 0, 1.0, 0.0], [0.6, 500, 0.8, 0.1], [1.5, 2000, 0.99, 0.001]])
        p[:] = every[r.integers(0, len(every), n)]
    return p


def _prepare_verify(case, seed):
    S, N, V = case["seqs"], case["nodes"], case["vocab"]
    g, r = _gen(seed), np.random.Generator(np.random.SFC64([int(seed) & 0x7FFFFFFF, 13]))
    logits = torch.randn(S * N, V, generator=g, device="cuda") * 2.5
    at = torch.randint(0, V, (S * N, 24), generator=g, device="cuda")      # a few tokens that the model holds for likely
    logits.scatter_add_(1, at, torch.rand(S * N, 24, generator=g, device="cuda") * 12.0)
    guess = logits + torch.randn(S * N, V, generator=g, device="cuda") * 0.6      # the draft model is nearly of the same mind
    # a node's parent lies before it; its token is one of its parent's row that the draft holds for likely
    parent = np.arange(-1, N - 1)[None].repeat(S, 0)
    if case["fan"] > 1:
        parent = np.concatenate([np.full((S, 1), -1), *(r.integers(max(0, i - case["fan"]), i, (S, 1)) for i in range(1, N))], 1)
    row = (np.arange(S)[:, None] * N + parent.clip(0)).reshape(-1)
    likely = torch.topk(guess, 12, dim=1)
    pick = (likely.values - torch.empty_like(likely.values).exponential_(generator=g).log())[torch.from_numpy(row).cuda()].argmax(1)
    tokens = likely.indices[torch.from_numpy(row).cuda(), pick].to(torch.int32)
    par = _settings(case["kind"], S, r).repeat(N, 0)
    table = np.zeros(S * N, np.dtype([("temperature", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")]))
    table["temperature"], table["top_k"], table["top_p"], table["min_p"] = par[:, 0], par[:, 1].astype(np.int32), par[:, 2], par[:, 3]
    return {"case": case, "logits": logits, "guess": guess if case["draft"] else None, "parents": torch.from_numpy(parent.reshape(-1).astype(np.int32)).cuda(), "tokens": tokens.contiguous(),
            "params": torch.from_numpy(table.view(np.int32).reshape(S * N, 4).copy()).cuda(), "u": torch.rand(S * N, generator=g, device="cuda"), "nodes": np.full(S, N, np.int32),
            "ids": torch.zeros(S, dtype=torch.int32, device="cuda"), "path": torch.zeros(S * N, dtype=torch.int32, device="cuda"), "n_path": torch.zeros(S, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    return {"attn": _prepare_attn, "store": _prepare_store, "room": _prepare_room, "fork": _prepare_fork, "compact": _prepare_compact, "verify": _prepare_verify}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _views(st):
    """codes as [layer][page][token / 8][token % 8][head][channel / 16][channel % 16] and [layer][page][token / 16][token % 16][head][channel], scales as [layer][page][block][head][K, V]"""
    _, G, D, _ = SHAPES[st["case"]["shape"]]
    P = st["case"]["page"]
    L, N = st["codes"].shape[:2]
    k = st["codes"][:, :, :, 0].view(L, N, G, P // 8, D // 16, 8, 16).permute(0, 1, 3, 5, 2, 4, 6)
    v = st["codes"][:, :, :, 1].view(L, N, G, P // 16, D, 16).permute(0, 1, 3, 5, 2, 4)
    return k, v, st["scales"].permute(0, 1, 4, 2, 3)


def _attn_plain(st):
    """out[t] = sum_j p_tj v_j, p = softmax over the slots that token t sees of scale q_t.k_j"""
    case = st["case"]
    H, G, D, _ = SHAPES[case["shape"]]
    S, R, T, P = case["seqs"], H // G, case["tok"], case["page"]
    dev, n_kv, n_tok = st["q"].device, st["n_kv"], st["n_tok"]
    pages = st["table"].clamp(min=0).long()
    n = pages.shape[1] * P
    kc, vc, sc = _views(st)
    k = kc[0][pages].float().reshape(S, n // BLOCK, BLOCK, G, D) * sc[0][pages].reshape(S, n // BLOCK, 1, G, 1, 2)[..., 0]
    v = vc[0][pages].float().reshape(S, n // BLOCK, BLOCK, G, D) * sc[0][pages].reshape(S, n // BLOCK, 1, G, 1, 2)[..., 1]
    t = torch.arange(T, device=dev)
    start = torch.cumsum(n_tok, 0) - n_tok
    row = (start[:, None] + t).clamp(max=st["q"].shape[0] - 1)
    there = t[None] < n_tok[:, None]                                    # [S][T]
    slot = torch.arange(n, device=dev)
    back = slot[None] - (n_kv - n_tok)[:, None]                         # the slot's number among the step's tokens
    inside = (back >= 0) & (back < n_tok[:, None])
    if st["mask"] is not None:
        first = torch.cumsum(n_tok * n_tok, 0) - n_tok * n_tok
        at = first[:, None, None] + t[None, :, None] * n_tok[:, None, None] + back[:, None, :]
        sees = st["mask"][at.clamp(0, st["mask"].numel() - 1)] != 0
    else:
        sees = back[:, None, :] <= t[None, :, None]
    sees = torch.where(inside[:, None, :], sees, (back < 0)[:, None, :]) & there[:, :, None]
    if st["hidden"] is not None:
        sees &= (st["hidden"][:, None, :n] == 0)
    k, v = k.reshape(S, n, G, D).permute(0, 2, 3, 1), v.reshape(S, n, G, D).permute(0, 2, 1, 3)
    q = st["q"].float()[row].view(S, T, G, R, D).permute(0, 2, 1, 3, 4).reshape(S, G, T * R, D) * st["scale"]
    s = torch.matmul(q, k).view(S, G, T, R, n)
    s = torch.where(sees[:, None, :, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(sees[:, None, :, None, :], torch.exp(s - torch.where(m > -math.inf, m, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(S, G, T * R, n), v).view(S, G, T, R, D).permute(0, 2, 1, 3, 4).reshape(S, T, H * D)
    st["out"][row[there]] = o[there].to(st["out"].dtype)
    return {"out": st["out"]}


def _slots(st):
    """(page, slot in it, whether it is the step's first token) of the step's tokens, sequence after sequence"""
    P, n_tok = st["case"]["page"], st["n_tok"]
    seq = torch.repeat_interleave(torch.arange(n_tok.numel(), device=n_tok.device), n_tok)
    t = torch.arange(seq.numel(), device=seq.device) - (torch.cumsum(n_tok, 0) - n_tok)[seq]
    slot = (st["n_kv"] - n_tok)[seq] + t
    return st["table"][seq, slot // P].long(), slot % P, t == 0


def _store_plain(st):
    """a block's scale is the largest of its old one, where slots were in it before, and its new numbers' largest / 127; codes are numbers / scale, rounded; older codes follow the scale"""
    case = st["case"]
    _, G, D, _ = SHAPES[case["shape"]]
    P, (kc, vc, sc) = case["page"], _views(st)
    page, slot, begins = _slots(st)
    N, B = st["codes"].shape[1], P // BLOCK
    x = torch.stack([st["k"].float(), st["v"].float()], 1).view(-1, 2, G, D)
    block = page * B + slot // BLOCK
    most = torch.zeros(N * B, 2, G, device=x.device).index_reduce_(0, block, x.abs().amax(-1), "amax")
    touched = torch.zeros(N * B, dtype=torch.bool, device=x.device).index_fill_(0, block, True)
    cont = begins & (slot % BLOCK > 0)                                  # blocks with older slots
    older = torch.zeros(N * B, dtype=torch.bool, device=x.device).index_fill_(0, block[cont], True)
    old = sc[0].reshape(N * B, G, 2).transpose(1, 2)
    new = torch.maximum(most / torch.full_like(most, 127.0), torch.where(older[:, None, None], old, 0.0))
    new = torch.where(touched[:, None, None], new, old)
    # the older slots of such blocks
    pc, oc, bc = page[cont], slot[cont] // BLOCK, block[cont]
    at = torch.arange(BLOCK, device=x.device)
    f = (old[bc] / torch.where(new[bc] > 0, new[bc], 1.0))[:, None]     # [blocks][1][2][G]
    own_slot = (oc * BLOCK)[:, None] + at
    was = at[None] < (slot[cont] % BLOCK)[:, None]
    for c, i in ((kc[0], 0), (vc[0], 1)):
        a, b = (own_slot // 8, own_slot % 8) if i == 0 else (own_slot // 16, own_slot % 16)
        h = c[pc[:, None], a, b]
        n = torch.round(h.float().reshape(*h.shape[:3], D) * f[:, :, i, :, None]).to(torch.int8).reshape(h.shape)
        c[pc[:, None], a, b] = torch.where(was.view(*was.shape, *[1] * (h.dim() - 2)), n, h)
    s = new[block]
    codes = torch.round(x / torch.where(s > 0, s, 1.0)[..., None]).clamp(-127, 127).to(torch.int8)
    kc[0][page, slot // 8, slot % 8] = codes[:, 0].view(-1, G, D // 16, 16)
    vc[0][page, slot // 16, slot % 16] = codes[:, 1]
    sc[0].copy_(new.transpose(1, 2).reshape(N, B, G, 2))
    # what the cache now holds for them
    held = codes.float() * s[..., None]
    st["k_held"].copy_(held[:, 0].reshape(-1, G * D))
    st["v_held"].copy_(held[:, 1].reshape(-1, G * D))
    return {"k": st["k_held"], "v": st["v_held"], "scales": st["scales"]}


def _share(refs, tables, begun, n, page):
    held = torch.arange(tables.shape[1], device=refs.device) < _up(n, page)[:, None]
    tables.copy_(torch.where(held, begun, tables))
    refs.index_add_(0, tables[held].long(), torch.ones(int(held.sum()), dtype=torch.int32, device=refs.device))


def _release(refs, tables, old, new, page):
    at = torch.arange(tables.shape[1], device=refs.device)
    gone = (at >= _up(new, page)[:, None]) & (at < _up(old, page)[:, None])
    refs.index_add_(0, tables[gone].long(), torch.full((int(gone.sum()),), -1, dtype=torch.int32, device=refs.device))


def _grow(refs, tables, old, new, grows, page):
    """pages, lowest free ones first, to the sequences in order; a shared last page gets a copy, but for its last holder's.  (lengths, copies)"""
    had, want, part = _up(old, page), _up(new, page), grows & (old % page > 0)
    last = tables.gather(1, (had - 1).clamp(min=0)[:, None])[:, 0].long().clamp(min=0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    rank = torch.tril(same, -1).sum(1)
    copies = part & (refs[last] - rank > 1)
    need = torch.where(grows, copies.long() + want - had, 0)
    free = (refs == 0).nonzero()[:, 0]
    cum = torch.cumsum(need, 0)
    fits = grows & ((cum <= free.numel()) | ((need == 0) & ~(part & (rank > 0))))
    copies, need, at = copies & fits, torch.where(fits, need, 0), cum - need
    first = torch.where(copies, had - 1, had)
    slot = torch.arange(tables.shape[1], device=refs.device)[None] - first[:, None]
    takes = (slot >= 0) & (slot < need[:, None])
    got = free[(at[:, None] + slot)[takes]]
    src = last[copies]
    tables[takes] = got.to(torch.int32)
    refs[got] = 1
    refs.index_add_(0, src, torch.full((src.numel(),), -1, dtype=torch.int32, device=refs.device))
    return torch.where(grows & ~fits, old, new), (src, tables[copies, had[copies] - 1].long(), _up(old[copies] % page, BLOCK))


def _copy(st, src, dst, blocks):
    """the blocks that are filled, in all layers"""
    B = st["scales"].shape[-1]
    L, N, G = st["codes"].shape[:3]
    inside = torch.arange(B, device=src.device) < blocks[:, None]
    codes = st["codes"].view(L, N, G, 2, B, -1)
    codes[:, dst] = torch.where(inside[None, :, None, None, :, None], codes[:, src], codes[:, dst])
    st["scales"][:, dst] = torch.where(inside[None, :, None, None], st["scales"][:, src], st["scales"][:, dst])


def _room_plain(st):
    for k, (_, tables, _, old, new) in enumerate(st["edits"]):
        _release(st["refs"], tables, old, torch.minimum(new, old), st["case"]["page"])
        held, copies = _grow(st["refs"], tables, old, new, new > old, st["case"]["page"])
        _copy(st, *copies)
        st["held"][k] = held.to(torch.int32)
    return {"table": st["table"], "refs": st["refs"], "held": st["held"]}


def _fork_plain(st):
    _, (gone, come), begun, old, new, n = st["turns"][st["turn"]]
    P, h = st["case"]["page"], n // 2
    _share(st["refs"], come, begun, old[h:], P)
    _release(st["refs"], gone, old[:h], new[:h], P)
    held, copies = _grow(st["refs"], come, old[h:], new[h:], new[h:] > old[h:], P)
    _copy(st, *copies)
    st["held"][:h] = 0
    st["held"][h:] = held.to(torch.int32)
    return _forked(st)


def _forked(st):
    st["turn"] ^= 1
    return {"tables": st["two"], "refs": st["refs"], "held": st["held"], "codes": st["codes"], "scales": st["scales"]}


def _compact_plain(st):
    """slot first + i takes what slot first + keep[i] holds; a block's scale becomes the largest of the scales that its slots come with, and their codes follow it"""
    case = st["case"]
    _, G, D, _ = SHAPES[case["shape"]]
    P, (kc, vc, sc), first = case["page"], _views(st), st["first"]
    S, K = st["keep"].shape
    # slots of the sequences from the beginning of the first block on: those before `first` stay
    lead = first % BLOCK
    i = torch.arange(K + BLOCK, device=first.device)[None] - lead[:, None]
    there = i < st["n_keep"][:, None]
    src = torch.where(i < 0, i, st["keep"].gather(1, i.clamp(0, K - 1)).long()) + first[:, None]
    dst = i + first[:, None]
    src, dst = torch.where(there, src, 0), torch.where(there, dst, 0)
    page = st["table"].long().gather(1, src // P)
    s = sc[:, page, src % P // BLOCK]                                   # [L][S][K + 16][G][2]
    L, B = s.shape[0], (K + 2 * BLOCK - 1) // BLOCK
    s_pad = torch.cat([torch.where(there[None, :, :, None, None], s, 0.0), s.new_zeros(L, S, B * BLOCK - s.shape[2], G, 2)], 2)
    new = s_pad.view(L, S, B, BLOCK, G, 2).amax(3)
    to = new.repeat_interleave(BLOCK, 2)[:, :, :K + BLOCK]
    f = s / torch.where(to > 0, to, 1.0)
    k = torch.round(kc[:, page, src % P // 8, src % P % 8].float() * f[..., 0, None, None]).to(torch.int8)
    v = torch.round(vc[:, page, src % P // 16, src % P % 16].float() * f[..., 1, None]).to(torch.int8)
    page = st["table"].long().gather(1, dst // P)[there]
    at = dst[there] % P
    kc[:, page, at // 8, at % 8] = k[:, there]
    vc[:, page, at // 16, at % 16] = v[:, there]
    sc[:, page, at // BLOCK] = to[:, there]
    return {"codes": st["codes"], "scales": st["scales"]}


def _weights(logits, par):
    """rows of the distributions that the settings leave of the logits, in 64 bits"""
    V = logits.shape[1]
    T, k, top_p, min_p = par[:, 0:1].view(torch.float32).double(), par[:, 1:2], par[:, 2:3].view(torch.float32).double(), par[:, 3:4].view(torch.float32).double()
    xs, order = torch.sort(logits, dim=1, descending=True, stable=True)
    greedy = T <= 0
    rank = torch.arange(V, device=logits.device)
    keep = ((k <= 0) | (rank < k)) & (xs > -math.inf)
    w = torch.where(keep, torch.exp((xs.double() - xs[:, :1].double()) / torch.where(greedy, 1.0, T)), 0.0)
    run_ = torch.cumsum(w, 1)
    keep &= ((run_ - w < top_p * run_[:, -1:]) | (top_p >= 1)) & (w >= min_p)
    w = torch.where(greedy, (rank == 0).double(), torch.where(keep, w, 0.0))
    w = torch.zeros_like(w).scatter_(1, order, w)
    return w / w.sum(1, keepdim=True)


def _verify_plain(st):
    """a node whose parent is the last accepted one is accepted where u < p(c) / q(c); after a rejection p becomes max(p - q, 0), normalised (without a draft's rows q is one at c: p loses c).
    In the end the first token, in the vocabulary's order, whose running mass is over u[first node]"""
    case = st["case"]
    S, N, V = case["seqs"], case["nodes"], case["vocab"]
    parent, token, u = st["parents"].view(S, N).long(), st["tokens"].view(S, N).long(), st["u"].view(S, N).double()
    P = _weights(st["logits"], st["params"]).view(S, N, V)
    Q = _weights(st["guess"], st["params"]).view(S, N, V) if st["guess"] is not None else None
    seq = torch.arange(S, device=u.device)
    cur, p, n = torch.zeros_like(seq), P[:, 0].clone(), torch.ones_like(seq)
    path = torch.full((S, N + 1), -1, dtype=torch.int32, device=u.device)
    path[:, 0] = 0
    for i in range(1, N):
        asked, c = parent[:, i] == cur, token[:, i]
        pc = p[seq, c]
        q = Q[seq, cur] if Q is not None else torch.zeros_like(p).scatter_(1, c[:, None], 1.0)
        yes = asked & (u[:, i] * q[seq, c] < pc)
        left = (p - q).clamp(min=0) if Q is not None else p * (1 - q)
        total = left.sum(1, keepdim=True)
        left = torch.where(total > 0, left / torch.where(total > 0, total, 1.0), p)
        p = torch.where(yes[:, None], P[:, i], torch.where(asked[:, None], left, p))
        cur = torch.where(yes, i, cur)
        path[seq, torch.where(yes, n, N)] = i
        n = n + yes
    run_ = torch.cumsum(p, 1)
    at = (run_ <= u[:, :1] * run_[:, -1:]).sum(1)
    at = torch.minimum(at, (p > 0).long().mul(torch.arange(V, device=u.device)).amax(1))
    path[:, :N] = torch.where(torch.arange(N, device=u.device) < n[:, None], path[:, :N], -1)
    st["ids"].copy_(at.int())
    st["path"].copy_(path[:, :N].reshape(-1))
    st["n_path"].copy_(n.int())
    return {"ids": st["ids"], "path": st["path"], "n_path": st["n_path"]}


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
_made = []


def _backend():
    """the program's context: made once"""
    if not _made:
        from powerserve_b200 import capi
        _made.append(capi.CudaBackend(capi.ModelDesc(512, 1536, 1, 8, 2, 64, 1024, 64, 1e-5, 64, 0, 5e5, 1.0, 1.0, 0, 1, 0, 1)))
    return _made[0]


def _paged(state):
    """the program's handle of the cache's memory"""
    if "paged" not in state:
        from powerserve_b200 import capi
        L, N, G = state["codes"].shape[:3]
        state["paged"] = capi.PagedCache(_backend(), L, N, state["case"]["page"], G, SHAPES[state["case"]["shape"]][2], codes=state["codes"], scales=state["scales"], refs=state.get("refs"))
    return state["paged"]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"attn": _attn_plain, "store": _store_plain, "room": _room_plain, "fork": _fork_plain, "compact": _compact_plain, "verify": _verify_plain}[op](state)
    be = _backend()
    if op == "verify":
        be.verify(state["ids"], state["path"], state["n_path"], state["nodes"], state["parents"], state["tokens"], state["logits"], case["vocab"], state["params"], state["u"],
                  draft_logits=state["guess"], draft_samplers=None if state["guess"] is None else state["params"])
        return {"ids": state["ids"], "path": state["path"], "n_path": state["n_path"]}
    cache = _paged(state)
    if op == "attn":
        be.paged_attn(cache, 0, state["out"], state["q"], state["seqs"], SHAPES[case["shape"]][0], state["scale"], tree_mask=state["mask"])
        return {"out": state["out"]}
    if op == "store":
        be.paged_store(cache, 0, state["k"], state["v"], state["seqs"])
        be.paged_load(cache, 0, state["k_held"], state["v_held"], state["seqs"])
        return {"k": state["k_held"], "v": state["v_held"], "scales": state["scales"]}
    if op == "room":
        be.paged_edit(cache, state["edits"][0][0], state["held"][0])
        be.paged_edit(cache, state["edits"][1][0], state["held"][1])
        return {"table": state["table"], "refs": state["refs"], "held": state["held"]}
    if op == "fork":
        be.paged_edit(cache, state["turns"][state["turn"]][0], state["held"])
        return _forked(state)
    be.paged_compact(cache, state["moves"])
    return {"codes": state["codes"], "scales": state["scales"]}


# ---------------------------------------------------------------------------------------------------------------- what a pass needs, and its exact result
def work(case):
    op = case["op"]
    if op == "verify":      # every row of logits once, but the draft's of nodes that have no child
        rows = case["seqs"] * (case["nodes"] + (case["nodes"] - 1 if case["draft"] and case["fan"] == 1 else case["nodes"] // 2 if case["draft"] else 0))
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}
    H, G, D, L = SHAPES[case["shape"]]
    P = case["page"]
    if op == "room":        # every page's holders once, the tables' new entries
        n = _lengths(case["past"], case["seqs"], True, 0)
        taken = float((_up(n + case["tok"], P) - _up(n, P)).sum())
        pages = float(np.maximum(_up(n, P), 1).sum()) + case["seqs"] * (_up(case["tok"], P) + 1) + case["spare"]
        return {"bytes": 2 * (4 * pages + 12 * taken + 36.0 * case["seqs"]), "flops": pages}
    if op == "fork":        # the filled blocks of the prompts' last pages, and the tables
        n = _lengths(case["past"], case["seqs"], True, 1)
        blocks = float(_up(n % P, BLOCK).sum()) * case["answers"]
        return {"bytes": 2 * blocks * L * 2 * G * (BLOCK * D + 4) + 12.0 * float(_up(n, P).sum()) * case["answers"], "flops": blocks * L * G}
    if op == "compact":     # kept slots, half of them at least
        slots = 0.75 * case["keep"] * case["seqs"] * case["layers"]
        return {"bytes": 4.0 * slots * G * (D + 4 / BLOCK), "flops": 4.0 * slots * G * D}
    tok, size = _tokens(case), 4 if case["io"] == "float32" else 2
    n_kv = _lengths(case["past"], case["seqs"], case["ragged"], 0) + tok
    if op == "store":       # numbers in, codes out; codes in, numbers out
        return {"bytes": 4.0 * float(tok.sum()) * G * (D * (size + 1) + 4 / BLOCK), "flops": 6.0 * float(tok.sum()) * G * D}
    slots = float(n_kv.sum())
    return {"bytes": 2 * slots * G * (D + 4 / BLOCK) + 2.0 * size * float(tok.sum()) * H * D, "flops": 4.0 * float((n_kv * tok).sum()) * H * D}


def exact(case, seed):
    if case["op"] in ("room", "verify"):    # whole numbers
        return None
    return {"attn": _exact_attn, "store": _exact_store, "fork": _exact_fork, "compact": _exact_compact}[case["op"]](prepare(case, seed))


def _held(st, layer, page, slot, kv):
    """[slots][kv heads][channels]: the numbers that slots of pages stand for"""
    _, G, D, _ = SHAPES[st["case"]["shape"]]
    P, d = st["case"]["page"], torch.arange(D, device="cuda")
    at = ((slot // 8)[:, None] * (D // 16) + d // 16) * 128 + (slot % 8)[:, None] * 16 + d % 16 if kv == 0 else ((slot // 16)[:, None] * D + d) * 16 + (slot % 16)[:, None]
    codes = st["codes"][layer, page, :, kv].gather(2, at[:, None].expand(-1, G, -1))
    return codes.double() * st["scales"][layer, page, :, kv].gather(2, (slot // BLOCK)[:, None, None].expand(-1, G, 1)).double()


def _exact_attn(st):
    case = st["case"]
    H, G, D, _ = SHAPES[case["shape"]]
    R, P, out = H // G, case["page"], torch.zeros_like(st["q"], dtype=torch.float64)
    t0 = m0 = 0
    for s in range(case["seqs"]):
        n, T = int(st["n_kv"][s]), int(st["n_tok"][s])
        sees = torch.ones(T, n, dtype=torch.bool, device="cuda")
        sees[:, n - T:] = torch.tril(torch.ones(T, T, device="cuda")).bool() if st["mask"] is None else st["mask"][m0:m0 + T * T].view(T, T).bool()
        if st["hidden"] is not None:
            sees &= ~st["hidden"][s, :n].bool()[None]
        j = torch.arange(n, device="cuda")
        page = st["table"][s, j // P].long()
        k, v = _held(st, 0, page, j % P, 0), _held(st, 0, page, j % P, 1)
        for h in range(H):
            z = st["q"][t0:t0 + T, h * D:(h + 1) * D].double() @ k[:, h // R].T * st["scale"]
            p = torch.softmax(z.masked_fill(~sees, -math.inf), -1).nan_to_num(0.0)
            out[t0:t0 + T, h * D:(h + 1) * D] = p @ v[:, h // R]
        t0, m0 = t0 + T, m0 + T * T
    return {"out": out}


def _exact_store(st):
    """(scales and quotients are numbers of 32 bits by definition: what is rounded to 8 bits is theirs)"""
    case = st["case"]
    _, G, D, _ = SHAPES[case["shape"]]
    P, scales = case["page"], st["scales"].double()
    held = [torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    t0 = 0
    for s in range(case["seqs"]):
        n, T = int(st["n_kv"][s]), int(st["n_tok"][s])
        for b in range((n - T) // BLOCK, (n - 1) // BLOCK + 1):
            lo, hi, page = max(b * BLOCK, n - T), min((b + 1) * BLOCK, n), int(st["table"][s, b * BLOCK // P])
            for kv, x in enumerate((st["k"], st["v"])):
                rows = x[t0 + lo - (n - T):t0 + hi - (n - T)].double().view(-1, G, D)
                c = (rows.abs().amax((0, 2)) / 127.0).float().double()
                if lo > b * BLOCK:
                    c = torch.maximum(c, scales[0, page, :, kv, b % (P // BLOCK)])
                scales[0, page, :, kv, b % (P // BLOCK)] = c
                code = (rows / torch.where(c > 0, c, 1.0)[None, :, None]).float().round().clamp(-127, 127).double()
                held[kv][t0 + lo - (n - T):t0 + hi - (n - T)] = (code * c[None, :, None]).view(-1, G * D)
        t0 += T
    return {"k": held[0], "v": held[1], "scales": scales}


def _exact_fork(st):
    """one after another: shares, releases, then pages to the answers in order"""
    case, P = st["case"], st["case"]["page"]
    _, (gone, come), begun, old, new, n = st["turns"][0]
    refs, gone, begun = st["refs"].tolist(), gone.tolist(), begun.tolist()
    old, new, h, scales = old.tolist(), new.tolist(), n // 2, st["scales"].double()
    for i in range(h):
        for p in begun[i][:_up(old[h + i], P)]:
            refs[p] += 1
    for i in range(h):
        for p in gone[i][_up(new[i], P):_up(old[i], P)]:
            refs[p] -= 1
    free = [p for p, r in enumerate(refs) if r == 0]
    for i in range(h):
        last, part = begun[i][_up(old[h + i], P) - 1], old[h + i] % P
        if part and refs[last] == 1:
            continue
        to = free.pop(0)
        if part:
            refs[last] -= 1
            scales[:, to, :, :, :_up(part, BLOCK)] = st["scales"][:, last, :, :, :_up(part, BLOCK)].double()
    return {"tables": None, "refs": None, "held": None, "codes": None, "scales": scales}


def _exact_compact(st):
    case, scales = st["case"], st["scales"].double()
    P, first, keep, n_keep, table = case["page"], st["first"].tolist(), st["keep"].tolist(), st["n_keep"].tolist(), st["table"].tolist()
    for s in range(case["seqs"]):
        source = list(range(first[s] // BLOCK * BLOCK, first[s])) + [first[s] + k for k in keep[s][:n_keep[s]]]
        for b in range(0, len(source), BLOCK):
            to = first[s] // BLOCK * BLOCK + b
            at = sorted({(table[s][j // P], j % P // BLOCK) for j in source[b:b + BLOCK]})
            scales[:, table[s][to // P], :, :, to % P // BLOCK] = torch.stack([st["scales"][:, p, :, :, c] for p, c in at]).amax(0).double()
    return {"codes": None, "scales": scales}
