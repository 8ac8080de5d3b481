"""Operators of a serving step that samples and drafts over long caches, and what each costs:

* attention of the tokens of one step - one per conversation, or a tree of drafted ones - over the conversations' caches (K in rows, V
  transposed, slots in any order), with the attention weight that every slot gathers added to a running sum;
* eviction: a cache is cut to the slots that gathered most, beside the first and the latest positions; kept rows move into freed slots;
* sampling with temperature, top-k, top-p and min-p, a setting per row, from given random numbers.

`run` computes the plain form, or where `own` is true makes the calls of this framework.
"""
import math

import numpy as np
import torch

own = False

F32, BF16 = 0, 30           # the cache's types, as the framework numbers them
TYPES = {"float32": (F32, torch.float32, 4), "bfloat16": (BF16, torch.bfloat16, 2)}
# one conversation's cache in one layer, as the framework's calls take it
CACHE = np.dtype([("k", "u8"), ("v", "u8"), ("weight", "u8"), ("weight_to", "u8"), ("pos", "u8"), ("pos_to", "u8"), ("hidden", "u8"),
                  ("n_ctx", "i4"), ("n_kv", "i4"), ("n_tok", "i4"), ("n_keep", "i4")])
# heads, kv heads, head size of the layers that the framework's models bring
SHAPES = {"qwen2-0.5b": (14, 2, 64), "llama-3.2-1b": (32, 8, 64), "llama-3.1-8b": (32, 8, 128)}


def listed():
    return [
        # the smallest step: four short chats of a small model, one token each
        {"name": "attn_chats_4", "op": "attn", "shape": "qwen2-0.5b", "type": "float32", "seqs": 4, "tok": 1, "past": 290, "ragged": True, "tree": False, "hidden": False, "weight": False},
        # a drafted tree of the speculative decoder's default size is checked against one conversation
        {"name": "attn_tree_12", "op": "attn", "shape": "llama-3.1-8b", "type": "float32", "seqs": 1, "tok": 12, "past": 1003, "ragged": False, "tree": True, "hidden": True, "weight": False},
        # a server's step: 64 conversations of all lengths, the slots' weights are gathered for a later eviction
        {"name": "attn_sessions_64", "op": "attn", "shape": "llama-3.1-8b", "type": "float32", "seqs": 64, "tok": 1, "past": 2040, "ragged": True, "tree": False, "hidden": False, "weight": True},
        # trees over caches in half the bytes, of different depths
        {"name": "attn_trees_bf16", "op": "attn", "shape": "llama-3.2-1b", "type": "bfloat16", "seqs": 8, "tok": 20, "past": 8100, "ragged": True, "tree": True, "hidden": True, "weight": False},
        # the widest tree over two long documents, weights gathered
        {"name": "attn_tree_32_long", "op": "attn", "shape": "llama-3.1-8b", "type": "float32", "seqs": 2, "tok": 32, "past": 32700, "ragged": False, "tree": True, "hidden": False, "weight": True},
        # every layer of a model at its budget: one token came, one goes
        {"name": "evict_step", "op": "evict", "shape": "llama-3.1-8b", "type": "float32", "sets": 32, "n": 1025, "keep": 1024, "sink": 4, "recent": 64, "ragged": False, "first": False},
        # after a prompt: four layers' caches are cut to a quarter
        {"name": "evict_prompt", "op": "evict", "shape": "llama-3.1-8b", "type": "float32", "sets": 4, "n": 8190, "keep": 2047, "sink": 4, "recent": 512, "ragged": False, "first": True},
        # caches of all lengths in half the bytes, some of them within their budget
        {"name": "evict_ragged_bf16", "op": "evict", "shape": "llama-3.2-1b", "type": "bfloat16", "sets": 12, "n": 5001, "keep": 1999, "sink": 1, "recent": 100, "ragged": True, "first": True},
        # one answer's next token
        {"name": "sample_1", "op": "sample", "rows": 1, "vocab": 151936, "pad": 0, "kind": "chat"},
        # the twelve rows of a drafted tree
        {"name": "sample_tree_12", "op": "sample", "rows": 12, "vocab": 128256, "pad": 0, "kind": "nucleus"},
        # a server's rows, each request with its own settings; rows further apart than the vocabulary
        {"name": "sample_sessions_64", "op": "sample", "rows": 64, "vocab": 128256, "pad": 64, "kind": "mixed"},
        # many answers to one question
        {"name": "sample_answers_256", "op": "sample", "rows": 256, "vocab": 151936, "pad": 0, "kind": "nucleus"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "evict", "sample"])
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 200), "vocab": _log(rng, 2000, 151936), "pad": rng.choice([0, 0, 1, 64]), "kind": rng.choice(["chat", "nucleus", "plain", "mixed"])}
    shape, typ = rng.choice(sorted(SHAPES)), rng.choice(["float32", "float32", "bfloat16"])
    if op == "evict":
        n = _log(rng, 64, 8192)
        keep = n - 1 if rng.random() < 0.4 else max(8, int(n * rng.uniform(0.1, 0.9)))
        return {"op": op, "shape": shape, "type": typ, "sets": _log(rng, 1, max(1, min(32, 32768 // n))), "n": n, "keep": keep, "sink": rng.choice([0, 1, 4]), "recent": _log(rng, 1, keep),
                "ragged": rng.random() < 0.5, "first": rng.random() < 0.5}
    seqs = _log(rng, 1, 64)
    tree = rng.random() < 0.5
    tok = _log(rng, 2, 32) if tree else rng.choice([1, 1, 1, _log(rng, 2, 32)])
    past = _log(rng, 1, max(32, min(32700, 65400 // seqs)))
    tok = max(1, min(tok, 2097152 // (seqs * (past + 32))))     # no dearer than the largest listed one
    return {"op": op, "shape": shape, "type": typ, "seqs": seqs, "tok": tok, "past": past, "ragged": rng.random() < 0.6, "tree": tree, "hidden": rng.random() < 0.4, "weight": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, most, count, least):
    r = np.random.Generator(np.random.SFC64([most, count]))     # a case's sizes are its own, whatever the seed
    if not case["ragged"]:
        return np.full(count, most, np.int64)
    n = np.exp(r.uniform(math.log(max(least, most // 8, 1)), math.log(most + 0.5), count)).astype(np.int64).clip(least, most)
    n[0] = most
    return n


def _tokens(case):
    if not (case["ragged"] and case["tree"]):
        return np.full(case["seqs"], case["tok"], np.int64)
    tok = np.random.Generator(np.random.SFC64([case["tok"], case["seqs"]])).integers(1, case["tok"] + 1, case["seqs"])
    tok[0] = case["tok"]
    return tok


def _tree(n, r):
    """mask [n][n] of a drafted tree: a node sees its ancestors and itself"""
    m = np.zeros((n, n), np.uint8)
    for i in range(n):
        if i:
            m[i] = m[int(r.integers(max(0, i - 4), i))]
        m[i, i] = 1
    return m


def _table(count, fields):
    t = np.zeros(count, CACHE)
    for name, v in fields.items():
        t[name] = [x.data_ptr() for x in v] if isinstance(v, torch.Tensor) else v
    return t


def _prepare_attn(case, seed):
    H, G, D = SHAPES[case["shape"]]
    S, (code, dt, _) = case["seqs"], TYPES[case["type"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    r = np.random.Generator(np.random.SFC64([int(seed) & 0x7FFFFFFF, 11]))
    past, tok = _lengths(case, case["past"], S, 0), _tokens(case)
    n_ctx = -(-(case["past"] + case["tok"] + 8) // 16) * 16
    k = torch.randn(S, n_ctx, G * D, generator=g, device="cuda")
    k[:, :, 0::D] += 3.0            # keys share a direction, as cached ones do
    k = k.to(dt)
    v = torch.randn(S, G * D, n_ctx, generator=g, device="cuda").to(dt)
    q = torch.randn(int(tok.sum()), H * D, generator=g, device="cuda") * 1.5
    weight = torch.rand(S, G, n_ctx, generator=g, device="cuda") if case["weight"] else None
    hidden = None
    if case["hidden"]:
        hidden = torch.rand(S, n_ctx, generator=g, device="cuda") < 0.03
        hidden &= torch.arange(n_ctx, device="cuda")[None] < torch.as_tensor(past, device="cuda")[:, None]
        hidden = hidden.to(torch.uint8)
    mask = torch.from_numpy(np.concatenate([_tree(int(t), r).reshape(-1) for t in tok])).cuda() if case["tree"] else None
    fields = {"k": k, "v": v, "n_ctx": n_ctx, "n_kv": past + tok, "n_tok": tok}
    fields |= {"weight": weight} if weight is not None else {}
    fields |= {"hidden": hidden} if hidden is not None else {}
    return {"case": case, "k": k, "v": v, "q": q, "out": torch.zeros_like(q), "weight": weight, "hidden": hidden, "mask": mask, "table": _table(S, fields),
            "n_kv": torch.as_tensor(past + tok, device="cuda"), "n_tok": torch.as_tensor(tok, device="cuda"), "n_max": int((past + tok).max()), "scale": 1.0 / math.sqrt(D), "type": code}


def _prepare_evict(case, seed):
    _, G, D = SHAPES[case["shape"]]
    S, (code, dt, _) = case["sets"], TYPES[case["type"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    n = _lengths(case, case["n"], S, 2)
    n_ctx = -(-(case["n"] + 8) // 16) * 16
    k = torch.randn(S, n_ctx, G * D, generator=g, device="cuda").to(dt)
    v = torch.randn(S, G * D, n_ctx, generator=g, device="cuda").to(dt)
    weight = torch.exp(torch.randn(S, G, n_ctx, generator=g, device="cuda") * 2.0)     # few slots gather most
    pos = torch.arange(n_ctx, device="cuda", dtype=torch.int32).expand(S, G, n_ctx).contiguous()
    if not case["first"]:       # earlier evictions have left the slots in no order; the newest token lies behind them
        order = torch.rand(S, G, n_ctx, generator=g, device="cuda")
        last = torch.as_tensor(n - 1, device="cuda")[:, None, None]
        order = torch.where(torch.arange(n_ctx, device="cuda") < last, order, 2.0)
        pos = (order.argsort(dim=-1, stable=True).to(torch.int32) * 3).contiguous()
    keep = np.minimum(n, case["keep"])
    to, pos_to = torch.zeros_like(weight), torch.zeros_like(pos)
    table = _table(S, {"k": k, "v": v, "weight": weight, "weight_to": to, "pos": pos, "pos_to": pos_to, "n_ctx": n_ctx, "n_kv": n, "n_keep": keep})
    return {"case": case, "k": k, "v": v, "weight": weight, "pos": pos, "weight_to": to, "pos_to": pos_to, "table": table, "n": torch.as_tensor(n, device="cuda"),
            "keep": torch.as_tensor(keep, device="cuda"), "n_max": int(n.max()), "type": code}


def _settings(case, r):
    """a row's [temperature, top-k, top-p, min-p]"""
    n, kind = case["rows"], case["kind"]
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


def _prepare_sample(case, seed):
    R, V = case["rows"], case["vocab"]
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    r = np.random.Generator(np.random.SFC64([int(seed) & 0x7FFFFFFF, 13]))
    logits = torch.randn(R, V + case["pad"], generator=g, device="cuda") * 2.5
    at = torch.randint(0, V, (R, 24), generator=g, device="cuda")      # a few tokens that the model holds for likely
    logits.scatter_add_(1, at, torch.rand(R, 24, generator=g, device="cuda") * 12.0)
    p = _settings(case, r)
    table = np.zeros(R, np.dtype([("temperature", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")]))
    table["temperature"], table["top_k"], table["top_p"], table["min_p"] = p[:, 0], p[:, 1].astype(np.int32), p[:, 2], p[:, 3]
    params = torch.from_numpy(table.view(np.int32).reshape(R, 4).copy()).cuda()
    u = torch.rand(R, generator=g, device="cuda")
    return {"case": case, "logits": logits, "params": params, "u": u, "ids": torch.zeros(R, dtype=torch.int32, device="cuda"), "probs": torch.zeros(R, device="cuda")}


def prepare(case, seed):
    return {"attn": _prepare_attn, "evict": _prepare_evict, "sample": _prepare_sample}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _attn_plain(st):
    """out[t] = sum_j p_tj v_j, p = softmax over the slots that token t sees of scale q_t.k_j; a slot's weight grows by its p of all tokens and heads"""
    case, n = st["case"], st["n_max"]
    H, G, D = SHAPES[case["shape"]]
    S, R, T = case["seqs"], H // G, case["tok"]
    dev, n_kv, n_tok = st["q"].device, st["n_kv"], st["n_tok"]
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
    k = st["k"][:, :n].float().view(S, n, G, D).permute(0, 2, 3, 1)
    v = st["v"][:, :, :n].float().view(S, G, D, n).transpose(2, 3)
    q = st["q"][row].view(S, T, G, R, D).permute(0, 2, 1, 3, 4).reshape(S, G, T * R, D) * st["scale"]
    s = torch.matmul(q, k).view(S, G, T, R, n)
    s = torch.where(sees[:, None, :, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.where(sees[:, None, :, None, :], torch.exp(s - torch.where(m > -math.inf, m, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.view(S, G, T * R, n), v).view(S, G, T, R, D).permute(0, 2, 1, 3, 4).reshape(S, T, H * D)
    st["out"][row[there]] = o[there]
    if st["weight"] is None:
        return {"out": st["out"]}
    st["weight"][:, :, :n] += p.sum((2, 3))
    return {"out": st["out"], "weight": st["weight"]}


def _evict_plain(st):
    """kept: the first and the latest positions, then the largest weights, the lower slot where equal; kept slots behind n_keep move into freed ones, in order"""
    case, n = st["case"], st["n_max"]
    _, G, D = SHAPES[case["shape"]]
    S, n_ctx = case["sets"], st["k"].shape[1]
    slot = torch.arange(n, device=st["k"].device)
    inside = (slot < st["n"][:, None])[:, None, :].expand(S, G, n)
    w, pos, keep = st["weight"][:, :, :n], st["pos"][:, :, :n], st["keep"][:, None, None]
    newest = torch.where(inside, pos, -1).amax(-1, keepdim=True)
    safe = inside & ((pos < case["sink"]) | (pos > newest - case["recent"]))
    order = torch.where(inside, w, -math.inf).argsort(dim=-1, descending=True, stable=True)
    rank = (safe.int() * 2 + inside.int()).gather(-1, order)
    order = order.gather(-1, rank.argsort(dim=-1, descending=True, stable=True))
    kept = torch.zeros_like(inside).scatter(-1, order, (slot < keep).expand(S, G, n))
    src, dst = (kept & (slot >= keep)).nonzero(as_tuple=True), (~kept & (slot < keep)).nonzero(as_tuple=True)
    k, v = st["k"].view(S, n_ctx, G, D), st["v"].view(S, G, D, n_ctx)
    k[dst[0], dst[2], dst[1]] = k[src[0], src[2], src[1]]
    v[dst[0], dst[1], :, dst[2]] = v[src[0], src[1], :, src[2]]
    front = (slot < keep).expand(S, G, n)
    st["weight_to"][:, :, :n] = torch.where(front, w, st["weight_to"][:, :, :n])
    st["pos_to"][:, :, :n] = torch.where(front, pos, st["pos_to"][:, :, :n])
    st["weight_to"][dst] = st["weight"][src]
    st["pos_to"][dst] = st["pos"][src]
    return {"k": st["k"], "v": st["v"], "weight": st["weight_to"], "pos": st["pos_to"]}


def _sample_plain(st):
    """of the sorted logits the first top_k, of those the fewest that hold top_p of the mass, of those the ones with min_p of the largest's; the first token, in the
    vocabulary's order, whose running mass is over u times all of it"""
    V = st["case"]["vocab"]
    par = st["params"]
    T, k, top_p, min_p = par[:, 0:1].view(torch.float32).double(), par[:, 1:2], par[:, 2:3].view(torch.float32).double(), par[:, 3:4].view(torch.float32).double()
    x = st["logits"][:, :V]
    x = torch.where(torch.isnan(x), -math.inf, x)
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = T <= 0
    rank = torch.arange(V, device=x.device)
    keep = ((k <= 0) | (rank < k)) & (xs > -math.inf)
    w = torch.where(keep, torch.exp((xs.double() - xs[:, :1].double()) / torch.where(greedy, 1.0, T)), 0.0)
    run = torch.cumsum(w, 1)
    keep &= ((run - w < top_p * run[:, -1:]) | (top_p >= 1)) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run = torch.cumsum(w, 1)
    at = (run <= st["u"].double()[:, None] * run[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).long().mul(rank).amax(1, keepdim=True))
    prob = w.gather(1, at) / run[:, -1:]
    at = torch.where(greedy, order[:, :1], at)
    st["ids"].copy_(at[:, 0].int())
    st["probs"].copy_(torch.where(greedy, 1.0, prob)[:, 0].float())
    return {"ids": st["ids"], "probs": st["probs"]}


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
_made = []


def _backend():
    """the program's context: made once"""
    if not _made:
        from powerserve_b200 import capi
        _made.append(capi.CudaBackend(capi.ModelDesc(512, 1536, 1, 8, 2, 64, 1024, 64, 1e-5, 64, 0, 5e5, 1.0, 1.0, 0, 1, 0, 1)))
    return _made[0]


def run(state):
    case = state["case"]
    if not own:
        return {"attn": _attn_plain, "evict": _evict_plain, "sample": _sample_plain}[case["op"]](state)
    be = _backend()
    if case["op"] == "sample":
        be.sample(state["ids"], state["probs"], state["logits"], case["vocab"], case["rows"], state["params"], state["u"], row_stride=case["vocab"] + case["pad"])
        return {"ids": state["ids"], "probs": state["probs"]}
    H, G, D = SHAPES[case["shape"]]
    if case["op"] == "evict":
        be.kv_evict(state["table"], G, D, n_sink=case["sink"], n_recent=case["recent"], cache_type=state["type"])
        return {"k": state["k"], "v": state["v"], "weight": state["weight_to"], "pos": state["pos_to"]}
    be.attn_tree(state["out"], state["q"], state["table"], H, G, D, state["scale"], tree_mask=state["mask"], cache_type=state["type"])
    return {"out": state["out"]} if state["weight"] is None else {"out": state["out"], "weight": state["weight"]}


# ---------------------------------------------------------------------------------------------------------------- what a pass needs, and its exact result
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 28.0 * case["rows"], "flops": 4.0 * n}
    H, G, D = SHAPES[case["shape"]]
    size = TYPES[case["type"]][2]
    if case["op"] == "evict":
        n = _lengths(case, case["n"], case["sets"], 2)
        keep = np.minimum(n, case["keep"])
        moved = (n - keep) * keep / n       # kept slots behind the new end, were they spread evenly
        return {"bytes": float(G * (8 * (n + keep) + 4 * moved * D * size).sum()), "flops": float(G * n.sum())}
    tok = _tokens(case)
    n_kv = _lengths(case, case["past"], case["seqs"], 0) + tok
    slots = float(n_kv.sum())
    return {"bytes": 2 * slots * G * D * size + 8.0 * float(tok.sum()) * H * D + (8.0 * slots * G if case["weight"] else 0.0), "flops": 4.0 * float((n_kv * tok).sum()) * H * D}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    return _exact_evict(st) if case["op"] == "evict" else _exact_attn(st)


def _exact_attn(st):
    case = st["case"]
    H, G, D = SHAPES[case["shape"]]
    R, out, weight = H // G, torch.zeros_like(st["q"], dtype=torch.float64), None if st["weight"] is None else st["weight"].double()
    t0 = m0 = 0
    for s in range(case["seqs"]):
        n, T = int(st["n_kv"][s]), int(st["n_tok"][s])
        sees = torch.ones(T, n, dtype=torch.bool, device="cuda")
        if st["mask"] is not None:
            sees[:, n - T:] = st["mask"][m0:m0 + T * T].view(T, T).bool()
        else:
            sees[:, n - T:] = torch.tril(torch.ones(T, T, device="cuda")).bool()
        if st["hidden"] is not None:
            sees &= ~st["hidden"][s, :n].bool()[None]
        for h in range(H):
            g = h // R
            z = st["q"][t0:t0 + T, h * D:(h + 1) * D].double() @ st["k"][s, :n, g * D:(g + 1) * D].double().T * st["scale"]
            p = torch.softmax(z.masked_fill(~sees, -math.inf), -1).nan_to_num(0.0)
            out[t0:t0 + T, h * D:(h + 1) * D] = p @ st["v"][s, g * D:(g + 1) * D, :n].double().T
            if weight is not None:
                weight[s, g, :n] += p.sum(0)
        t0, m0 = t0 + T, m0 + T * T
    return {"out": out} if weight is None else {"out": out, "weight": weight}


def _exact_evict(st):
    case = st["case"]
    _, G, D = SHAPES[case["shape"]]
    k, v, to, pos_to = st["k"].clone(), st["v"].clone(), st["weight_to"].double(), st["pos_to"].clone()
    for s in range(case["sets"]):
        n, keep = int(st["n"][s]), int(st["keep"][s])
        for g in range(G):
            w, pos = st["weight"][s, g, :n].double().cpu().numpy(), st["pos"][s, g, :n].cpu().numpy()
            safe = (pos < case["sink"]) | (pos > pos.max() - case["recent"])
            kept = set(np.lexsort((np.arange(n), -w, ~safe))[:keep].tolist())
            holes, movers = [j for j in range(keep) if j not in kept], sorted(j for j in kept if j >= keep)
            old = np.arange(keep)
            old[holes] = movers
            old = torch.from_numpy(old).cuda()
            k[s, :keep, g * D:(g + 1) * D] = st["k"][s, old, g * D:(g + 1) * D]
            v[s, g * D:(g + 1) * D, :keep] = st["v"][s, g * D:(g + 1) * D][:, old]
            to[s, g, :keep], pos_to[s, g, :keep] = st["weight"][s, g, old].double(), st["pos"][s, g, old]
    return {"k": k, "v": v, "weight": to, "pos": pos_to}


def _exact_sample(st):
    case, ids, probs = st["case"], [], []
    par = st["params"].cpu().numpy()
    u = st["u"].double().cpu().numpy()
    for r in range(case["rows"]):
        x = st["logits"][r, :case["vocab"]].double().cpu().numpy()
        T, top_p, min_p = (float(f) for f in par[r].view(np.float32)[[0, 2, 3]])
        if T <= 0:
            ids.append(int(np.argmax(x)))
            probs.append(1.0)
            continue
        best = np.argsort(-x, kind="stable")
        best = best[:int(par[r, 1])] if par[r, 1] > 0 else best
        w = np.exp((x[best] - x[best[0]]) / T)
        if top_p < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            best, w = best[before < top_p * w.sum()], w[before < top_p * w.sum()]
        best, w = best[w >= min_p], w[w >= min_p]
        order = np.argsort(best)
        best, w = best[order], w[order]
        at = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(w) - 1)
        ids.append(int(best[at]))
        probs.append(w[at] / w.sum())
    return {"ids": np.array(ids, np.int32), "probs": np.array(probs)}
