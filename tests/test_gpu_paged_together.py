"""The operators on paged caches and the verification of drafted tokens as a server uses them, one after another: steps of conversations that draft, with no look at the device in between; between a caller's own
torch operations, in its graphs, from several threads, and on caches past 32 bits."""
import threading

import numpy as np
import pytest
import torch

from powerserve_b200 import capi
from tests import _paged as P
from tests import _serve as S
from tests.test_gpu_serve_attention import be  # noqa: F401
from tests.test_gpu_serve_paths import backend
from tests.test_gpu_serve_streams import busy, stream  # noqa: F401

pytestmark = pytest.mark.gpu


def records(kind, **fields):
    n = max(len(v) for v in fields.values() if hasattr(v, "__len__"))
    t = np.zeros(n, kind)
    for k, v in fields.items():
        t[k.rstrip("_")] = v
    return t


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (96, 32)])
@pytest.mark.parametrize("draft", [False, True])
def test_steps_of_conversations_that_draft(be, D, page, draft):  # noqa: F811
    """room is taken, drafted tokens are stored, attend, are verified, the accepted ones move together by the path that the verification left on the device, the rest is given back; a fourth conversation forks from the
    first one in between.  Everything is followed on the host by the plain forms"""
    G, H, V, S_, L = 2, 8, 300, 4, 2
    lens = [37, 5, 2 * page, 0]
    c = P.Cache(be, lens, G, D, page, layers=L, spare=60, room=12, seed=D, junk=False)
    r = np.random.default_rng(D)
    lens = [37, 5, 2 * page, 0]
    kinds = [(1.0, 0, 0.95, 0.0), (0.8, 40, 1.0, 0.0), (1.2, 0, 1.0, 0.02), (1.0, 0, 1.0, 0.0)]
    for step in range(6):
        if step == 3:       # the fourth begins with what the first one has
            rec = records(capi.PAGE_EDIT, table=[c.dev[3].ptr], from_=[c.dev[0].ptr], n_old=[lens[0]], n_new=[lens[0]], n_table=[len(c.tables[3])])
            be.paged_edit(c.cache, rec)
            P.edit(c.refs, page, [(c.tables[3], c.tables[0], lens[0], lens[0])])
            lens[3] = lens[0]
        live = [i for i in range(S_) if lens[i] > 0]
        nodes = [int(r.integers(2, 9)) for _ in live]
        past = [lens[i] for i in live]
        n = sum(nodes)
        # room
        edits = [(c.tables[i], None, lens[i], lens[i] + m) for i, m in zip(live, nodes)]
        be.paged_edit(c.cache, records(capi.PAGE_EDIT, table=[c.dev[i].ptr for i in live], n_old=past, n_new=[p + m for p, m in zip(past, nodes)], n_table=[len(c.tables[i]) for i in live]))
        held, copies = P.edit(c.refs, page, edits)
        assert held == [p + m for p, m in zip(past, nodes)]
        shape = (L, c.n_pages, G, 2, page // 16, -1)
        for src, dst, b in copies:
            c.codes.reshape(shape)[:, dst, :, :, :b] = c.codes.reshape(shape)[:, src, :, :, :b]
            c.scales[:, dst, :, :, :b] = c.scales[:, src, :, :, :b]
        c.lens = [lens[i] + (nodes[live.index(i)] if i in live else 0) for i in range(S_)]
        toks = [nodes[live.index(i)] if i in live else 0 for i in range(S_)]
        # both layers: rows in, attention
        masks, t0 = [], 0
        parents = np.full(n, -1, np.int32)
        for m in nodes:
            mask = np.zeros((m, m), np.uint8)
            for i in range(m):
                if i:
                    parents[t0 + i] = r.integers(max(0, i - 2), i)
                    mask[i] = mask[parents[t0 + i]]
                mask[i, i] = 1
            masks.append(mask)
            t0 += m
        every = [masks[live.index(i)] if i in live else np.zeros((0, 0), np.uint8) for i in range(S_)]
        md = torch.from_numpy(np.concatenate([m.reshape(-1) for m in masks])).cuda()
        outs = []
        for layer in range(L):
            k, v, q = [r.standard_normal((n, w)).astype(np.float32) for w in (G * D, G * D, H * D)]
            kd, vd, qd = [torch.from_numpy(x).cuda() for x in (k, v, q)]
            od = torch.zeros_like(qd)
            be.paged_store(c.cache, layer, kd, vd, c.seqs(toks))
            be.paged_attn(c.cache, layer, od, qd, c.seqs(toks), H, S.scale_of(D), tree_mask=md)
            kd.zero_(), vd.zero_(), qd.zero_()
            P.store(c, layer, k, v, toks)
            outs.append((od, *P.attention(q, c, toks, H, S.scale_of(D), every, layer=layer)))
        # verification, and the accepted slots move together
        logits, guess = [(r.standard_normal((n, V)) * 1.5).astype(np.float32) for _ in range(2)]
        guess = (logits + 0.3 * guess).astype(np.float32)
        sets = np.zeros(n, capi.SAMPLER)
        tokens, t0 = np.zeros(n, np.int32), 0
        for i, m in zip(live, nodes):
            sets[t0:t0 + m] = kinds[i]
            for j in range(1, m):
                tokens[t0 + j] = r.choice(V, p=P.distribution(guess[t0 + parents[t0 + j]], *sets[t0].tolist()))
            t0 += m
        u = r.random(n).astype(np.float32)
        dev = lambda x: torch.from_numpy(x).cuda()      # noqa: E731
        sd = dev(sets.view(np.int32).reshape(n, 4).copy())
        ids, path, n_path = [torch.full((k,), -9, dtype=torch.int32, device="cuda") for k in (len(live), n, len(live))]
        be.verify(ids, path, n_path, nodes, dev(parents), dev(tokens), dev(logits), V, sd, dev(u), draft_logits=dev(guess) if draft else None, draft_samplers=sd if draft else None)
        at = np.cumsum([0] + nodes[:-1])
        be.paged_compact(c.cache, records(capi.PAGE_MOVE, table=[c.dev[i].ptr for i in live], keep=[path.data_ptr() + 4 * int(a) for a in at], n_keep_dev=[n_path.data_ptr() + 4 * e for e in range(len(live))],
                                          first=past, n_kv=[p + m for p, m in zip(past, nodes)], n_keep=nodes, n_table=[len(c.tables[i]) for i in live]))
        # only now the host looks
        kept = []
        for e, (i, m) in enumerate(zip(live, nodes)):
            x = slice(at[e], at[e] + m)
            want, token = P.verify(parents[x], tokens[x], u[x], logits[x], sets[x].tolist(), guess[x] if draft else None, sets[x].tolist() if draft else None)
            assert path[x].tolist() == want + [-1] * (m - len(want)) and int(n_path[e]) == len(want) and int(ids[e]) == token
            P.compact(c, i, past[e], want)
            kept.append(past[e] + len(want))
        for od, want, bound in outs:
            assert (np.abs(od.cpu().numpy() - want).max(-1) <= bound).all()
        # the rest is given back
        be.paged_edit(c.cache, records(capi.PAGE_EDIT, table=[c.dev[i].ptr for i in live], n_old=[p + m for p, m in zip(past, nodes)], n_new=kept, n_table=[len(c.tables[i]) for i in live]))
        P.edit(c.refs, page, [(c.tables[i], None, p + m, k) for i, p, m, k in zip(live, past, nodes, kept)])
        for i, k in zip(live, kept):
            lens[i] = k
        c.lens = list(lens)
        codes, scales, refs = c.read()
        assert np.array_equal(refs, c.refs) and np.array_equal(codes, c.codes) and np.array_equal(scales.view(np.uint32), c.scales.view(np.uint32))
        assert all(np.array_equal(d.numpy(np.int32), t) for d, t in zip(c.dev, c.tables))
    be.sync()
    c.free()


def test_between_a_caller_s_operations(stream):  # noqa: F811
    be = backend()
    H, G, D = 8, 2, 64
    c = P.Cache(be, [900, 200, 3], G, D, 32, seed=5)
    toks = [20, 1, 3]
    r = np.random.default_rng(2)
    k, v, q = [r.standard_normal((24, w)).astype(np.float32) for w in (G * D, G * D, H * D)]
    P.store(c, 0, k, v, toks)
    want, bound = P.attention(q, c, toks, H, S.scale_of(D))
    with stream():
        src = [torch.from_numpy(x).cuda() for x in (k, v, q)]
        dst = [torch.zeros_like(x) for x in src]
        out, ko = torch.zeros(24, H * D, device="cuda"), torch.zeros(24, G * D, device="cuda")
        busy()
        for a, b in zip(dst, src):
            a.copy_(b)
        be.paged_store(c.cache, 0, dst[0], dst[1], c.seqs(toks))
        be.paged_attn(c.cache, 0, out, dst[2], c.seqs(toks), H, S.scale_of(D))
        be.paged_load(c.cache, 0, ko, None, c.seqs(toks))
        for a in dst:
            a.fill_(3.0)
        got, held = (out * 2).cpu().numpy() / 2, (ko * 2).cpu().numpy() / 2
    assert (np.abs(got - want).max(-1) <= bound).all()
    assert np.array_equal(held, np.concatenate([c.values(i, 0, dtype=np.float32)[c.lens[i] - t:].reshape(t, -1) for i, t in enumerate(toks)]))
    c.free()
    be.close()


@pytest.mark.parametrize("toks", [[20, 7, 1], [1, 1, 1], [20, 20, 12]])
def test_captured_and_replayed(toks):
    """two graphs of one context, which share its workspace, replayed in turn with other inputs, and eager calls between them"""
    be = backend()
    H, G, D, V, n = 8, 2, 64, 4000, sum(toks)
    caches = [P.Cache(be, [3900, 200, 70], G, D, 64, seed=s) for s in range(2)]
    r = np.random.default_rng(3)
    graphs = []
    for c in caches:
        q, k, v = [torch.zeros(n, w, device="cuda") for w in (H * D, G * D, G * D)]
        x, u = torch.zeros(n, V, device="cuda"), torch.rand(n, device="cuda")
        out = torch.zeros_like(q)
        ids, path, n_path = [torch.zeros(m, dtype=torch.int32, device="cuda") for m in (3, n, 3)]
        par = np.concatenate([np.arange(-1, t - 1) for t in toks]).astype(np.int32)
        parents, tokens = torch.from_numpy(par).cuda(), torch.zeros(n, dtype=torch.int32, device="cuda")
        sd = torch.from_numpy(S.settings([(1.0, 0, 1.0, 0.0)] * n).view(np.int32).reshape(n, 4).copy()).cuda()
        seqs = c.seqs(toks)

        def step():
            y = q * 2.0
            be.paged_store(c.cache, 0, k, v, seqs)
            be.paged_attn(c.cache, 0, out, y, seqs, H, S.scale_of(D))
            z = x * 2.0
            be.verify(ids, path, n_path, toks, parents, tokens, z, V, sd, u)
            return out + 1.0, ids + 5

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got, (q, k, v, x, u, tokens, path, n_path), c, (out, ids, parents, sd)))     # (all that the graph names is kept)
    for turn in range(6):
        g, (got_o, got_i), (q, k, v, x, u, tokens, path, n_path), c, _ = graphs[turn % 2]
        new = [r.standard_normal(t.shape).astype(np.float32) for t in (q, k, v, x)]
        for t, a in zip((q, k, v, x), new):
            t.copy_(torch.from_numpy(a))
        tok = r.integers(0, V, n).astype(np.int32)
        tok[1:] = np.where(r.random(n - 1) < 0.7, (new[3] * 2).argmax(1)[:-1], tok[1:])
        tokens.copy_(torch.from_numpy(tok))
        g.replay()
        if turn == 2:
            be.paged_load(graphs[1][3].cache, 0, torch.zeros(n, G * D, device="cuda"), None, graphs[1][3].seqs(toks))
        o, ids = got_o.cpu().numpy() - 1, (got_i - 5).cpu().tolist()
        if turn < 2:        # (what the eager call and the capture's own inputs stored)
            P.store(c, 0, np.zeros_like(new[1]), np.zeros_like(new[2]), toks)
        P.store(c, 0, new[1], new[2], toks)
        want, bound = P.attention(new[0] * 2, c, toks, H, S.scale_of(D))
        assert (np.abs(o - want).max(-1) <= bound + 2 * S.EPS * (np.abs(want).max(-1) + 1)).all()
        t0, un = 0, u.cpu().numpy()
        for s, t in enumerate(toks):
            e = slice(t0, t0 + t)
            w, token = P.verify(np.arange(-1, t - 1), tok[e], un[e], new[3][e] * 2, [(1.0, 0, 1.0, 0.0)] * t)
            assert path[e].tolist()[:len(w)] == w and int(n_path[s]) == len(w) and ids[s] == token
            t0 += t
    del graphs, g
    torch.cuda.synchronize()
    for c in caches:
        c.free()
    be.close()


def test_a_capture_that_asks_for_workspace_is_refused_and_goes_on():
    be = backend()
    c = P.Cache(be, [60000], 2, 64, 64, seed=6)
    q = torch.zeros(1, 8 * 64, device="cuda")
    out, one = torch.zeros_like(q), torch.zeros(4, device="cuda")
    small = P.Cache(be, [100], 2, 64, 64, seed=6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        a = one + 1.0
        with pytest.raises(capi.PsCudaError, match="workspace"):
            be.paged_attn(c.cache, 0, out, q, c.seqs([1]), 8, 0.125)
        be.paged_attn(small.cache, 0, out, q, small.seqs([1]), 8, 0.125)    # (nothing is left to join: no workspace)
        b = a + 1.0
    g.replay()
    assert b.cpu().tolist() == [2.0] * 4 and torch.isfinite(out).all()
    del g
    torch.cuda.synchronize()
    c.free()
    small.free()
    be.close()


def test_threads_on_one_context(be):  # noqa: F811
    caches = [P.Cache(be, [4000 + 300 * s, 30], 2, 64 if s < 2 else 128, 32, seed=s) for s in range(4)]
    bad = []

    def work(s):
        try:
            c = caches[s]
            toks = [9, 2] if s % 2 else [1, 1]
            n = sum(toks)
            q = np.random.default_rng(s).standard_normal((n, 8 * c.D)).astype(np.float32)
            want, bound = P.attention(q, c, toks, 8, S.scale_of(c.D))
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(40):
                    qd, out = torch.from_numpy(q).cuda(), torch.zeros(n, 8 * c.D, device="cuda")
                    be.paged_attn(c.cache, 0, out, qd, c.seqs(toks), 8, S.scale_of(c.D))
                    qd.zero_()
                    if not (np.abs(out.cpu().numpy() - want).max(-1) <= bound).all():
                        bad.append((s, k))
        except Exception as e:      # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    for c in caches:
        c.free()


def test_pages_past_32_bits(be):  # noqa: F811
    """attention, copies and compaction of pages whose codes lie behind 2^32 bytes, and of layers that do"""
    G, D, page, n_pages, L = 2, 128, 128, 34000, 3
    cache = capi.PagedCache(be, L, n_pages, page, G, D, refs=(refs := be.upload(np.concatenate([np.ones(n_pages - 6, np.int32), np.zeros(6, np.int32)]))),
                            codes=torch.zeros(L, n_pages, G, 2, page * D, dtype=torch.int8, device="cuda"), scales=torch.zeros(L, n_pages, G, 2, page // 16, device="cuda"))
    r = np.random.default_rng(8)
    tables = be.upload(np.full((2, 4), -1, np.int32))
    be.paged_edit(cache, records(capi.PAGE_EDIT, table=[tables.ptr], n_old=[0], n_new=[300], n_table=[4]))
    assert tables.numpy(np.int32)[:3].tolist() == [n_pages - 6, n_pages - 5, n_pages - 4]
    k, v, q = [r.standard_normal((m, w)).astype(np.float32) for m, w in ((300, G * D), (300, G * D), (2, 4 * G * D))]
    seqs = records(capi.PAGED_SEQ, table=[tables.ptr], n_kv=[300], n_tok=[300], n_table=[4])
    kd, vd, qd = [torch.from_numpy(x).cuda() for x in (k, v, q)]
    out, ko, vo = torch.zeros_like(qd), torch.zeros_like(kd), torch.zeros_like(vd)
    for layer in (0, 2):
        be.paged_store(cache, layer, kd, vd, seqs)
    be.paged_edit(cache, records(capi.PAGE_EDIT, table=[tables.ptr + 16], from_=[tables.ptr], n_old=[300], n_new=[301], n_table=[4]))     # (its last page is copied in all layers)
    keep = torch.arange(5, 250, dtype=torch.int32, device="cuda")
    be.paged_edit(cache, records(capi.PAGE_EDIT, table=[tables.ptr], n_old=[300], n_new=[0], n_table=[4]))
    be.paged_compact(cache, records(capi.PAGE_MOVE, table=[tables.ptr + 16], keep=[keep.data_ptr()], first=[0], n_kv=[300], n_keep=[245], n_table=[4]))
    two = records(capi.PAGED_SEQ, table=[tables.ptr + 16], n_kv=[245], n_tok=[245], n_table=[4])
    for layer in (0, 2):
        be.paged_load(cache, layer, ko, vo, two)
        for x, y in ((kd, ko), (vd, vo)):
            step = x.abs().max() / 127
            assert (y[:245] - x[5:250]).abs().max() <= 1.01 * step     # (two roundings to codes of half a step each)
        last = two.copy()
        last["n_tok"] = 2
        be.paged_attn(cache, layer, out, qd, last, 4 * G, S.scale_of(D))
        ks, vs = [y[:245].double().view(245, G, D).repeat_interleave(4, 1) for y in (ko, vo)]
        z = torch.einsum("thd,jhd->thj", qd.double().view(2, 4 * G, D), ks) * S.scale_of(D)
        z[0, :, 244] = -torch.inf
        want = torch.einsum("thj,jhd->thd", z.softmax(-1), vs).reshape(2, -1)
        assert (out - want).norm() <= 64 * S.EPS * want.norm()
    be.sync()
    tables.free()
    refs.free()
