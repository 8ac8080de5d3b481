"""Calls that the serving operators' documentation allows and that are easily forgotten: the output in the queries' place, sequences that share their K and V, arrays that begin
anywhere, odd scales, more gathered weights than a launch's workspace takes, empty caches, weights in place with positions elsewhere, more rows than a launch has."""
import numpy as np
import pytest
import torch

from powerserve_b200 import capi
from tests import _serve as S
from tests import test_gpu_serve_attention as A
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu
LAYOUTS = [([300, 40], [1, 2]), ([6000] * 3, [1] * 3), ([1000], [1]), ([900, 200], [20, 7]), ([100, 30], [30, 9])]


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("lens,toks", LAYOUTS)
def test_the_output_in_the_queries_place(be, D, lens, toks):  # noqa: F811
    c = S.Caches(be, lens, toks, 2, D, seed=D, weight=True)
    q, want = A.run(be, c, 8)
    for i in range(len(lens)):
        be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.bufs[4 * i + 2].ptr, c.w[i].ctypes.data, c.w[i].nbytes))
    qd = be.upload(q)
    be.attn_tree(qd, qd, c.table, 8, 2, D, S.scale_of(D))
    assert np.array_equal(qd.numpy(np.uint32, q.shape), want.view(np.uint32))
    qd.free()
    c.free()


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("toks", [[1, 1, 1], [12, 3, 5]])
def test_sequences_that_share_their_cache(be, D, toks):  # noqa: F811
    """a common beginning, of which each sees as much as it has, itself the last tokens of it"""
    c = S.Caches(be, [700, 650, 300], toks, 2, D, n_ctx=704, seed=D, weight=True)
    for i in (1, 2):
        c.table["k"][i], c.table["v"][i] = c.table["k"][0], c.table["v"][0]
        c.k[i], c.v[i] = c.k[0], c.v[0]
    A.check(be, c, 8, weight=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("lens,toks", LAYOUTS[:1] + LAYOUTS[2:4])
@pytest.mark.parametrize("which", ["k", "v", "all"])
def test_arrays_that_begin_anywhere(be, dtype, D, lens, toks, which):  # noqa: F811
    H, G, n = 8, 2, sum(toks)
    c = S.Caches(be, lens, toks, G, D, dtype=dtype, n_ctx=-(-max(lens) // 8) * 8, hidden=True, weight=True, seed=D)
    es = 4 if dtype == "f32" else 2
    bufs = []

    def moved(a, by):
        a = np.ascontiguousarray(a)
        b = be.upload(np.concatenate([np.zeros(by, np.uint8), a.reshape(-1).view(np.uint8)]))
        bufs.append(b)
        return b.ptr + by

    for i in range(len(lens)):
        for name, a in (("k", c.k[i]), ("v", c.v[i])):
            if which in (name, "all"):
                c.table[name][i] = moved(a if dtype == "f32" else S.bf16(a)[0], es)
        if which == "all":
            c.table["weight"][i], c.table["hidden"][i] = moved(c.w[i], 4), moved(c.hid[i], 3)
    r = np.random.default_rng(n)
    q, masks = r.standard_normal((n, H * D)).astype(np.float32), [S.tree(t, r) for t in toks]
    odd = 4 if which == "all" else 0
    out = be.upload(np.full(n * H * D + 8, 7.0, np.float32))
    be.attn_tree(out.ptr + odd, moved(q, odd), c.table, H, G, D, S.scale_of(D), tree_mask=moved(np.concatenate([m.reshape(-1) for m in masks]), 1), cache_type=c.type)
    want, w, bound, wbound = S.attention(q, c, H, S.scale_of(D), masks)
    got = out.numpy(np.float32)
    assert (got[:odd // 4] == 7).all() and (got[odd // 4 + n * H * D:] == 7).all()
    assert (np.abs(got[odd // 4:odd // 4 + n * H * D].reshape(n, -1) - want).max(-1) <= bound).all()
    for i, l in enumerate(lens):
        a = be.read_device(int(c.table["weight"][i]), c.w[i].size).reshape(c.w[i].shape)
        assert np.abs(a[:, :l] - c.w[i][:, :l] - w[i]).max() <= wbound[i] + 8 * S.EPS * (w[i].max() + 1) and (a[:, l:] == c.w[i][:, l:]).all()
    out.free()
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
def test_odd_scales(be, D, scale):  # noqa: F811
    """zero: every slot that a token sees weighs the same"""
    for lens, toks in LAYOUTS[:1] + LAYOUTS[3:4]:
        c = S.Caches(be, lens, toks, 2, D, seed=D, weight=True)
        n = sum(toks)
        q = np.random.default_rng(n).standard_normal((n, 8 * D)).astype(np.float32)
        qd, od = be.upload(q), be.empty(q.size)
        be.attn_tree(od, qd, c.table, 8, 2, D, scale)
        want, _, bound, _ = S.attention(q, c, 8, float(np.float32(scale)))
        assert (np.abs(od.numpy(np.float32, q.shape) - want).max(-1) <= bound + 2.0 ** -38 * 8).all()
        qd.free()
        od.free()
        c.free()


def test_more_weights_than_a_launch_takes(be):  # noqa: F811
    """three sequences whose scores need 0.4 GB each: two launches, in one workspace.  All keys equal: outputs are means of the values, weights shares of one"""
    H, G, D, T, n = 32, 8, 64, 32, 100000
    c = 100032
    k, v = torch.zeros(c, G * D, device="cuda"), torch.zeros(3, G * D, c, device="cuda")
    for s in range(3):
        v[s, :, :1000 * (s + 1)] = 1.0
    w = torch.zeros(3, G, c, device="cuda")
    q, out = torch.ones(3 * T, H * D, device="cuda"), torch.zeros(3 * T, H * D, device="cuda")
    t = np.zeros(3, capi.CACHE)
    for s in range(3):
        t[s] = (k.data_ptr(), v[s].data_ptr(), w[s].data_ptr(), 0, 0, 0, 0, c, n - 1000 * s, T, 0)
    mask = torch.ones(3 * T * T, dtype=torch.uint8, device="cuda")
    be.attn_tree(out, q, t, H, G, D, 1.0, tree_mask=mask)
    o, ws = out.cpu().numpy().reshape(3, -1), w.cpu().numpy()
    for s in range(3):
        m = n - 1000 * s
        # sums in parts, as of any long cache: a few steps of the whole
        assert np.abs(o[s] * m / (1000 * (s + 1)) - 1).max() <= 256 * S.EPS
        assert np.abs(ws[s, :, :m].astype(np.float64) * m / (T * H // G) - 1).max() <= 256 * S.EPS and (ws[s, :, m:] == 0).all()


@pytest.mark.parametrize("go", [3, 100])
@pytest.mark.parametrize("place", ["weight", "pos"])
def test_weights_in_place_and_positions_elsewhere_and_empty_caches(be, go, place):  # noqa: F811
    G, D, lens = 2, 64, [500, 0, 300]
    r = np.random.default_rng(go)
    t, host, dev = np.zeros(3, capi.CACHE), [], []
    for i, n in enumerate(lens):
        c = n + 4
        a = [r.standard_normal((c, G * D)).astype(np.float32), r.standard_normal((G * D, c)).astype(np.float32), r.random((G, c)).astype(np.float32), np.stack([r.permutation(c).astype(np.int32) for _ in range(G)]),
             np.full((G, c), -5, np.float32 if place == "pos" else np.int32)]
        b = [be.upload(x) for x in a]
        host.append(a)
        dev.append(b)
        t[i] = (b[0].ptr, b[1].ptr, b[2].ptr, b[2].ptr if place == "weight" else b[4].ptr, b[3].ptr, b[3].ptr if place == "pos" else b[4].ptr, 0, c, n, 0, max(n - go, 0))
    be.kv_evict(t, G, D, 2, 10)
    for i, n in enumerate(lens):
        k, v, w, p, to = host[i]
        keep, wk, wv = max(n - go, 0), k.copy(), v.copy()
        ww, wp = (w.copy(), to.copy()) if place == "weight" else (to.copy(), p.copy())
        for g in range(G):
            src, dst = S.evict(w[g], p[g], n, keep, 2, 10) if n else ([], [])
            at = slice(g * D, (g + 1) * D)
            wk[dst, at], wv[at, dst] = k[src, at], v[at, src]
            ww[g, :keep], wp[g, :keep] = w[g, :keep], p[g, :keep]
            ww[g, dst], wp[g, dst] = w[g, src], p[g, src]
        b = dev[i]
        assert np.array_equal(b[0].numpy(np.float32, k.shape), wk) and np.array_equal(b[1].numpy(np.float32, v.shape), wv)
        assert np.array_equal((b[2] if place == "weight" else b[4]).numpy(np.float32, w.shape), ww) and np.array_equal((b[3] if place == "pos" else b[4]).numpy(np.int32, p.shape), wp)
        for x in b:
            x.free()


def test_caches_that_nothing_names(be):  # noqa: F811
    """no slots filled, no arrays: nothing to attend to, nothing to cut"""
    t = np.zeros(2, capi.CACHE)
    t["n_ctx"] = 16
    be.kv_evict(t, 2, 64)
    be.attn_tree(0, 0, t, 4, 2, 64, 1.0)
    be.sync()


def test_more_rows_than_a_launch(be):  # noqa: F811
    V, R = 8, (1 << 20) + 5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(R, V, generator=g, device="cuda")
    u = torch.rand(R, generator=g, device="cuda")
    table = np.zeros(R, capi.SAMPLER)
    table["temperature"], table["top_p"] = np.arange(R) % 2, 1.0        # every other row: the largest logit
    sd = torch.from_numpy(table.view(np.float32).reshape(R, 4)).cuda()
    ids, probs = torch.full((R + 2,), -7, dtype=torch.int32, device="cuda"), torch.full((R + 2,), -7.0, device="cuda")
    be.sample(ids, probs, x, V, R, sd, u)
    assert ids[R:].tolist() == [-7, -7] and probs[R:].tolist() == [-7.0, -7.0]
    w = torch.exp(x.double() - x.double().amax(1, keepdim=True))
    run = torch.cumsum(w, 1)
    goal = u.double()[:, None] * run[:, -1:]
    want = torch.where(torch.arange(R, device="cuda") % 2 == 0, x.argmax(1), (run <= goal).sum(1))
    sure = ((run - goal).abs().amin(1) > 1e-12) | (torch.arange(R, device="cuda") % 2 == 0)      # (weights are whole numbers of 2^-44)
    assert bool((ids[:R].long() == want)[sure].all()) and int((~sure).sum()) < 10
