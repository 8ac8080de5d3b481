"""Attention over 8-bit pages against a plain form in 64 bits: head layouts, page sizes, lengths from one slot on, trees, hidden slots, rows that see nothing, split lengths, sequences that take no part,
what lies behind the last slot."""
import numpy as np
import pytest

from powerserve_b200 import capi
from tests import _paged as P
from tests import _serve as S
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu


def run(be, c, toks, H, masks=None, hidden=None, seed=0, q_scale=1.0, scale=None, dtype="f32", layer=0, q=None, in_place=False):  # noqa: F811
    n = sum(toks)
    if q is None:
        q = (np.random.default_rng(seed + 99).standard_normal((max(n, 1), H * c.D)) * q_scale).astype(np.float32)
    scale = S.scale_of(c.D) if scale is None else scale
    io, bits = capi.F32, np.uint32
    qh = q
    if dtype == "bf16":
        qh, q = S.bf16(q)
        io, bits = capi.BF16, np.uint16
    qd, od = be.upload(np.concatenate([qh, np.zeros((2, H * c.D), qh.dtype)])), be.upload(np.full((n + 2, H * c.D), 7, bits))     # (rows behind the last one stay)
    md = None if masks is None else be.upload(np.concatenate([m.reshape(-1) for m in masks] + [np.zeros(16, np.uint8)]))
    hd = None if hidden is None else [be.upload(h) for h in hidden]
    be.paged_attn(c.cache, layer, qd if in_place else od, qd, c.seqs(toks, hd), H, scale, tree_mask=md, io_type=io)
    out = (qd if in_place else od).numpy(bits, (n + 2, H * c.D))
    assert (out[n:] == (0 if in_place else 7)).all()
    be.sync()
    for b in [qd, od] + ([md] if md else []) + (hd or []):
        b.free()
    out = out[:n].view(np.float32) if dtype == "f32" else (out[:n].astype(np.uint32) << 16).view(np.float32)
    return q, out


def check(be, c, toks, H, masks=None, hidden=None, dtype="f32", layer=0, **more):  # noqa: F811
    scale = more.get("scale") or S.scale_of(c.D)
    q, out = run(be, c, toks, H, masks, hidden, dtype=dtype, layer=layer, **more)
    want, bound = P.attention(q, c, toks, H, scale, masks, hidden, layer)
    assert np.isfinite(out).all()
    off = np.abs(out - want)
    lim = bound[:, None] + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)     # (bfloat16: half a step of the result)
    assert (off <= lim + 1e-30).all(), (off.max(), bound[off.max(-1).argmax()])
    # beside that bound, which every rounding at its worst would reach: roundings of either sign leave a few steps
    assert np.linalg.norm(out - want) <= (64 * S.EPS + (2.0 ** -8 if dtype == "bf16" else 0.0)) * np.linalg.norm(want) + 1e-30
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (14, 2, 64), (8, 8, 128), (32, 8, 128), (6, 2, 96), (3, 1, 32), (4, 2, 256), (33, 3, 160), (64, 2, 64), (10, 2, 128), (18, 2, 64)])
def test_one_token_of_each(be, dtype, page, H, G, D):  # noqa: F811
    c = P.Cache(be, [1, 2, 127, 128, 129, 300], G, D, page, seed=H + D)
    check(be, c, [1] * 6, H, dtype=dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96, 256])
@pytest.mark.parametrize("toks", [[5, 1, 16, 3], [12, 32, 0, 20], [1, 2, 3, 40], [0, 0, 9, 0]])
@pytest.mark.parametrize("hidden", [False, True])
def test_trees(be, dtype, D, toks, hidden):  # noqa: F811
    lens, r = [300, 40, 700, 61], np.random.default_rng(D)
    c = P.Cache(be, lens, 2, D, 32, layers=2, seed=D)
    hid = [np.where(np.arange(n) < n - t, r.random(n) < 0.2, False).astype(np.uint8) for n, t in zip(lens, toks)] if hidden else None
    check(be, c, toks, 8, masks=[S.tree(t, r) for t in toks], hidden=hid, dtype=dtype, layer=1)


@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("R", [1, 3, 4, 8, 32])
def test_chunks_that_see_what_came_before(be, D, R):  # noqa: F811
    c = P.Cache(be, [200, 256, 64, 500], 1, D, 64, seed=R)
    check(be, c, [200, 33, 64, 256], R)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("toks", [[1], [7], [32]])
@pytest.mark.parametrize("G,D", [(2, 64), (1, 128)])
def test_long_caches(be, page, toks, G, D):  # noqa: F811
    c = P.Cache(be, [9001], G, D, page, seed=3)
    check(be, c, toks, 4 * G)


@pytest.mark.parametrize("n", [31, 200, 600])
def test_many_sequences_of_all_lengths(be, n):  # noqa: F811
    r = np.random.default_rng(n)
    lens = np.exp(r.uniform(0, np.log(900), n)).astype(int).clip(1, 900).tolist()
    toks = [int(r.integers(0, min(4, x) + 1)) for x in lens]
    c = P.Cache(be, lens, 1, 64, 16, seed=n)
    check(be, c, toks, 4)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tok", [1, 9, 40])
def test_rows_that_see_nothing(be, D, tok):  # noqa: F811
    """hidden past and a mask without ones: zeros; the other rows are what they are without them"""
    c = P.Cache(be, [150, 90], 2, D, 16, seed=1)
    masks = [np.tril(np.ones((tok, tok), np.uint8)) for _ in range(2)]
    masks[0][tok // 2] = 0
    hidden = [np.concatenate([np.ones(150 - tok), np.zeros(tok)]).astype(np.uint8), np.zeros(90, np.uint8)]
    q, out = run(be, c, [tok, tok], 8, masks, hidden)
    assert (out[tok // 2] == 0).all()
    check(be, c, [tok, tok], 8, masks, hidden)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tok", [1, 20])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_queries_that_are_no_numbers(be, D, tok, bad):  # noqa: F811
    """such a row is NaN, all others stay what they are"""
    c = P.Cache(be, [170, 400], 2, D, 32, seed=2)
    q, out = run(be, c, [tok, tok], 8)
    q = q.copy()
    q[tok, 3 * D + 5] = bad
    _, got = run(be, c, [tok, tok], 8, q=q)
    hit = np.zeros(out.shape, bool)
    hit[tok, 3 * D:4 * D] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit].view(np.uint32), out[~hit].view(np.uint32))
    c.free()


@pytest.mark.parametrize("tok", [1, 20])
def test_scores_above_the_range(be, tok):  # noqa: F811
    c = P.Cache(be, [170], 2, 64, 32, seed=2)
    q, out = run(be, c, [tok], 8)
    q = q.copy()
    q[0, :64] *= np.float32(1e37)
    _, got = run(be, c, [tok], 8, q=q, scale=100.0)
    assert np.isnan(got[0, :64]).all() and np.isfinite(got[0, 64:]).all()
    c.free()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30, 3.0])
@pytest.mark.parametrize("D", [64, 128])
def test_odd_scales(be, scale, D):  # noqa: F811
    c = P.Cache(be, [300, 20], 2, D, 16, seed=4)
    q, out = run(be, c, [9, 1], 8, scale=scale)
    want, bound = P.attention(q, c, [9, 1], 8, scale)
    assert (np.abs(out - want).max(-1) <= bound + 1e-30).all()
    c.free()


def test_queries_of_zeros_and_of_one_large_number(be):  # noqa: F811
    c = P.Cache(be, [300], 2, 64, 16, seed=5)
    q = np.random.default_rng(5).standard_normal((3, 512)).astype(np.float32)
    q[0, :64] = 0.0
    q[1, 64:128] *= np.float32(1e-20)
    q[1, 70] = 4.0
    q[2, :64] = np.float32(1e-42)
    q, out = run(be, c, [3], 8, q=q)
    want, bound = P.attention(q, c, [3], 8, S.scale_of(64))
    assert (np.abs(out - want).max(-1) <= bound + 1e-30).all()
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("toks", [[1, 1, 1], [12, 3, 5]])
@pytest.mark.parametrize("D", [64, 128])
def test_the_output_in_the_queries_place_and_pages_that_are_shared(be, dtype, toks, D):  # noqa: F811
    c = P.Cache(be, [700, 650, 300], 2, D, 64, seed=D)
    for i in (1, 2):        # a common beginning
        c.tables[i][:4] = c.tables[0][:4]
        be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.dev[i].ptr, c.tables[i].ctypes.data, c.tables[i].nbytes))
    _, a = run(be, c, toks, 8, dtype=dtype)
    _, b = run(be, c, toks, 8, dtype=dtype, in_place=True)
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    check(be, c, toks, 8, dtype=dtype)


def test_rows_that_begin_anywhere(be):  # noqa: F811
    for D in (64, 128):
        c = P.Cache(be, [300, 40], 2, D, 16, seed=6)
        toks = [3, 1]
        q, want = run(be, c, toks, 8)
        qd = be.upload(np.concatenate([np.zeros(1, np.float32), q.reshape(-1)]))
        od = be.upload(np.zeros(q.size + 3, np.float32))
        be.paged_attn(c.cache, 0, od.ptr + 4, qd.ptr + 4, c.seqs(toks), 8, S.scale_of(D))
        assert np.array_equal(od.numpy(np.uint32)[1:q.size + 1].reshape(q.shape), want.view(np.uint32))
        qd.free()
        od.free()
        c.free()


@pytest.mark.parametrize("tok", [1, 20])
def test_a_table_that_names_no_page(be, tok):  # noqa: F811
    """its slots are left out, other sequences are what they were, the next sync reports it"""
    for D in (64, 128):
        c = P.Cache(be, [300, 290], 2, D, 16, seed=7)
        q, want = run(be, c, [tok, tok], 8)
        for bad in (-1, c.n_pages, 2 ** 31 - 1):
            t = c.tables[0].copy()
            t[5] = bad
            be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.dev[0].ptr, t.ctypes.data, t.nbytes))
            with pytest.raises(capi.PsCudaError, match="names what is not there"):
                run(be, c, [tok, tok], 8)
            qd, od = be.upload(q), be.empty(q.size)
            be.paged_attn(c.cache, 0, od, qd, c.seqs([tok, tok]), 8, S.scale_of(D))
            with pytest.raises(capi.PsCudaError, match="names what is not there"):
                be.sync()
            be._ck(be.L.ps_cuda_memcpy_d2h(be.h, (buf := np.empty_like(q)).ctypes.data, od.ptr, q.nbytes))
            assert np.array_equal(buf[tok:].view(np.uint32), want[tok:].view(np.uint32)) and np.isfinite(buf).all()
            qd.free()
            od.free()
        c.free()


def test_the_same_bits_every_time(be):  # noqa: F811
    c = P.Cache(be, [900, 1300, 77, 5000], 2, 128, 64, seed=8)
    for toks in ([1, 1, 1, 1], [20, 3, 9, 31]):
        _, a = run(be, c, toks, 16)
        for _ in range(5):
            _, b = run(be, c, toks, 16)
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    c.free()


@pytest.mark.parametrize("tok,R,many", [(1, 4, 50), (1, 8, 50), (2, 8, 30), (8, 4, 18)])
@pytest.mark.parametrize("D", [64, 160])
@pytest.mark.parametrize("at,spread", [(0, 0.0), (0, 1.0), (100, 0.0), (5000, 0.3), (11990, 0.0)])
def test_one_heavy_slot_and_a_long_tail(be, tok, R, many, D, at, spread):  # noqa: F811
    """A slot that has nearly all of the mass, and twelve thousand whose weights are 2^-24 of it or less and together up to a thousandth; the heavy one's V is zero, so that the output is theirs.  Sequences share the pages,
    so many that a CTA takes all tiles of one.

    The bound, with e = 2^-24: a score is off by e (2 D M + 6 Z) as elsewhere, and by 6 Z e more for the difference of its tile's reference and the row's (all in units of e^x: numerator and denominator);
    exponentials, factors and the digits' sums by 40 e twice.  A weight is rounded by e of its tile's largest, so a tile's 128 slots by 128 e of that one, and the tiles' largest are at most the whole mass: 130 e max|v|.
    The numerator is one addition a tile, n / 128; the denominator in a lane four a tile at most, n / 32, and a factor a tile: n / 8 e for both."""
    n, G = 12000, 8
    c = P.Cache(be, [n], G, D, P=64, layers=1, seed=51, junk=False)
    r = np.random.default_rng([52, D, at])
    j = np.arange(n)
    page, slot = c.tables[0][j // 64], j % 64
    k, v = r.integers(-100, 101, (n, G, D)), r.integers(100, 128, (n, G, D))
    k[at], v[at] = 127, 0
    for kv, x in enumerate((k, v)):
        c.codes[0, page[:, None, None], np.arange(G)[None, :, None], kv, c.index[kv][slot][:, None, :]] = x
    sk, sv = np.full((n // 16, G), 0.01 * spread / np.sqrt(D)), 0.01 * (1 + r.random((n // 16, G)))
    sk[at // 16], k16 = 0.01, at // 16 * 16
    k[k16:k16 + 16][np.arange(k16, k16 + 16) != at] = 0
    c.codes[0, page[k16:k16 + 16, None, None], np.arange(G)[None, :, None], 0, c.index[0][slot[k16:k16 + 16]][:, None, :]] = k[k16:k16 + 16]
    b = np.arange(n // 16) * 16
    for kv, s in enumerate((sk, sv)):
        c.scales[0, c.tables[0][b // 64], :, kv, b % 64 // 16] = s
    c.cache.codes.free(), c.cache.scales.free()
    cache = capi.PagedCache(be, 1, c.n_pages, 64, G, D, codes=be.upload(c.codes), scales=be.upload(c.scales), refs=c.cache.refs)
    seqs = np.zeros(many, capi.PAGED_SEQ)
    seqs["table"], seqs["n_kv"], seqs["n_tok"], seqs["n_table"] = c.dev[0].ptr, n, tok, len(c.tables[0])
    H, rows = G * R, many * tok
    top = np.log(2.0) * r.choice([24.02, 24.05, 24.4, 25.0, 22.0], (rows, H))
    q = np.repeat((top / (127 * 0.01 * D))[..., None], D, 2)
    q = q.astype(np.float32).reshape(rows, H * D)
    out = be.upload(np.full((rows, H * D), 7, np.float32))
    up = be.upload(q)
    mask = be.upload(np.ones((many, tok, tok), np.uint8))
    be.paged_attn(cache, 0, out, up, seqs, H, 1.0, tree_mask=mask)
    got = out.numpy(np.float32, (rows, H, D)).astype(np.float64)
    kk, vv = c.values(0, 0), c.values(0, 1)
    for h in range(H):
        z = q[:, h * D:(h + 1) * D].astype(np.float64) @ kk[:, h // R].T
        p = np.exp(z - z.max(-1, keepdims=True))
        want = p @ vv[:, h // R] / p.sum(-1, keepdims=True)
        M = np.abs(q[:, h * D:(h + 1) * D]).max(-1) * np.abs(kk[:, h // R]).max()
        bound = S.EPS * (2 * (2 * D * M + 12 * np.abs(z).max(-1)) + 80 + 130 + n / 8) * np.abs(vv[:, h // R]).max()
        off = np.abs(got[:, h] - want).max(-1)
        assert (off <= bound).all(), (h, (off / bound).max(), off.max() / np.abs(want).max())
    for x in (out, up, mask, cache.codes, cache.scales):
        x.free()
    c.cache.refs.free()
    for d in c.dev:
        d.free()


@pytest.mark.parametrize("tok,R", [(1, 4), (1, 8), (4, 4), (8, 4), (20, 4)])
@pytest.mark.parametrize("D", [64, 160])
@pytest.mark.parametrize("block,q_scale,k_scale,rest", [(3, 1.0, 1e37, 1e-3), (20, 1e30, 1e8, 1e-33), (39, 1e30, 1e8, 1e-33)])
def test_scores_outside_float32_in_one_tile(be, tok, R, D, block, q_scale, k_scale, rest):  # noqa: F811
    """sixteen of 640 slots with scores above float32's range: no number; below it: the others are what there is.  In the first tile, inside, in the last one"""
    n, G = 640, 2
    for above in (True, False):
        c = P.Cache(be, [n, n], G, D, P=32, layers=1, seed=61, junk=False)
        for i in range(2):
            page, o = c.tables[i][block * 16 // 32], block * 16 % 32
            c.scales[0, c.tables[i][:n // 32], :, 0] = rest
            c.scales[0, page, :, 0, o // 16] = k_scale
            for s in range(16):
                c.codes[0, page[None], np.arange(G)[:, None], 0, c.index[0][o + s]] = 100 if above else -100
        q = np.abs(np.random.default_rng(62).standard_normal((2 * tok, G * R * D)) + 2.0).astype(np.float32) * np.float32(q_scale)
        hidden = np.zeros(n, np.uint8)
        if not above:
            hidden[block * 16:block * 16 + 16] = 1
        masks = [np.ones((tok, tok), np.uint8)] * 2
        if not above:
            c2 = P.Cache(be, [n, n], G, D, P=32, layers=1, seed=61, junk=False)
            c2.codes, c2.scales = c.codes.copy(), c.scales.copy()
            for i in range(2):
                c2.scales[0, c2.tables[i][block * 16 // 32], :, 0, block * 16 % 32 // 16] = rest
            want, bound = P.attention(q, c2, [tok, tok], G * R, 1.0, masks, [hidden, hidden])
            c2.free()
        c.cache.free()
        c.cache = capi.PagedCache(be, 1, c.n_pages, 32, G, D, codes=be.upload(c.codes), scales=be.upload(c.scales), refs=be.upload(c.refs))
        _, out = run(be, c, [tok, tok], G * R, masks, scale=1.0, q=q)
        if above:
            assert np.isnan(out).all()
        else:
            assert (np.abs(out - want) <= bound[:, None]).all(), (np.abs(out - want).max(), bound.max())
        c.free()
