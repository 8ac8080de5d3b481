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
