"""Rows of K and V into the 8-bit pages and back: codes, scales and values bit for bit against plain float32 arithmetic (numpy's division and rounding are IEEE's)."""
import numpy as np
import pytest

from powerserve_b200 import capi
from tests import _paged as P
from tests import _serve as S
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu
LAYOUTS = [([1], [1]), ([16, 17, 40], [16, 1, 40]), ([100, 37, 5], [1, 1, 1]), ([300, 129, 64], [290, 20, 64]), ([50, 33, 20], [0, 20, 0])]


def rows(c, toks, seed, scale=1.0):
    r = np.random.default_rng(seed)
    return [(r.standard_normal((sum(toks), c.G * c.D)) * scale).astype(np.float32) for _ in range(2)]


def same(c):
    codes, scales, _ = c.read()
    assert np.array_equal(codes, c.codes)
    assert np.array_equal(scales.view(np.uint32), c.scales.view(np.uint32))


@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_codes_and_scales(be, D, page, dtype):  # noqa: F811
    for n, (lens, toks) in enumerate(LAYOUTS):
        c = P.Cache(be, lens, 3, D, page, layers=2, seed=D + n)
        k, v = rows(c, toks, n, 0.3)
        if dtype == "bf16":
            (kb, k), (vb, v) = S.bf16(k), S.bf16(v)
        kd, vd = be.upload(kb if dtype == "bf16" else k), be.upload(vb if dtype == "bf16" else v)
        io = capi.F32 if dtype == "f32" else capi.BF16
        be.paged_store(c.cache, 1, kd, vd, c.seqs(toks), io_type=io)
        P.store(c, 1, k, v, toks)
        same(c)
        ko, vo = be.upload(np.full_like(k, np.nan)), be.upload(np.full_like(v, np.nan))
        be.paged_load(c.cache, 1, ko, vo, c.seqs(toks), io_type=io)
        t0 = 0
        for i, t in enumerate(toks):
            for d, kv in ((ko, 0), (vo, 1)):
                want = c.values(i, kv, 1, dtype=np.float32)[c.lens[i] - t:].reshape(t, c.G * D)
                got = d.numpy(np.float32 if dtype == "f32" else np.uint16)[:sum(toks) * c.G * D].reshape(sum(toks), -1)[t0:t0 + t]
                assert np.array_equal(got, want if dtype == "f32" else S.bf16(want)[0])
            t0 += t
        for b in (kd, vd, ko, vo):
            b.free()
        c.free()


def test_a_block_that_fills_token_by_token(be):  # noqa: F811
    """numbers that grow: every token raises its block's scale, and the codes before follow it"""
    c = P.Cache(be, [64], 2, 64, 32, seed=5)
    r = np.random.default_rng(6)
    for n in range(1, 41):
        c.lens[0] = n
        k, v = [(r.standard_normal((1, 128)) * 1.2 ** n).astype(np.float32) for _ in range(2)]
        kd, vd = be.upload(k), be.upload(v)
        be.paged_store(c.cache, 0, kd, vd, c.seqs([1]))
        P.store(c, 0, k, v, [1])
        kd.free()
        vd.free()
    same(c)
    c.free()


@pytest.mark.parametrize("which", ["zeros", "tiny", "ties", "large"])
def test_odd_numbers(be, which):  # noqa: F811
    c = P.Cache(be, [30, 20], 2, 64, 16, seed=7)
    toks = [30, 7]
    k, v = rows(c, toks, 8)
    if which == "zeros":
        k[:], v[3:20] = 0.0, -0.0
    elif which == "tiny":       # scales and quotients below the least normal number
        k *= np.float32(1e-40)
        v *= np.float32(1e-37)
    elif which == "ties":       # numbers between two codes
        k[:] = np.random.default_rng(1).integers(-253, 254, k.shape).astype(np.float32) / 2
        k[::16] = 127.0
        v[:] = 127.0
    else:
        k *= np.float32(5e37)
    kd, vd = be.upload(k), be.upload(v)
    be.paged_store(c.cache, 0, kd, vd, c.seqs(toks))
    P.store(c, 0, k, v, toks)
    same(c)
    kd.free()
    vd.free()
    c.free()


def test_numbers_that_are_none(be):  # noqa: F811
    """no number is held as 0; a block with an infinite one holds nothing else; neighbours keep what is theirs"""
    c = P.Cache(be, [48], 1, 64, 16, seed=9)
    k, v = rows(c, [48], 10)
    kk, vk = k.copy(), v.copy()
    k[3, 5], v[20, 60] = np.nan, np.nan
    kk[3, 5], vk[20, 60] = 0.0, 0.0
    kd, vd = be.upload(k), be.upload(v)
    be.paged_store(c.cache, 0, kd, vd, c.seqs([48]))
    P.store(c, 0, kk, vk, [48])
    same(c)
    k[40, 1] = np.inf
    be._ck(be.L.ps_cuda_memcpy_h2d(be.h, kd.ptr, k.ctypes.data, k.nbytes))
    be.paged_store(c.cache, 0, kd, vd, c.seqs([48]))
    codes, scales, _ = c.read()
    last = c.tables[0][2]
    assert (codes[0, last, 0, 0] == 0).all() and np.isinf(scales[0, last, 0, 0, 0])
    for p in c.tables[0][:2]:
        assert np.array_equal(codes[0, p], c.codes[0, p])
    assert np.array_equal(codes[0, last, 0, 1], c.codes[0, last, 0, 1])
    kd.free()
    vd.free()
    c.free()


@pytest.mark.parametrize("by", [4, 8, 12])
def test_rows_that_begin_anywhere(be, by):  # noqa: F811
    c = P.Cache(be, [40, 21], 2, 64, 16, seed=11)
    toks = [23, 21]
    k, v = rows(c, toks, 12)
    b = [be.upload(np.concatenate([np.zeros(by, np.uint8), a.reshape(-1).view(np.uint8)])) for a in (k, v)]
    be.paged_store(c.cache, 0, b[0].ptr + by, b[1].ptr + by, c.seqs(toks))
    P.store(c, 0, k, v, toks)
    same(c)
    out = be.upload(np.zeros(k.size + 4, np.float32))
    be.paged_load(c.cache, 0, out.ptr + by, None, c.seqs(toks))
    want = np.concatenate([c.values(i, 0, dtype=np.float32)[c.lens[i] - t:].reshape(t, -1) for i, t in enumerate(toks)])
    assert np.array_equal(out.numpy(np.float32)[by // 4:][:k.size].reshape(k.shape), want)
    for x in (*b, out):
        x.free()
    c.free()


def test_many_sequences(be):  # noqa: F811
    """more than a launch's table takes, some that take no part"""
    r = np.random.default_rng(13)
    lens = r.integers(1, 40, 600).tolist()
    toks = [int(r.integers(0, n + 1)) for n in lens]
    c = P.Cache(be, lens, 1, 32, 16, seed=14)
    k, v = rows(c, toks, 15)
    kd, vd = be.upload(k), be.upload(v)
    be.paged_store(c.cache, 0, kd, vd, c.seqs(toks))
    P.store(c, 0, k, v, toks)
    same(c)
    kd.free()
    vd.free()
    c.free()


def test_pages_past_32_bits(be):  # noqa: F811
    """a page whose codes lie behind 2^32 bytes"""
    G, D, page, n_pages = 8, 256, 128, 9000
    cache = capi.PagedCache(be, 1, n_pages, page, G, D)
    t = be.upload(np.array([n_pages - 1, n_pages - 2], np.int32))
    seqs = np.array([(t.ptr, 0, 130, 130, 2, 0)], capi.PAGED_SEQ)
    r = np.random.default_rng(16)
    k, v = [r.standard_normal((130, G * D)).astype(np.float32) for _ in range(2)]
    kd, vd = be.upload(k), be.upload(v)
    be.paged_store(cache, 0, kd, vd, seqs)
    ko, vo = be.empty(k.size), be.empty(v.size)
    be.paged_load(cache, 0, ko, vo, seqs)
    for x, d in ((k, ko), (v, vo)):
        got = d.numpy(np.float32, x.shape)
        step = np.abs(x.reshape(130, G, D)).max() / 127
        assert np.abs(got - x).max() <= 0.5001 * step
    be.sync()
    for b in (t, kd, vd, ko, vo):
        b.free()
    cache.free()


def test_a_table_that_names_no_page(be):  # noqa: F811
    """it is left out, nothing else changes, and the next sync reports it"""
    c = P.Cache(be, [40, 40], 2, 64, 16, seed=17)
    toks = [40, 40]
    k, v = rows(c, toks, 18)
    kd, vd = be.upload(k), be.upload(v)
    for bad in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        t = c.tables[0].copy()
        t[1] = bad
        be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.dev[0].ptr, t.ctypes.data, t.nbytes))
        be.paged_store(c.cache, 0, kd, vd, c.seqs(toks))
        with pytest.raises(capi.PsCudaError, match="names what is not there"):
            be.sync()
        be.paged_load(c.cache, 0, kd, vd, c.seqs([0, 0]))
        be.sync()
    P.store(c, 0, k, v, toks)
    codes, scales, _ = c.read()
    for i, p in enumerate(c.tables[0][:3].tolist() + c.tables[1][:3].tolist()):
        if i != 1:
            assert np.array_equal(codes[0, p], c.codes[0, p]) and np.array_equal(scales[0, p], c.scales[0, p])
    kd.free()
    vd.free()
    c.free()
