"""ps_cuda_kv_evict against a plain form: which slots stay, where the others go, and what is left as it was."""
import numpy as np
import pytest

from powerserve_b200 import capi
from tests import _serve as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = capi.CudaBackend(capi.ModelDesc(512, 1536, 1, 8, 2, 64, 1024, 64, 1e-5, 64, 0, 5e5, 1.0, 1.0, 0, 1, 0, 1))
    yield b
    b.close()


def check(be, lens, keeps, G, D, dtype="f32", n_sink=0, n_recent=0, pos=True, same=False, odd=0, seed=0, weights=None, order=False):
    r = np.random.default_rng(seed)
    t = np.zeros(len(lens), capi.CACHE)
    host, dev = [], []
    for i, (n, keep) in enumerate(zip(lens, keeps)):
        c = n + 2 + odd
        kind = np.uint32 if dtype == "f32" else np.uint16
        k, v = r.integers(0, np.iinfo(kind).max, (c, G * D), kind), r.integers(0, np.iinfo(kind).max, (G * D, c), kind)     # any bits move as they are
        w = np.exp(r.standard_normal((G, c)) * 2).astype(np.float32) if weights is None else weights((G, c), r).astype(np.float32)
        p = np.broadcast_to(np.arange(c, dtype=np.int32), (G, c)).copy()
        if order:
            p = np.stack([r.permutation(c).astype(np.int32) * 3 for _ in range(G)])
        wt, pt = np.full((G, c), -5.0, np.float32), np.full((G, c), -5, np.int32)
        host.append((k, v, w, p, wt, pt))
        b = [be.upload(a) for a in host[-1]]
        dev.append(b)
        t[i] = (b[0].ptr, b[1].ptr, b[2].ptr, b[2].ptr if same else b[4].ptr, b[3].ptr if pos else 0, (b[3].ptr if same else b[5].ptr) if pos else 0, 0, c, n, 0, keep)
    be.kv_evict(t, G, D, n_sink, n_recent, cache_type=capi.F32 if dtype == "f32" else capi.BF16)
    for i, (n, keep) in enumerate(zip(lens, keeps)):
        k, v, w, p, wt, pt = host[i]
        wk, wv, ww, wp = k.copy(), v.copy(), (w if same else wt).copy(), (p if same else pt).copy()
        for g in range(G):
            src, dst = S.evict(w[g], p[g] if pos else None, n, keep, n_sink, n_recent)
            assert len(src) == len(dst)
            at = slice(g * D, (g + 1) * D)
            wk[dst, at] = k[src, at]
            wv[at, dst] = v[at, src]
            ww[g, :keep] = w[g, :keep]
            ww[g, dst] = w[g, src]
            if pos:
                wp[g, :keep] = p[g, :keep]
                wp[g, dst] = p[g, src]
        b = dev[i]
        assert np.array_equal(b[0].numpy(k.dtype, k.shape), wk), "K rows"
        assert np.array_equal(b[1].numpy(v.dtype, v.shape), wv), "V columns"
        got = (b[2] if same else b[4]).numpy(np.uint32, w.shape)
        assert np.array_equal(got, ww.view(np.uint32)), "weights"
        assert np.array_equal((b[3] if same else b[5]).numpy(np.int32, p.shape), wp), "positions"
        if not same:
            assert np.array_equal(b[2].numpy(np.uint32, w.shape), w.view(np.uint32)) and np.array_equal(b[3].numpy(np.int32, p.shape), p)
        for x in b:
            x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("n,keep", [(1, 1), (1, 0), (2, 1), (65, 64), (100, 0), (100, 100), (1000, 100), (1000, 900), (1025, 1024), (3001, 1500)])
def test_sizes(be, dtype, D, n, keep):
    check(be, [n], [keep], 2, D, dtype=dtype, odd=n % 3, seed=n + D)


@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("order", [False, True])
@pytest.mark.parametrize("n_sink,n_recent", [(0, 0), (4, 0), (0, 32), (4, 64), (1000000, 0), (0, 1 << 30), (2, 299)])
def test_first_and_latest_positions(be, same, order, n_sink, n_recent):
    """(among them: more safe slots than are kept)"""
    check(be, [500, 2100, 31], [301, 2000, 30], 3, 64, n_sink=n_sink, n_recent=n_recent, same=same, order=order, seed=n_recent % 97)


@pytest.mark.parametrize("gone", [2, 3, 5, 7, 8, 9])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_few_go(be, gone, dtype):
    """what goes lies before the new end, behind it, and on both sides"""
    lens = [gone, gone + 1, 40, 300, 1026, 2049]
    check(be, lens, [n - gone for n in lens], 5, 64, dtype=dtype, n_sink=2, n_recent=9, order=True, seed=gone)
    check(be, lens, [n - gone for n in lens], 3, 128, dtype=dtype, n_recent=1, same=True, seed=gone, weights=lambda shape, r: r.integers(0, 4, shape))


@pytest.mark.parametrize("lens,keeps", [([40001], [9000]), ([50001], [300]), ([50001, 17, 33000], [49970, 9, 12345]), ([49152, 49153], [5000, 5000])])
@pytest.mark.parametrize("n_recent", [100, 20000])
def test_long_caches(be, lens, keeps, n_recent):
    """more slots than a thread has bits for, than shared memory has keys for, and more safe ones than are kept"""
    check(be, lens, keeps, 2, 32, dtype="bf16", n_sink=4, n_recent=n_recent, order=True, seed=len(lens) + n_recent)


@pytest.mark.parametrize("same", [False, True])
def test_without_positions(be, same):
    check(be, [700, 5], [350, 2], 2, 128, pos=False, same=same)


@pytest.mark.parametrize("what", ["equal", "few", "zeros", "odd", "tiny"])
@pytest.mark.parametrize("n,keep", [(400, 133), (5000, 4999), (5000, 17)])
def test_weights_that_tie_and_odd_ones(be, what, n, keep):
    def weights(shape, r):
        if what == "equal":
            return np.full(shape, 0.25)
        if what == "few":
            return r.integers(0, 3, shape) * 0.5
        if what == "zeros":
            return np.where(r.random(shape) < 0.5, 0.0, -0.0)
        if what == "tiny":
            return r.integers(0, 50, shape) * 1e-45
        return r.choice([np.nan, np.inf, -np.inf, 0.0, -1.0, 2.0], shape)

    check(be, [n], [keep], 2, 64, n_sink=1, n_recent=3, seed=n, weights=weights)


def test_more_caches_than_a_table(be):
    lens = [1 + (i * 53) % 300 for i in range(140)]
    check(be, lens, [n - n // (2 + i % 5) if i % 7 else n for i, n in enumerate(lens)], 2, 32, n_sink=2, n_recent=5)


def test_a_long_cache(be):
    check(be, [70001], [20000], 1, 32, n_sink=4, n_recent=1000)


def test_refusals(be):
    w, p, x = be.empty(64), be.empty(64), be.empty(64 * 64)
    t = np.zeros(1, capi.CACHE)
    t[0] = (x.ptr, x.ptr, w.ptr, w.ptr, p.ptr, p.ptr, 0, 16, 12, 0, 8)

    def bad(match, D=32, G=2, n_sink=0, n_recent=0, **fields):
        u = t.copy()
        for k, v in fields.items():
            u[k] = v
        with pytest.raises(capi.PsCudaError, match=match):
            be.kv_evict(u, G, D, n_sink, n_recent)

    bad("keeps", n_keep=13)
    bad("keeps", n_keep=-1)
    bad("holds", n_kv=17)
    bad("gathered", weight=0)
    bad("gathered", weight_to=0)
    bad("go together", pos_to=0)
    bad("positions", pos=0, pos_to=0, n_sink=1)
    bad("hidden", hidden=x.ptr)
    bad("first and", n_sink=-1)
    bad("head size", D=40)
    bad("no rows", v=0)
    be.kv_evict(t[:0], 2, 32)
    for b in (w, p, x):
        b.free()
