"""ps_cuda_sample against a plain form in 64 bits: every filter alone and together, ties, rows of equal logits, odd logits, odd settings."""
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


def check(be, x, rows, u, pad=0):
    n, V = x.shape
    p = S.settings(rows)
    full = np.full((n, V + pad), 1e30, np.float32)      # (between the rows: what would win)
    full[:, :V] = x
    xd, pd, ud, idd, prd = be.upload(full), be.upload(p), be.upload(np.asarray(u, np.float32)), be.upload(np.full(n + 1, -7, np.int32)), be.upload(np.full(n + 1, -7, np.float32))
    be.sample(idd, prd, xd, V, n, pd, ud, row_stride=V + pad)
    ids, probs = idd.numpy(np.int32), prd.numpy()
    assert ids[n] == -7 and probs[n] == -7
    for r in range(n):
        with np.errstate(all="ignore"):
            i, pr = S.sample(x[r], *(float(p[r][f]) if f != "top_k" else int(p[r][f]) for f in ("temperature", "top_k", "top_p", "min_p")), float(np.float32(u[r])))
        assert ids[r] == i, (r, rows[r], u[r], ids[r], i)
        assert abs(probs[r] - pr) <= 2 * S.EPS * pr + 1e-12, (r, probs[r], pr)      # rounded once; weights are whole numbers of 2^-44
    be.sample(idd, None, xd, V, n, pd, ud, row_stride=V + pad)
    assert np.array_equal(idd.numpy(np.int32), ids)
    for b in (xd, pd, ud, idd, prd):
        b.free()


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.2, 0, 1.0, 0.1), (0.8, 50, 0.95, 0.02), (1.5, 2000, 0.99, 0.001), (0.0, 0, 1.0, 0.0), (5.0, 0, 0.999, 0.0), (3.0, 700, 0.5, 0.0),
           (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (0.01, 0, 0.9, 0.0), (30.0, 0, 0.7, 0.0), (1.0, 64, 0.3, 0.5)]


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 1000, 4097, 32000, 128256, 151936, 262144])
@pytest.mark.parametrize("pad", [0, 3])
def test_filters(be, V, pad):
    r = np.random.default_rng(V)
    n = len(FILTERS) * 2
    x = (r.standard_normal((n, V)) * 2.5).astype(np.float32)
    x[:, r.integers(0, V, 8)] += 6
    check(be, x, FILTERS * 2, r.random(n), pad)


@pytest.mark.parametrize("V", [500, 32000, 128256])
def test_equal_logits(be, V):
    """the border lies inside a run of equal logits: lower tokens come first"""
    r = np.random.default_rng(V)
    x = np.stack([np.zeros(V), np.full(V, -3.0), np.where(np.arange(V) % 2, 1.0, 0.5), r.integers(0, 4, V), np.where(r.random(V) < 0.5, 0.0, -0.0), np.round(r.standard_normal(V) * 2)]).astype(np.float32)
    for f in [(1.0, V // 3, 1.0, 0.0), (1.0, 0, 0.35, 0.0), (0.5, V // 2, 0.77, 0.0), (2.0, 0, 1.0, 0.9), (0.0, 0, 1.0, 0.0), (1e30, 7, 1.0, 0.0), (1e30, 0, 0.25, 0.0)]:
        check(be, x, [f] * len(x), r.random(len(x)))


def test_neighbouring_floats(be):
    """thousands of logits that differ in their last bits alone"""
    V = 20000
    r = np.random.default_rng(1)
    x = (np.float32(8.0).view(np.uint32) + r.integers(0, 3000, (6, V)).astype(np.uint32)).view(np.float32)
    check(be, x, [(1.0, 5000, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (0.3, 9999, 0.6, 0.0), (0.001, 0, 0.5, 0.0), (1e-6, 100, 1.0, 0.0), (1e-6, 0, 0.99, 0.0)], r.random(6))


def test_odd_logits(be):
    V = 5000
    r = np.random.default_rng(2)
    x = (r.standard_normal((10, V)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, :4999] = -np.inf
    x[4, [7, 70, 4000]] = np.inf
    x[5] = np.where(r.random(V) < 0.99, -np.inf, x[5])
    x[6] = np.finfo(np.float32).min
    x[7] = np.where(np.arange(V) % 3, np.finfo(np.float32).min, np.finfo(np.float32).max)
    x[8, 17] = np.inf
    x[9] = np.float32(1e-42) * np.arange(V, dtype=np.float32)
    for f in FILTERS:
        check(be, x, [f] * 10, r.random(10))


def test_odd_settings(be):
    V = 3000
    r = np.random.default_rng(3)
    rows = [(-1.0, 0, 1, 0), (np.nan, 0, 1, 0), (np.inf, 0, 1, 0), (1e-38, 0, 1, 0), (1.0, -5, 1, 0), (1.0, 10 ** 9, 1, 0), (1.0, 0, np.nan, 0), (1.0, 0, -1, 0), (1.0, 0, 2, 0), (1.0, 0, 1, np.nan),
            (1.0, 0, 1, -1), (1.0, 0, 1, 7), (np.inf, 100, 0.5, 0), (1.0, 3000, 1, 0), (1.0, 2999, 1, 0)]
    x = (r.standard_normal((len(rows), V)) * 2).astype(np.float32)
    check(be, x, rows, r.random(len(rows)))


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan])
def test_ends_of_the_random_numbers(be, u):
    r = np.random.default_rng(4)
    x = (r.standard_normal((len(FILTERS), 9000)) * 2).astype(np.float32)
    check(be, x, FILTERS, [u] * len(FILTERS))


def test_many_rows_and_the_share_of_each_token(be):
    """drawn with an even grid of numbers, every token comes as often as its probability says"""
    V, n = 50, 4096
    x = np.broadcast_to(np.random.default_rng(5).standard_normal(V).astype(np.float32), (n, V)).copy()
    xd, pd, ud, idd = be.upload(x), be.upload(S.settings([(1.0, 0, 1.0, 0.0)] * n)), be.upload(((np.arange(n) + 0.5) / n).astype(np.float32)), be.upload(np.zeros(n, np.int32))
    be.sample(idd, None, xd, V, n, pd, ud)
    got = np.bincount(idd.numpy(np.int32), minlength=V) / n
    p = np.exp(x[0].astype(np.float64))
    assert np.abs(got - p / p.sum()).max() <= 1.0 / n + 1e-6      # (an interval of the grid holds its length times n points, to one)
    for b in (xd, pd, ud, idd):
        b.free()


def test_refusals(be):
    x = be.empty(64)
    for match, a in [("rows of", dict(vocab=0)), ("rows of", dict(vocab=1 << 19, row_stride=1 << 19)), ("rows of", dict(row_stride=3)), ("rows of", dict(rows=-1)), ("null", dict(ids=0)), ("null", dict(logits=0)),
                     ("null", dict(samplers=0)), ("null", dict(u=0)), ("aligned", dict(u=x.ptr + 2))]:
        args = dict(ids=x, probs=x, logits=x, vocab=4, rows=1, samplers=x, u=x, row_stride=4) | a
        with pytest.raises(capi.PsCudaError, match=match):
            be.sample(**args)
    be.sample(x, x, x, 4, 0, x, x)
    x.free()
