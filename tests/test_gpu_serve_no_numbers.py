"""ps_cuda_attn_tree on queries that hold no numbers, and on scores beyond float32: such a row is NaN in every channel, whatever kernel and number of splits it
meets; zeros say that a row sees nothing.  The rows beside it are what they are without it."""
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


def attend(be, c, q, H):
    qd, od = be.upload(q), be.upload(np.full(q.shape, 7.0, np.float32))
    be.attn_tree(od, qd, c.table, H, c.G, c.D, S.scale_of(c.D), cache_type=c.type)
    out = od.numpy(np.float32, q.shape)
    qd.free()
    od.free()
    return out


# one token and several, caches of one split, of a few and of many
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("lens,toks", [([40], [1]), ([100], [2]), ([700], [1]), ([6000] * 4, [1] * 4), ([300] * 80, [1] * 80), ([40], [9]), ([5000], [30])])
def test_queries_that_are_no_numbers(be, dtype, D, lens, toks):
    H, G, n = 8, 2, sum(toks)
    c = S.Caches(be, lens, toks, G, D, dtype=dtype, weight=True, seed=D + n)
    r = np.random.default_rng(n)
    q = r.standard_normal((n, H * D)).astype(np.float32)
    want = attend(be, c, q, H)
    t, h = n - 1, 5
    for bad in (np.nan, np.inf):
        x = q.copy()
        x[t, h * D + 3] = bad
        out = attend(be, c, x, H).reshape(n, H, D)
        assert np.isnan(out[t, h]).all(), (bad, out[t, h])
        ok = np.ones((n, H), bool)
        ok[t, h] = False
        assert np.array_equal(out[ok].view(np.uint32), want.reshape(n, H, D)[ok].view(np.uint32))
    c.free()


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("lens,toks", [([40], [1]), ([700], [1]), ([300] * 80, [1] * 80), ([5000], [30])])
def test_scores_beyond_float32(be, D, lens, toks):
    """finite operands, a product above float32's largest number"""
    H, G, n = 8, 2, sum(toks)
    c = S.Caches(be, lens, toks, G, D, seed=D)
    q = np.random.default_rng(n).standard_normal((n, H * D)).astype(np.float32)
    q[0, :D] = 1e30 * np.sign(c.k[0][7, :D])
    for b in range(2):      # (one key, by 1e12)
        c.k[0][7] = c.k[0][7] * np.float32(1e6)
    kd = be.upload(c.k[0])
    c.table["k"][0] = kd.ptr
    out = attend(be, c, q, H)
    assert np.isnan(out[0, :D]).all()
    kd.free()
    c.free()


def test_a_row_that_sees_nothing_is_zeros_though_its_query_is_no_number(be):
    for D in (64, 128, 96):
        for tok in (1, 12):
            c = S.Caches(be, [90], [tok], 2, D, hidden=True, seed=D)
            c.hid[0][:] = 1
            c.bufs[3].free()
            c.bufs[3] = be.upload(c.hid[0])
            c.table["hidden"][0] = c.bufs[3].ptr
            assert (attend(be, c, np.full((tok, 8 * D), np.nan, np.float32), 8) == 0).all()
            c.free()
