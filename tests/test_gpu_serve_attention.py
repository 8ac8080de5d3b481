"""ps_cuda_attn_tree against a plain form in 64 bits: cache types, head layouts, lengths from one slot on, trees, hidden slots, rows that see
nothing, gathered weights, sequences that take no part, more sequences than a launch's table holds."""
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


def run(be, c, H, masks=None, seed=0, q_scale=1.0, scale=None):
    D, n = c.D, sum(c.toks)
    q = (np.random.default_rng(seed + 99).standard_normal((max(n, 1), H * D)) * q_scale).astype(np.float32)
    scale = S.scale_of(D) if scale is None else scale
    qd, od = be.upload(q), be.upload(np.full((n + 2, H * D), 7.0, np.float32))     # (rows behind the last one stay)
    md = None if masks is None else be.upload(np.concatenate([m.reshape(-1) for m in masks] + [np.zeros(16, np.uint8)]))
    be.attn_tree(od, qd, c.table, H, c.G, D, scale, tree_mask=md, cache_type=c.type)
    out = od.numpy(np.float32, (n + 2, H * D))
    for b in (qd, od) + ((md,) if md else ()):
        b.free()
    assert (out[n:] == 7.0).all()
    return q, out[:n]


def check(be, c, H, masks=None, weight=False, **more):
    scale = more.get("scale") or S.scale_of(c.D)
    q, out = run(be, c, H, masks, **more)
    want, w, bound, wbound = S.attention(q, c, H, scale, masks)
    assert np.isfinite(out).all()
    off = np.abs(out - want).max(-1)
    assert (off <= bound + 1e-30).all(), (off.max(), bound[off.argmax()])
    norm = np.linalg.norm(want)
    # beside that bound, which every rounding at its worst would reach: roundings of either sign leave a few steps
    assert np.linalg.norm(out - want) <= 64 * S.EPS * norm + 1e-30
    for i, n in enumerate(c.lens):
        got, old = c.weights(i), c.w[i]
        exp = old.astype(np.float64)
        if weight:
            exp[:, :n] += w[i]
        assert np.abs(got - exp).max(initial=0.0) <= wbound[i] + 4 * S.EPS * (np.abs(exp).max(initial=0.0)) * (1 if weight else 0)
        assert (got[:, n:] == old[:, n:]).all()
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (14, 2, 64), (8, 8, 128), (32, 8, 128), (6, 2, 96), (3, 1, 32), (4, 2, 256), (33, 3, 160), (64, 2, 64)])
def test_one_token_of_each(be, dtype, H, G, D):
    c = S.Caches(be, [1, 2, 63, 64, 65, 300], [1] * 6, G, D, dtype=dtype, seed=H + D)
    check(be, c, H)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 192])
@pytest.mark.parametrize("toks", [[12], [1, 7, 33], [32, 5], [64, 0, 2], [100]])
@pytest.mark.parametrize("hidden", [False, True])
def test_trees(be, dtype, D, toks, hidden):
    r = np.random.default_rng(D + len(toks))
    lens = [t + int(r.integers(1, 500)) for t in toks]
    c = S.Caches(be, lens, toks, 2, D, dtype=dtype, hidden=hidden, weight=True, seed=D)
    check(be, c, 8, masks=[S.tree(t, r) for t in toks], weight=True)


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("odd", [0, 1, 2, 5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_chunk_and_slots_that_end_anywhere(be, D, odd, dtype):
    c = S.Caches(be, [17, 200, 129], [17, 40, 1], 2, D, dtype=dtype, odd=odd, weight=True, seed=odd)
    check(be, c, 4, weight=True)


@pytest.mark.parametrize("D", [64, 128, 32])
def test_rows_that_see_nothing(be, D):
    """a tree whose rows are empty, over a cache that holds the tree alone, and one whose past is hidden"""
    r = np.random.default_rng(3)
    masks = [S.tree(5, r), S.tree(4, r)]
    masks[0][2] = 0
    masks[0][:, 1] = 0      # and a slot that no token sees
    masks[1][:] = 0
    c = S.Caches(be, [5, 70], [5, 4], 2, D, hidden=True, weight=True, seed=1)
    c.hid[1][:66] = 1
    c.bufs[7].free()
    c.bufs[7] = be.upload(c.hid[1])
    c.table["hidden"][1] = c.bufs[7].ptr
    q, out = run(be, c, 4, masks)
    want, w, bound, _ = S.attention(q, c, 4, S.scale_of(D), masks)
    assert (out[2] == 0).all() and (out[5:] == 0).all()
    assert (np.abs(out - want).max(-1) <= bound).all()
    assert np.array_equal(c.weights(1), c.w[1])
    c.free()


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("magnitude", [1e-12, 1e-4, 1e4, 1e12])
def test_magnitudes(be, D, magnitude):
    """values far from one: the products keep their relative precision"""
    c = S.Caches(be, [150, 33], [3, 1], 2, D, seed=5, scale=magnitude, weight=True)
    check(be, c, 8, weight=True, q_scale=1.0 / magnitude)


@pytest.mark.parametrize("D", [64, 128])
def test_magnitudes_that_differ_from_slot_to_slot(be, D):
    c = S.Caches(be, [200], [6], 2, D, seed=6)
    f = np.exp2(np.random.default_rng(1).integers(-20, 4, 200)).astype(np.float32)
    c.k[0][:200] *= f[:, None]
    c.v[0][:, :200] *= f[::-1][None]
    kd, vd = be.upload(c.k[0]), be.upload(c.v[0])
    c.table["k"], c.table["v"] = kd.ptr, vd.ptr
    check(be, c, 8)
    kd.free()
    vd.free()


def test_large_scores(be):
    """scores of some hundreds: nearly one slot takes all"""
    c = S.Caches(be, [300], [12], 2, 128, seed=8, weight=True)
    check(be, c, 8, weight=True, q_scale=30.0)


@pytest.mark.parametrize("D,H,G", [(128, 8, 2), (64, 4, 4)])
def test_long_caches(be, D, H, G):
    c = S.Caches(be, [9001, 4096], [4, 1], G, D, seed=9, weight=True)
    check(be, c, H, weight=True)


@pytest.mark.parametrize("D,dtype", [(64, "f32"), (64, "bf16"), (128, "f32"), (128, "bf16")])
@pytest.mark.parametrize("lens,toks", [([1000, 130, 700], [1, 0, 2]), ([129, 64], [2, 1]), ([513, 511], [1, 1]), ([1023], [2]), ([1100], [1]), ([2100, 5], [1, 1]), ([1000] * 20, [1] * 20)])
def test_few_rows_whose_splits_are_a_cluster_or_joined(be, D, dtype, lens, toks):
    c = S.Caches(be, lens, toks, 2, D, dtype=dtype, hidden=True, weight=True, seed=sum(lens) + D)
    check(be, c, 8, weight=True, seed=D)


def test_more_sequences_than_a_table(be):
    lens = [1 + (i * 37) % 90 for i in range(150)]
    c = S.Caches(be, lens, [min(n, 1 + i % 3) if i % 11 else 0 for i, n in enumerate(lens)], 2, 64, seed=10, weight=True)
    check(be, c, 4, weight=True)


def test_the_most_tokens(be):
    c = S.Caches(be, [400], [capi.TREE_TOKENS], 1, 64, seed=11)
    check(be, c, 4)


def test_the_same_bits_again_and_beside_others(be):
    """a sequence's result does not hang on the call before it"""
    c = S.Caches(be, [700, 90], [12, 3], 2, 128, seed=12)
    _, a = run(be, c, 8)
    _, b = run(be, c, 8)
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    c.free()


def test_refusals(be):
    c = S.Caches(be, [20], [2], 2, 64, seed=1)
    x = be.empty(2 * 4 * 64)

    def bad(match, H=4, G=2, D=64, cache_type=0, out=x, **fields):
        t = c.table.copy()
        for k, v in fields.items():
            t[k] = v
        with pytest.raises(capi.PsCudaError, match=match):
            be.attn_tree(out, x, t, H, G, D, 1.0, cache_type=cache_type)

    bad("heads over", H=5)
    bad("heads over", H=66)
    bad("head size", D=48)
    bad("head size", D=288)
    bad("kv heads", G=0)
    bad("cache type", cache_type=8)
    bad("holds", n_kv=30)
    bad("holds", n_kv=-1)
    bad("brings", n_tok=21)
    bad("brings", n_tok=-1)
    bad("no rows", k=0)
    bad("aligned", k=int(c.table["k"][0]) + 2)
    bad("null argument", out=0)
    with pytest.raises(capi.PsCudaError):
        be.attn_tree(x, x, np.zeros(1, [("k", "u8")]), 4, 2, 64, 1.0)
    be.attn_tree(x, x, c.table[:0], 4, 2, 64, 1.0)      # nobody: nothing happens
    c.free()
    x.free()
