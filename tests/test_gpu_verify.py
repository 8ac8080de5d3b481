"""Verification of drafted tokens against the definition in 64 bits: paths and next tokens are equal; chains and trees, with the draft's rows and without, every kind of settings, rows that are odd; and the
distribution that comes out is the target's."""
import numpy as np
import pytest

from powerserve_b200 import capi
from tests import _paged as P
from tests import _serve as S
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu
KINDS = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 500, 0.8, 0.1), (1.5, 2000, 0.99, 0.001), (1.0, 1, 1.0, 0.0)]


def make(V, sizes, fan, seed, near=0.6, draft=True, kinds=KINDS):
    """(parents, tokens, u, logits, settings, draft logits, draft settings), all sequences after one another"""
    r = np.random.default_rng(seed)
    n = sum(sizes)
    logits = (r.standard_normal((n, V)) * 2.5).astype(np.float32)
    for row in logits:
        row[r.integers(0, V, 12)] += r.random(12).astype(np.float32) * 10
    guess = (logits + r.standard_normal((n, V)) * near).astype(np.float32)
    parents, tokens, t0 = np.zeros(n, np.int32), np.zeros(n, np.int32), 0
    sets = np.zeros(n, capi.SAMPLER)
    for s, m in enumerate(sizes):
        sets[t0:t0 + m] = tuple(kinds[s % len(kinds)])
        parents[t0] = -1
        for i in range(1, m):
            p = int(r.integers(max(0, i - fan), i))
            d = P.distribution(guess[t0 + p], *sets[t0 + p].tolist())
            parents[t0 + i] = p
            tokens[t0 + i] = r.choice(V, p=d) if r.random() < 0.9 else int(r.integers(0, V))
        t0 += m
    return parents, tokens, r.random(n).astype(np.float32), logits, sets, guess if draft else None, sets if draft else None


def run(be, V, sizes, parents, tokens, u, logits, sets, guess=None, guess_sets=None, pad=0):  # noqa: F811
    n, S_ = sum(sizes), len(sizes)
    wide = lambda x: np.concatenate([x, np.full((n, pad), 1e30, np.float32)], 1) if pad else x      # noqa: E731
    up = [be.upload(a) for a in (parents, tokens, wide(logits), sets, u)]
    g = [None, None] if guess is None else [be.upload(wide(guess)), be.upload(guess_sets)]
    ids, path, n_path = be.upload(np.full(S_ + 1, -9, np.int32)), be.upload(np.full(n + 1, -9, np.int32)), be.upload(np.full(S_ + 1, -9, np.int32))
    be.verify(ids, path, n_path, sizes, up[0], up[1], up[2], V, up[3], up[4], draft_logits=g[0], draft_samplers=g[1], row_stride=V + pad)
    got = ids.numpy(np.int32), path.numpy(np.int32), n_path.numpy(np.int32)
    for b in up + [x for x in g if x] + [ids, path, n_path]:
        b.free()
    assert got[0][-1] == got[1][-1] == got[2][-1] == -9
    return got[0][:-1], got[1][:-1], got[2][:-1]


def check(be, V, sizes, parents, tokens, u, logits, sets, guess=None, guess_sets=None, pad=0):  # noqa: F811
    ids, path, n_path = run(be, V, sizes, parents, tokens, u, logits, sets, guess, guess_sets, pad)
    t0 = 0
    for s, m in enumerate(sizes):
        e = slice(t0, t0 + m)
        want, token = P.verify(parents[e], tokens[e], u[e], logits[e], sets[e].tolist(), None if guess is None else guess[e], None if guess is None else guess_sets[e].tolist())
        assert path[e].tolist() == want + [-1] * (m - len(want)) and n_path[s] == len(want), s
        assert ids[s] == token, (s, ids[s], token)
        t0 += m
    return n_path


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [5, 100, 2049, 32000])
@pytest.mark.parametrize("fan", [1, 3])
def test_trees_of_all_sizes(be, draft, V, fan):  # noqa: F811
    for seed in range(3):
        check(be, V, [1, 2, 5, 12, 8, 3, 1, 20], *make(V, [1, 2, 5, 12, 8, 3, 1, 20], fan, 100 * V + seed, draft=draft))


@pytest.mark.parametrize("draft", [False, True])
def test_large_vocabulary(be, draft):  # noqa: F811
    a = make(151936, [5, 12], 2, 7, draft=draft)
    check(be, 151936, [5, 12], *a)
    check(be, 151936, [5, 12], *a, pad=3)


@pytest.mark.parametrize("draft", [False, True])
def test_many_sequences(be, draft):  # noqa: F811
    sizes = [1 + i % 3 for i in range(1100)]
    n = check(be, 300, sizes, *make(300, sizes, 2, 8, draft=draft))
    assert len(set(n.tolist())) == 3


def test_widest_tree(be):  # noqa: F811
    for fan in (1, 200):
        check(be, 500, [256, 256], *make(500, [256, 256], fan, fan, near=0.1))
        check(be, 500, [256, 256], *make(500, [256, 256], fan, fan, near=0.1, draft=False))


def test_a_draft_of_the_same_mind_is_always_right(be):  # noqa: F811
    parents, tokens, u, logits, sets, _, _ = make(4000, [9] * 8, 1, 9, near=0.0)
    for s in range(8):          # (drawn tokens only)
        for i in range(1, 9):
            d = P.distribution(logits[9 * s + i - 1], *sets[9 * s].tolist())
            tokens[9 * s + i] = np.random.default_rng(s * 10 + i).choice(4000, p=d)
    u[:] = np.float32(1) - np.float32(2.0 ** -24)
    n = check(be, 4000, [9] * 8, parents, tokens, u, logits, sets, logits, sets)
    assert (n == 9).all()


def test_the_same_sibling_twice_and_tokens_outside(be):  # noqa: F811
    """a token that was rejected has nothing left; one outside the vocabulary changes nothing"""
    for draft in (False, True):
        parents, tokens, u, logits, sets, g, gs = make(64, [8] * 40, 8, 10, draft=draft, kinds=[(1.0, 0, 1.0, 0.0)])
        parents.reshape(40, 8)[:, 1:] = 0
        tokens.reshape(40, 8)[:, 2] = tokens.reshape(40, 8)[:, 1]
        tokens.reshape(40, 8)[:, 3], tokens.reshape(40, 8)[:, 5], tokens.reshape(40, 8)[:, 6] = -1, 64, 2 ** 31 - 1
        u.reshape(40, 8)[:, 1:] = 0.9
        check(be, 64, [8] * 40, parents, tokens, u, logits, sets, g, gs)


def test_odd_rows(be):  # noqa: F811
    """no numbers, nothing but -inf, one infinite logit, all equal, one token that has all"""
    for draft in (False, True):
        parents, tokens, u, logits, sets, g, gs = make(200, [4] * 12, 2, 11, draft=draft, kinds=KINDS[:2] + KINDS[4:5])
        L = logits.reshape(12, 4, 200)
        L[0, :, ::3] = np.nan
        L[1] = -np.inf
        L[2, 1] = np.nan
        L[3, :, 17] = np.inf
        L[4] = 1.5
        L[5, :, :] = -1e30
        L[5, :, 40] = 50.0
        tokens.reshape(12, 4)[5, 1:] = 40
        tokens.reshape(12, 4)[3, 1:] = 17
        if draft:
            g.reshape(12, 4, 200)[6] = -np.inf
            g.reshape(12, 4, 200)[7, 0] = np.nan
            g.reshape(12, 4, 200)[8, :, 3] = np.inf
        check(be, 200, [4] * 12, parents, tokens, u, logits, sets, g, gs)


@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("V", [40, 3001])
def test_odd_rows_under_every_kind_of_settings(be, kind, V):  # noqa: F811
    """few rows, which clusters look at, and many, which a CTA each looks at first"""
    for sizes in ([3, 2], [4] * 24):
        for draft in (False, True):
            parents, tokens, u, logits, sets, g, gs = make(V, sizes, 2, 20 + kind, draft=draft, kinds=[KINDS[kind]])
            r = np.random.default_rng(kind)
            for x in (logits,) if g is None else (logits, g):
                x[r.integers(0, len(x), len(x) // 4), :] = 0.25                                  # all equal
                x[r.integers(0, len(x), len(x) // 4), int(r.integers(0, V))] = np.inf
                x[r.integers(0, len(x), len(x) // 8), :] = -np.inf
                x[r.integers(0, len(x), len(x) // 4), ::2] = np.nan
                x[r.integers(0, len(x), len(x) // 8), int(r.integers(0, V))] = 80.0
            check(be, V, sizes, parents, tokens, u, logits, sets, g, gs)


def test_rows_that_a_cta_cannot_decide(be):  # noqa: F811
    """many rows, flat ones: thousands of likely tokens; top_k above what is kept of them; a top-p whose border lies among the unlikely ones"""
    V, sizes = 20000, [3] * 30
    for draft in (False, True):
        parents, tokens, u, logits, sets, g, gs = make(V, sizes, 1, 31, draft=draft, kinds=[(1.0, 0, 0.9, 0.0), (1.0, 3000, 1.0, 0.0), (2.0, 600, 0.7, 0.0), (1.0, 0, 0.99999, 0.0), (0.05, 0, 0.999, 0.0), (1.0, 0, 0.95, 0.5)])
        for x in (logits,) if g is None else (logits, g):
            x[::2] *= 0.1
            x[1::7, 5] = 40.0
        check(be, V, sizes, parents, tokens, u, logits, sets, g, gs)


@pytest.mark.parametrize("u0", [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan])
def test_random_numbers_at_the_ends(be, u0):  # noqa: F811
    for draft in (False, True):
        parents, tokens, u, logits, sets, g, gs = make(3000, [3] * 8, 2, 12, draft=draft)
        u.reshape(8, 3)[:, 0] = u0
        args = parents, tokens, u, logits, sets, g, gs
        ids, path, n_path = run(be, 3000, [3] * 8, *args)
        for s in range(8):
            e, clamped = slice(3 * s, 3 * s + 3), u.copy()
            clamped[3 * s] = min(max(u0, 0.0), 1.0) if u0 == u0 else 0.0
            want, token = P.verify(parents[e], tokens[e], clamped[e], logits[e], sets[e].tolist(), None if g is None else g[e], None if g is None else gs[e].tolist())
            assert path[e].tolist()[:len(want)] == want and ids[s] == token


def test_tests_at_the_ends(be):  # noqa: F811
    """u = 0 accepts what the target may draw at all, u = 1 only what the draft does not hold for likelier"""
    for draft in (False, True):
        for u1 in (0.0, 1.0):
            parents, tokens, u, logits, sets, g, gs = make(500, [4] * 16, 2, 13, draft=draft)
            u.reshape(16, 4)[:, 1:] = u1
            check(be, 500, [4] * 16, parents, tokens, u, logits, sets, g, gs)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("fan", [1, 3])
def test_what_comes_out_is_the_targets_distribution(be, draft, fan):  # noqa: F811
    """the first token after the root over 60 000 trials of one tree, drafted tokens drawn anew: counts within six standard deviations of what the target's own draws would give.
    (Without the draft's rows the drafted tokens are fixed, and the law holds for those too.)"""
    V, N, m = 8, 60000, 3
    r = np.random.default_rng(14)
    logits, guess = [(r.standard_normal((m, V)) * 1.2).astype(np.float32) for _ in range(2)]
    sets = np.zeros(N * m, capi.SAMPLER)
    sets[:] = (1.0, 0, 1.0, 0.0)
    parents = np.tile(np.array([-1, 0, 0 if fan > 1 else 1], np.int32), N)
    q = P.distribution(guess[0], 1.0, 0, 1.0, 0.0)
    q1 = P.distribution(guess[1], 1.0, 0, 1.0, 0.0)
    tokens = np.zeros((N, m), np.int32)
    tokens[:, 1] = r.choice(V, N, p=q) if draft else 2
    tokens[:, 2] = (r.choice(V, N, p=q if fan > 1 else q1)) if draft else 5
    u = r.random((N, m)).astype(np.float32)
    every = lambda x: np.ascontiguousarray(np.broadcast_to(x, (N, m, V))).reshape(-1, V)    # noqa: E731
    got = np.zeros(V)
    ids, path, n_path = run(be, V, [m] * N, parents, tokens.reshape(-1), u.reshape(-1), every(logits), sets, every(guess) if draft else None, sets if draft else None)
    first = np.where(n_path > 1, tokens[np.arange(N), path.reshape(N, m)[:, 1].clip(0)], ids)
    got = np.bincount(first, minlength=V)
    p = P.distribution(logits[0], 1.0, 0, 1.0, 0.0)
    assert (np.abs(got - N * p) <= 6 * np.sqrt(N * p * (1 - p))).all(), (got / N, p)


def test_sampling_is_what_it_was(be):  # noqa: F811
    """a sequence of one node is a row of ps_cuda_sample"""
    r = np.random.default_rng(15)
    V, n = 32000, 40
    logits = (r.standard_normal((n, V)) * 3).astype(np.float32)
    sets = S.settings([KINDS[i % len(KINDS)] for i in range(n)])
    u = r.random(n).astype(np.float32)
    ids, path, n_path = run(be, V, [1] * n, np.full(n, -1, np.int32), np.zeros(n, np.int32), u, logits, sets)
    up = [be.upload(a) for a in (logits, sets, u)]
    want = be.upload(np.zeros(n, np.int32))
    be.sample(want, None, up[0], V, n, up[1], up[2])
    assert np.array_equal(want.numpy(np.int32), ids) and (n_path == 1).all() and (path == 0).all()
    for b in up + [want]:
        b.free()


def test_a_row_alone_and_among_many(be):  # noqa: F811
    """Rows of nearly equal logits that fall with the token's number, and a random number that asks for the last token of what top-p leaves: the border is the same one whatever the call's other rows are"""
    V, n = 100001, 48
    r = np.random.default_rng(32)
    logits = -np.sort((r.random((n, V)) * 0.2).astype(np.float32), axis=1)
    kinds = [(1.0, 0, 0.7, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 0, 0.6, 2.0 ** -10), (1.3, 60000, 0.9, 0.0), (1.1, 0, 0.35, 0.0)]
    sets = S.settings([kinds[i % len(kinds)] for i in range(n)])
    u = np.full(n, 1.0 - 2.0 ** -24, np.float32)
    minus, zero = np.full(n, -1, np.int32), np.zeros(n, np.int32)
    ids = run(be, V, [1] * n, minus, zero, u, logits, sets)[0]
    assert len(set(ids.tolist())) > n // 2
    for size in (1, 8, 20):
        for i in range(0, n - size + 1, size):
            e = slice(i, i + size)
            assert np.array_equal(run(be, V, [1] * size, minus[e], zero[e], u[e], logits[e], sets[e])[0], ids[e]), (size, i)


@pytest.mark.parametrize("n", [1, 30, 700])
def test_clusters_meet_soon_after_they_begin(be, n):  # noqa: F811
    """sequences of their last tokens alone: nothing lies between a cluster's beginning and its first exchange but a row's record.  In few clusters, and in more than run at a time"""
    r = np.random.default_rng(40 + n)
    V = 3000
    logits = (r.standard_normal((n, V)) * 3).astype(np.float32)
    sets = S.settings([KINDS[i % len(KINDS)] for i in range(n)])
    args = np.full(n, -1, np.int32), np.zeros(n, np.int32), r.random(n).astype(np.float32), logits, sets
    for _ in range(3):
        check(be, V, [1] * n, *args)


@pytest.mark.parametrize("sizes", [[2] * 10, [2] * 24, [5] * 4, [5] * 12, [1] * 48])
@pytest.mark.parametrize("min_p", [1e-5, 1e-7])
@pytest.mark.parametrize("draft", [False, True])
def test_a_min_p_below_what_is_listed(be, sizes, min_p, draft):  # noqa: F811
    """One likely token and tens of thousands whose weights lie between min-p and 2^-16, which together hold about as much, and as many below min-p: few rows and many"""
    V, n = 80000, sum(sizes)
    r = np.random.default_rng([41, n, draft])

    def rows():
        least = np.log(min_p * 1.01)
        x = r.uniform(max(least, np.log(1.15e-5)), np.log(1.5e-5), (n, V))
        x[:, 1::2] = r.uniform(least, np.log(1.5e-5), (n, V // 2))
        x[:, ::5] = np.log(min_p) - r.uniform(0.01, 8.0, x[:, ::5].shape)
        x[:, 77] = 0.0
        return (x + r.uniform(-3, 3, (n, 1))).astype(np.float32)
    logits, guess = rows(), rows() if draft else None
    sets = S.settings([(1.0, 0, 1.0, min_p)] * n)
    u = r.random(n).astype(np.float32)
    parents, tokens = np.concatenate([np.arange(m) - 1 for m in sizes]).astype(np.int32), np.full(n, 77, np.int32)
    if draft:                               # (drafted tokens of p < q and of p > q)
        guess[::3, 77] -= 0.7
        tokens[::4] = r.integers(0, V // 2, len(tokens[::4])) * 2 + 1
    n_path = check(be, V, sizes, parents, tokens, u, logits, sets, guess, sets if draft else None)
    assert draft or sizes[0] == 1 or len(set(n_path.tolist())) > 1     # (the likely token's own share decides)


@pytest.mark.parametrize("sizes", [[2] * 15, [2] * 40])
@pytest.mark.parametrize("draft", [False, True])
def test_random_numbers_beside_the_border(be, sizes, draft):  # noqa: F811
    """Rows without filters: one likely token, and a tail of equal ones that together hold from a hundredth to nine tenths; the likely one's test is 2^-22 of p(c) / q(c) above it or below.  (Masses are sums of whole numbers
    of 2^-44, each off by half a one at most: 128 255 of them by 2^-28 of the mass; a random number of float32 by 2^-24.)"""
    V, n = 128256, sum(sizes)
    r = np.random.default_rng([42, n, draft])

    def rows():
        x = np.repeat(r.uniform(-12.5, -9.5, (n, 1)).astype(np.float32), V, 1)
        x[:, 1001] = 0.0
        return x + r.uniform(-2, 2, (n, 1)).astype(np.float32)
    logits, guess = rows(), rows() if draft else None
    sets = S.settings([(float(np.float32(t)), 0, 1.0, 0.0) for t in r.uniform(0.95, 1.1, n)])
    parents, tokens, u = np.tile(np.array([-1, 0], np.int32), len(sizes)), np.full(n, 1001, np.int32), r.random(n).astype(np.float32)
    side = np.where(np.arange(len(sizes)) % 2, 1, -1)
    for s in range(len(sizes)):
        p = P.distribution(logits[2 * s], *sets[2 * s].tolist())[1001]
        q = P.distribution(guess[2 * s], *sets[2 * s].tolist())[1001] if draft else 1.0
        u[2 * s + 1] = p / q * (1 + side[s] * 2.0 ** -22)
    n_path = check(be, V, sizes, parents, tokens, u, logits, sets, guess, sets if draft else None)
    assert (n_path[side < 0] == 2).all() and ((n_path[side > 0] == 1) | (u[1::2][side > 0] > 1)).all()


def test_the_same_border_as_samplings(be):  # noqa: F811
    """top-p over one likely token and a tail of equal ones: the last token that is left is the one that ps_cuda_sample draws, in few rows and in many"""
    V, n = 128256, 240
    r = np.random.default_rng(43)
    logits = np.repeat(r.uniform(-11.5, -9.0, (n, 1)).astype(np.float32), V, 1)
    logits[:, 7] = 0.0
    sets = S.settings([(1.0, 0, float(p), 0.0) for p in r.uniform(0.6, 0.99, n)])
    sets["min_p"][::3] = 2.0 ** -18
    sets["min_p"][1::9] = 2.0 ** -17
    u, minus, zero = np.full(n, 1.0 - 2.0 ** -24, np.float32), np.full(n, -1, np.int32), np.zeros(n, np.int32)
    up = [be.upload(a) for a in (logits, sets, u)]
    want = be.upload(np.zeros(n, np.int32))
    be.sample(want, None, up[0], V, n, up[1], up[2])
    ids = want.numpy(np.int32)
    assert len(set(ids.tolist())) > n // 2
    assert np.array_equal(run(be, V, [1] * n, minus, zero, u, logits, sets)[0], ids)
    for i in range(0, n, 20):
        e = slice(i, i + 20)
        assert np.array_equal(run(be, V, [1] * 20, minus[e], zero[e], u[e], logits[e], sets[e])[0], ids[e]), i
    for b in up + [want]:
        b.free()


@pytest.mark.parametrize("V,k", [(60, 3), (60, 50), (5000, 40), (5000, 600), (30000, 3000)])
@pytest.mark.parametrize("sizes", [[2] * 6, [2] * 50])
@pytest.mark.parametrize("draft", [False, True])
def test_a_top_k_whose_border_weighs_nothing(be, V, k, sizes, draft):  # noqa: F811
    """Peaked rows, in which all tokens but one lie below 2^-46 of it, those around the border of top-k too: at u = 0, or where the draft holds them for less likely still, the ones inside are accepted and no other one"""
    n, r = sum(sizes), np.random.default_rng([44, V, k])
    logits = (np.stack([r.permutation(V) for _ in range(n)]) * (-10.0 / V) - 40).astype(np.float32)
    best = r.integers(0, V, n)
    logits[np.arange(n), best] = 0.0
    order = np.argsort(-logits, 1, kind="stable")
    guess = None
    if draft:
        guess = np.full((n, V), -60, np.float32)
        guess[np.arange(n), (best + 1) % V] = 0.0
    sets = S.settings([(1.0, k, 1.0, 0.0)] * n)
    parents, tokens, u = np.tile(np.array([-1, 0], np.int32), len(sizes)), np.zeros(n, np.int32), r.random(n).astype(np.float32)
    rank = np.resize([1, k - 1, k, k + 1, V - 1], n // 2)
    tokens[1::2] = order[::2][np.arange(n // 2), rank]
    u[1::2][::2] = 0
    n_path = check(be, V, sizes, parents, tokens, u, logits, sets, guess, S.settings([(1.0, 0, 1.0, 0.0)] * n) if draft else None)
    assert (n_path[rank >= k] == 1).all() and (n_path == 2).any()
