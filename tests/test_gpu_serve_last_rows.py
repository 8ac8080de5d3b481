"""The rows that the last pass left: ps_cuda_sample_last and ps_cuda_sample_topk after every kind of pass - trees, chunks, sessions, the greedy loop, passes
without logits - on both model families.  A row that the last pass did not leave is refused."""
import numpy as np
import pytest

from powerserve_b200 import arch, arch_synth, capi
from tests import _serve as S
from tests.test_gpu_serve_paths import model

pytestmark = pytest.mark.gpu
V = 5000
ROWS = [(1.0, 0, 0.9, 0.0), (0.7, 50, 0.95, 0.01), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.1), (1.0, 0, 1.0, 0.0)]


def drawn(m, logits, seed=0):
    """the rows' tokens, as the plain form draws them from `logits`"""
    n = len(logits)
    u = np.random.default_rng(seed).random(n).astype(np.float32)
    rows = [ROWS[i % len(ROWS)] for i in range(n)]
    ids, probs = m.sample(rows, u)
    for i in range(n):
        t, p = S.sample(logits[i], *(float(np.float32(f)) if isinstance(f, float) else f for f in rows[i]), float(u[i]))
        assert ids[i] == t and abs(probs[i] - p) <= 4 * S.EPS * p + 1e-12


def refused(m, n):
    with pytest.raises(capi.PsCudaError, match="rows"):
        m.sample(ROWS[0], np.full(n, 0.5, np.float32))
    with pytest.raises(capi.PsCudaError, match="row"):
        m.sample_topk(3, row=n - 1)


def tree(m, n, seed=0, **how):
    r = np.random.default_rng(seed)
    mask = S.tree(n, r)
    depth = [int(mask[i].sum()) - 1 for i in range(n)]
    return m.forward_tree(r.integers(0, V, n), np.array([m.position + d for d in depth], np.int32), mask, **how)


def test_a_tree_s_rows_after_a_prefill():
    m = model(V, 16)
    m.prefill(list(range(1, 40)), 16)       # (no logits)
    logits = tree(m, 12)
    drawn(m, logits)
    for row in (0, 11):
        vals, ids = m.sample_topk(5, row=row)
        assert list(ids) == list(np.argsort(-logits[row].astype(np.float64), kind="stable")[:5]) and np.array_equal(vals, logits[row][ids])
    drawn(m, logits[:5], seed=1)            # fewer rows than there are
    refused(m, 13)
    m.close()


def test_a_wider_pass_before_a_narrower_one():
    """what the earlier pass left behind the later one's rows are old logits"""
    m = model(V, 16)
    m.forward_lazy([1, 2, 3, 4, 5, 6, 7, 8])
    logits = tree(m, 3)
    refused(m, 4)
    refused(m, 8)
    drawn(m, logits)
    m.forward_lazy(list(range(9, 21)))
    drawn(m, m.be.read_device(m.be.logits_dev(), 12 * V).reshape(12, V))
    drawn(m, m.forward([3]))
    refused(m, 2)
    m.close()


def test_the_greedy_loop_leaves_one_row():
    m = model(V, 16)
    m.prefill([1, 2, 3, 4], 8)
    m.forward_lazy([5, 6, 7, 8])
    ids = m.decode_greedy(9, 6)
    refused(m, 2)
    assert m.sample((0.0, 0, 1.0, 0.0), [0.5])[0][0] == ids[-1] == m.sample_topk(1)[1][0]
    drawn(m, m.be.read_device(m.be.logits_dev(), V).reshape(1, V))
    m.close()


def test_passes_without_logits_leave_none():
    m = model(V, 16)
    refused(m, 1)                           # no pass at all
    m.forward_lazy([1, 2, 3])
    m.forward([4, 5], lm_head=False)
    refused(m, 1)
    m.forward_lazy([6])
    tree(m, 3, lm_head=False)
    refused(m, 1)
    sids = [m.session_create() for _ in range(2)]
    want, _ = m.forward_sessions(sids, [7, 8])
    drawn(m, want)
    refused(m, 3)
    m.forward_sessions(sids, [7, 8], lm_head=False)
    refused(m, 1)
    m.forward_lazy([7])
    with pytest.raises(capi.PsCudaError):   # a pass that is refused leaves what was there
        m.forward([V + 1])
    drawn(m, m.be.read_device(m.be.logits_dev(), V).reshape(1, V))
    m.close()


def test_a_tree_s_rows_that_stay_on_the_device():
    """a tree verified by draws: ids and probabilities come back, no logits"""
    m = model(V, 16)
    m.prefill(list(range(1, 40)), 16)
    want = tree(m, 12, seed=5)
    m.be.kv_rollback(12)
    before = m.be.counter("d2h_bytes")
    assert tree(m, 12, seed=5, want_logits=False) is None
    drawn(m, want)
    assert m.be.counter("d2h_bytes") - before == 12 * 8
    refused(m, 13)
    with pytest.raises(capi.PsCudaError, match="greedy ids"):
        tree(m, 2, lm_head=2, want_logits=False)
    drawn(m, want)          # (it was refused before anything ran)
    m.close()


def test_a_layer_list_model(tmp_path):
    layer = arch_synth.nufusun_layer
    cfg = arch_synth.nufusun_config(64, 500, [layer(2, 1, 16, 16, bias_max=9.0)], eps=1e-5, embed_scale=0.5)
    arch_synth.write_model_dir(str(tmp_path), cfg, arch_synth.nufusun_weights(cfg, seed=3, rel_rows=8))
    m = arch.load_model(str(tmp_path), dtype="float32", max_batch=8, n_ctx=64)
    refused(m, 1)
    logits = m.forward([1, 2, 3, 4, 5])
    drawn(m, logits)
    refused(m, 6)
    m.prefill([6, 7, 8], 8)
    refused(m, 1)
    m.forward_lazy([9, 10])
    ids = m.decode_greedy(11, 5)
    refused(m, 2)
    assert m.sample((0.0, 0, 1.0, 0.0), [0.5])[0][0] == ids[-1]
    m.close()
