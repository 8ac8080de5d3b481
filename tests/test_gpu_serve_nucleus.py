"""ps_cuda_sample with top-p beside min-p and no top-k - rows that first look whether the rough mass of all tokens decides - on both cluster sizes (up to nine rows, and more),
where top-p cuts what min-p leaves, where it does not, at the border, and where the mass is no number."""
import numpy as np
import pytest

from tests import _serve as S
from tests.test_gpu_serve_sample import be, check  # noqa: F401

pytestmark = pytest.mark.gpu
NUCLEUS = [(1.0, 0, 0.9, 0.02), (0.7, 0, 0.95, 0.05), (1.0, 0, 0.2, 0.001), (1.5, 0, 0.999, 0.3), (1.0, 0, 0.5, 2.0 ** -16), (1.0, 0, 0.5, 1.5e-5), (3.0, 0, 0.6, 0.001), (0.3, 0, 0.99, 1.0), (1.0, 0, 0.0, 0.1)]


@pytest.mark.parametrize("V", [33, 5000, 128256, 151936])
@pytest.mark.parametrize("n", [1, 9, 10, 18])
def test_top_p_beside_min_p(be, V, n):  # noqa: F811
    r = np.random.default_rng(V + n)
    x = (r.standard_normal((n, V)) * 2.5).astype(np.float32)
    x[:, r.integers(0, V, 24)] += r.random(24).astype(np.float32) * 12
    for shift in range(0, len(NUCLEUS), 1 if n == 1 else 4):
        rows = [NUCLEUS[(i + shift) % len(NUCLEUS)] for i in range(n)]
        check(be, x, rows, r.random(n))


@pytest.mark.parametrize("n", [4, 12])
def test_top_p_next_to_what_min_p_leaves(be, n):  # noqa: F811
    """shares of top-p on either side of the mass that min-p leaves: the rough mass, known to a thousandth, decides the far ones alone"""
    V = 128256
    r = np.random.default_rng(n)
    x = (r.standard_normal((n, V)) * 2.0).astype(np.float32)
    w = np.exp((x - x.max(-1, keepdims=True)).astype(np.float64))
    share = (w * (w >= np.float32(0.01))).sum(-1) / w.sum(-1)
    for off in (-0.05, -1.5e-3, -5e-4, 5e-4, 1.5e-3, 0.05):
        rows = [(1.0, 0, float(s * (1 + off)), 0.01) for s in share]
        check(be, x, rows, np.linspace(0.0, 0.9999, n))


@pytest.mark.parametrize("n", [9, 12])
def test_odd_logits(be, n):  # noqa: F811
    V = 131072
    r = np.random.default_rng(2)
    x = (r.standard_normal((n, V)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1, ::2] = np.nan
    x[2, [7, 70, 40000]] = np.inf
    x[3, :V - 1] = -np.inf
    x[4] = np.where(r.random(V) < 0.99, -np.inf, x[4])
    x[5] = np.where(np.arange(V) % 3, np.finfo(np.float32).min, np.finfo(np.float32).max)
    x[6, ::V // 16] = np.inf
    x[7] = 1.0
    for f in NUCLEUS:
        check(be, x, [f] * n, r.random(n))


@pytest.mark.parametrize("n", [8, 12])
def test_a_temperature_without_end(be, n):  # noqa: F811
    """all tokens weigh the same, and those that are ruled out (-inf) nothing, though -inf times zero is no number: one of them in every sixteenth of a row, in one sixteenth
    another; and rows with any number of them"""
    V = 131072
    r = np.random.default_rng(3)
    x = r.standard_normal((n, V)).astype(np.float32)
    x[:, ::V // 16] = -np.inf
    x[:, 1] = -np.inf
    for i in range(2, n):
        x[i, r.random(V) < 0.1 * i / n] = -np.inf
    check(be, x, [(np.inf, 0, 0.9, 0.5)] * n, np.linspace(0.5, 0.9999, n))
