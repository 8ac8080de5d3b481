"""What the serving operators work in: it grows where the memory for half as much again is not there, what is outgrown goes back unless a captured graph holds it, and calls
that join nothing ask for nothing."""
import numpy as np
import pytest
import torch

from powerserve_b200 import capi
from tests import _serve as S
from tests.test_gpu_memory_yields import MB, Filler
from tests.test_gpu_serve_paths import backend

pytestmark = pytest.mark.gpu
H, G, D, TOK = 32, 8, 64, 32        # 128 rows of a kv head: scores of n slots are 4096 n bytes


class Steps:
    """calls over a cache of which any beginning is filled; all keys equal, so that every output is the values' mean"""

    def __init__(self, n_ctx):
        self.be, self.n_ctx = backend(), n_ctx
        self.k, self.v = torch.zeros(n_ctx, G * D, device="cuda"), torch.ones(G * D, n_ctx, device="cuda")
        self.w, self.q, self.out = torch.zeros(G, n_ctx, device="cuda"), torch.ones(TOK, H * D, device="cuda"), torch.zeros(TOK, H * D, device="cuda")
        self.mask = torch.ones(TOK, TOK, dtype=torch.uint8, device="cuda")
        self.graphs = []
        torch.cuda.synchronize()

    def call(self, n, tok=TOK, weight=True):
        t = np.zeros(1, capi.CACHE)
        t["k"], t["v"], t["n_ctx"], t["n_kv"], t["n_tok"] = self.k.data_ptr(), self.v.data_ptr(), self.n_ctx, n, tok
        t["weight"] = self.w.data_ptr() if weight else 0
        self.be.attn_tree(self.out, self.q, t, H, G, D, 1.0, tree_mask=self.mask)

    def check(self, n, calls):
        """after `calls` calls over n slots (on the host: the device may have no room)"""
        self.be.sync()
        torch.cuda.synchronize()
        assert np.abs(self.out.cpu().numpy() - 1).max() <= S.EPS * (n + 64)
        got = self.w.cpu().numpy()[:, :n].astype(np.float64) * n / (TOK * H // G * calls)
        assert np.abs(got - 1).max() <= S.EPS * (n + 64)
        self.w.zero_()
        self.out.zero_()

    def close(self):
        self.graphs.clear()
        torch.cuda.synchronize()
        self.be.close()


def free():
    """without what torch's allocator keeps"""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0]


def test_outgrown_memory_goes_back():
    s = Steps(24000)
    before = None
    for n in (4000, 6100, 9200, 13900, 20900):      # each more than half as much again: 16 to 86 MB, 212 together
        s.call(n)
        s.check(n, 1)
        if before is None:
            before = free() + 4096 * n
    assert before - free() <= 4096 * 20900 * 1.1 + 16 * MB
    s.close()


def test_room_for_the_new_where_the_old_one_goes():
    s = Steps(24000)
    s.call(16000)
    s.check(16000, 1)
    fill = Filler(100 * MB)         # about 50 MB are left; 79 are needed, 66 are held
    try:
        assert fill.free < 70 * MB
        s.call(19000)
        s.check(19000, 1)
    finally:
        fill.close()
    s.close()


def test_a_graph_s_memory_stays_and_the_new_is_no_more_than_must():
    s = Steps(24000)
    s.call(16000)
    s.check(16000, 1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        s.call(16000)
    s.graphs.append(g)
    fill = Filler(176 * MB)         # about 88 MB are left: enough for 79, not for half as much again as 66
    try:
        n = min(19000, (fill.free - 8 * MB) // 4096)
        assert n > 16500 and fill.free < 97 * MB
        s.call(n)
        s.check(n, 1)
        g.replay()
        s.check(16000, 1)
        s.call(n)
        g.replay()
        s.be.sync()
        torch.cuda.synchronize()
        assert np.abs(s.out.cpu().numpy() - 1).max() <= S.EPS * 16064
        with pytest.raises(capi.PsCudaError, match="cudaMalloc"):       # and no room at all is said
            s.call(24000, tok=TOK)
            s.call(24000, tok=TOK)
    finally:
        fill.close()
    del g
    s.close()


def test_a_call_that_joins_nothing_can_be_captured_first():
    s = Steps(4000)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        s.call(40, tok=2, weight=False)
    g.replay()
    s.be.sync()
    torch.cuda.synchronize()
    assert np.abs(s.out[:2].cpu().numpy() - 1).max() <= S.EPS * 128
    del g
    s.close()
