"""The serving operators between a caller's own torch operations, with no synchronisation of its own: inputs that the caller's stream has yet to write, results that
it reads and inputs that it overwrites next, on the default stream and on another one, and captured from the caller's stream."""
import contextlib

import numpy as np
import pytest
import torch

from powerserve_b200 import capi
from tests import _serve as S
from tests.test_gpu_serve_paths import backend

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["default", "own"])
def stream(request):
    if request.param == "default":
        yield contextlib.nullcontext
    else:
        s = torch.cuda.Stream()
        yield lambda: torch.cuda.stream(s)
        s.synchronize()


def busy():
    """some tens of milliseconds of work on the current stream"""
    a = torch.ones(4096, 4096, device="cuda")
    for _ in range(40):
        a = (a @ a) * 1e-4
    return a


def test_attention(stream):
    be = backend()
    H, G, D = 8, 2, 64
    for lens, toks in (([300, 70], [1, 1]), ([900, 200], [20, 7])):
        c = S.Caches(be, lens, toks, G, D, seed=5)
        n = sum(toks)
        src = np.random.default_rng(n).standard_normal((n, H * D)).astype(np.float32)
        want, _, bound, _ = S.attention(src, c, H, S.scale_of(D))
        with stream():
            q, out, later = torch.zeros(n, H * D, device="cuda"), torch.zeros(n, H * D, device="cuda"), torch.from_numpy(src).cuda()
            busy()
            q.copy_(later)
            be.attn_tree(out, q, c.table, H, G, D, S.scale_of(D))
            q.fill_(3.0)
            got = (out * 2).cpu().numpy()
        assert (np.abs(got / 2 - want).max(-1) <= bound).all()
        c.free()
    be.close()


def test_eviction(stream):
    """arrays that only the records name"""
    be = backend()
    G, D, n, n_ctx, keep = 2, 64, 500, 512, 120
    r = np.random.default_rng(1)
    k0, v0, w0 = r.standard_normal((n_ctx, G * D)).astype(np.float32), r.standard_normal((G * D, n_ctx)).astype(np.float32), r.random((G, n_ctx)).astype(np.float32)
    with stream():
        k, v, w = (torch.zeros(a.shape, device="cuda") for a in (k0, v0, w0))
        later = [torch.from_numpy(a).cuda() for a in (k0, v0, w0)]
        t = np.zeros(1, capi.CACHE)
        t[0] = (k.data_ptr(), v.data_ptr(), w.data_ptr(), w.data_ptr(), 0, 0, 0, n_ctx, n, 0, keep)
        busy()
        for a, b in zip((k, v, w), later):
            a.copy_(b)
        be.kv_evict(t, G, D)
        got = [a.clone() for a in (k, v, w)]
        for a in (k, v, w):
            a.zero_()
        got = [a.cpu().numpy() for a in got]
    for g in range(G):
        src, dst = S.evict(w0[g], None, n, keep, 0, 0)
        at = slice(g * D, (g + 1) * D)
        k0[dst, at], v0[at, dst], w0[g, dst] = k0[src, at], v0[at, src], w0[g, src]
    for a, b in zip(got, (k0, v0, w0)):
        assert np.array_equal(a, b)
    be.close()


def test_sampling(stream):
    be = backend()
    V, rows = 30000, [(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05)]
    r = np.random.default_rng(2)
    x, u = (r.standard_normal((4, V)) * 3).astype(np.float32), r.random(4).astype(np.float32)
    want = [S.sample(x[i], *(float(np.float32(f)) if isinstance(f, float) else f for f in rows[i]), float(u[i]))[0] for i in range(4)]
    with stream():
        logits, later, ud = torch.zeros(4, V, device="cuda"), torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
        sd = torch.from_numpy(S.settings(rows).view(np.float32).reshape(4, 4).copy()).cuda()
        ids = torch.full((4,), -1, dtype=torch.int32, device="cuda")
        busy()
        logits.copy_(later)
        be.sample(ids, None, logits, V, 4, sd, ud)
        next_ids = ids.long() + 0
        logits.zero_()
        assert next_ids.cpu().tolist() == want
    be.close()


@pytest.mark.parametrize("mode", ["global", "thread_local"])
def test_captured_from_the_caller_s_stream(mode):
    """the calls become part of the caller's graph, in order with what it captures before and after them"""
    be = backend()
    H, G, D, V = 8, 2, 64, 20000
    c = S.Caches(be, [900, 200], [20, 7], G, D, seed=6)
    r = np.random.default_rng(3)
    rows = [(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0)]
    q, x, u = torch.zeros(27, H * D, device="cuda"), torch.zeros(2, V, device="cuda"), torch.rand(2, device="cuda")
    out, ids = torch.zeros_like(q), torch.zeros(2, dtype=torch.int32, device="cuda")
    sd = torch.from_numpy(S.settings(rows).view(np.float32).reshape(2, 4).copy()).cuda()

    def step():
        y = q * 2.0
        be.attn_tree(out, y, c.table, H, G, D, S.scale_of(D))
        z = x * 3.0
        be.sample(ids, None, z, V, 2, sd, u)
        return out + 1.0, ids + 5

    step()      # (the workspace is asked for)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode=mode):
        got_o, got_i = step()
    for k in range(3):
        qn, xn = r.standard_normal((27, H * D)).astype(np.float32), r.standard_normal((2, V)).astype(np.float32)
        q.copy_(torch.from_numpy(qn))
        x.copy_(torch.from_numpy(xn))
        g.replay()
        o, i = got_o.cpu().numpy(), got_i.cpu().tolist()
        want, _, bound, _ = S.attention(qn * np.float32(2), c, H, S.scale_of(D))
        assert (np.abs(o - 1 - want).max(-1) <= bound + 2 * S.EPS * (np.abs(want).max(-1) + 1)).all()
        xs, un = xn * np.float32(3), u.cpu().numpy()
        assert i == [5 + S.sample(xs[j], *(float(np.float32(f)) if isinstance(f, float) else f for f in rows[j]), float(un[j]))[0] for j in range(2)]
    be.attn_tree(out, q, c.table, H, G, D, S.scale_of(D))       # and eager calls go on
    want, _, bound, _ = S.attention(qn, c, H, S.scale_of(D))
    assert (np.abs(out.cpu().numpy() - want).max(-1) <= bound).all()
    del g
    torch.cuda.synchronize()
    c.free()
    be.close()


def test_a_call_that_is_refused_in_a_capture_leaves_the_capture_whole():
    be = backend()
    c = S.Caches(be, [900, 200], [20, 7], 2, 64, seed=6)
    q = torch.zeros(27, 8 * 64, device="cuda")
    out, one = torch.zeros_like(q), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        a = one + 1.0
        with pytest.raises(capi.PsCudaError, match="workspace"):
            be.attn_tree(out, q, c.table, 8, 2, 64, 0.125)
        b = a + 1.0
    g.replay()
    assert b.cpu().tolist() == [2.0] * 4
    del g
    torch.cuda.synchronize()
    c.free()
    be.close()
