"""The serving operators as they are used: after one another on a model's own cache and logits, behind the command line, captured into a graph, from
several threads and contexts at once, and on caches whose offsets pass 32 bits."""
import json
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from powerserve_b200 import capi, gguf, synth
from tests import _model as M
from tests import _serve as S

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def backend(max_batch=1):
    return capi.CudaBackend(capi.ModelDesc(512, 1536, 1, 8, 2, 64, 1024, 64, 1e-5, 64, 0, 5e5, 1.0, 1.0, 0, max_batch, 0, 1))


def model(vocab=5000, max_batch=8):
    shape = synth.ModelShape("serve", "llama", 256, 256, 2, 4, 2, 64, vocab, True, 0, 1e4, 1e-5, gguf.GGML_Q8_0, n_ctx=256)
    tensors = {n: gguf.GGUFTensor(n, t, tuple(s), np.ascontiguousarray(d).view(np.uint8).reshape(-1)) for n, t, s, d in synth.generate_tensors(shape, 1)}
    return capi.CudaModel(desc=capi.desc_from_model_json(synth.model_json(shape), max_batch=max_batch, n_ctx=256), tensors=tensors)


def test_samples_of_a_pass_and_of_sessions():
    m = model()
    r = np.random.default_rng(1)
    rows = [(1.0, 0, 0.9, 0.0), (0.7, 50, 0.95, 0.01), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.1), (1.0, 0, 1.0, 0.0)]
    m.forward_lazy([1, 2, 3, 4, 5])
    logits = m.be.read_device(m.be.logits_dev(), 5 * 5000).reshape(5, 5000)
    u = r.random(5).astype(np.float32)
    ids, probs = m.sample(rows, u)
    for i, row in enumerate(rows):
        t, p = S.sample(logits[i], *row, float(u[i]))
        assert ids[i] == t and abs(probs[i] - p) <= 4 * S.EPS * p
    one = m.sample(rows[0], u[:2])      # one setting for all, fewer rows
    assert one[0][0] == ids[0]
    with pytest.raises(capi.PsCudaError, match="rows"):
        m.sample(rows[0], r.random(6))
    # a server's step: sessions of their own lengths, their next tokens drawn in one call
    sids = [m.session_create() for _ in range(3)]
    for k, sid in enumerate(sids):
        m.session_select(sid)
        m.prefill(list(range(1, 5 + 3 * k)), 8)
    m.session_select(0)
    want, _ = m.forward_sessions(sids, [7, 8, 9])
    for sid in sids:
        m.session_select(sid)
        m.be.kv_rollback(1)
    m.session_select(0)
    m.forward_sessions(sids, [7, 8, 9], want_logits=False)
    got, _ = m.sample(rows[:3], u[:3])
    assert [S.sample(want[i], *rows[i], float(u[i]))[0] for i in range(3)] == list(got)
    m.close()


def test_command_line(tmp_path):
    d = M.model_dir("tiny-llama")
    exe = os.path.join(ROOT, "bin", "ps_generate")

    def run(*args):
        r = subprocess.run([sys.executable, exe, "--model", d, "--ids", "5 17 3", "--n", "12", *args], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.strip().splitlines()[-1])["ids"]

    greedy = run()
    assert run("--top-k", "0", "--top-p", "0") == greedy            # only the likeliest is left
    assert run("--top-k", "200", "--min-p", "1") == greedy
    drawn = run("--top-p", "0.95", "--min-p", "0.01", "--temperature", "1.5", "--seed", "3")
    assert drawn == run("--top-k", "0", "--top-p", "0.95", "--min-p", "0.01", "--temperature", "1.5", "--seed", "3")
    m = capi.CudaModel(d, max_batch=8)
    m.reset()
    m.prefill([5, 17, 3])
    rng, tok = np.random.default_rng(3), 3
    for want in drawn:
        logits = m.forward([tok])[0]
        tok = S.sample(logits, 1.5, 0, float(np.float32(0.95)), float(np.float32(0.01)), float(np.float32(rng.random(1)[0])))[0]
        assert tok == want
    m.close()


def test_a_drafted_step_on_the_model_s_own_cache():
    """prefill, a drafted tree's attention over the layer's cache, the cache cut by the gathered weights, a token's attention over what stayed"""
    m = model(vocab=512)
    m.prefill(list(np.random.default_rng(2).integers(0, 512, 121)), 8)
    n, H, G, D, n_ctx = m.position, 4, 2, 64, 256
    assert n == 120
    be, r = m.be, np.random.default_rng(3)
    for layer in range(2):
        k = be.read_device(be.kv_k(layer), n_ctx * G * D).reshape(n_ctx, G * D)
        v = be.read_device(be.kv_v(layer), n_ctx * G * D).reshape(G * D, n_ctx)

        class Own:
            pass

        c = Own()
        c.lens, c.toks, c.G, c.D, c.k, c.v, c.hid = [n], [6], G, D, [k], [v], [np.zeros(n_ctx, np.uint8)]
        mask = [S.tree(6, r)]
        q = r.standard_normal((6, H * D)).astype(np.float32)
        want, w, bound, wbound = S.attention(q, c, H, S.scale_of(D), mask)
        zero, pos = np.zeros((G, n_ctx), np.float32), np.broadcast_to(np.arange(n_ctx, dtype=np.int32), (G, n_ctx)).copy()
        qd, od, wd, pd, md = be.upload(q), be.empty(q.size), be.upload(zero), be.upload(pos), be.upload(mask[0])
        t = np.zeros(1, capi.CACHE)
        t[0] = (be.kv_k(layer), be.kv_v(layer), wd.ptr, wd.ptr, pd.ptr, pd.ptr, 0, n_ctx, n, 6, 50)
        be.attn_tree(od, qd, t, H, G, D, S.scale_of(D), tree_mask=md)
        assert (np.abs(od.numpy(np.float32, q.shape) - want).max(-1) <= bound).all()
        got_w = wd.numpy(np.float32, (G, n_ctx))
        assert np.abs(got_w[:, :n] - w[0]).max() <= wbound[0]
        be.kv_evict(t, G, D, n_sink=2, n_recent=8)
        for g in range(G):
            src, dst = S.evict(got_w[g], pos[g], n, 50, 2, 8)
            at = slice(g * D, (g + 1) * D)
            k[dst, at], v[at, dst], pos[g, dst] = k[src, at], v[at, src], pos[g, src]
            assert {0, 1} | set(range(n - 8, n)) <= set(pos[g, :50].tolist())
        assert np.array_equal(be.read_device(be.kv_k(layer), n_ctx * G * D).reshape(n_ctx, G * D), k)
        assert np.array_equal(be.read_device(be.kv_v(layer), n_ctx * G * D).reshape(G * D, n_ctx), v)
        assert np.array_equal(pd.numpy(np.int32, pos.shape), pos)
        t["n_kv"], t["n_tok"], c.lens, c.toks = 50, 1, [50], [1]
        be.attn_tree(od, qd, t, H, G, D, S.scale_of(D))
        want, _, bound, _ = S.attention(q[:1], c, H, S.scale_of(D))
        assert (np.abs(od.numpy(np.float32, q.shape)[:1] - want).max(-1) <= bound).all()
        for b in (qd, od, wd, pd, md):
            b.free()
    m.close()


def test_captured_and_replayed():
    import torch
    be = backend()
    c = S.Caches(be, [300, 70, 1000], [1, 1, 1], 2, 64, seed=5, weight=True)
    t = S.Caches(be, [900, 200], [20, 7], 2, 128, seed=6, weight=True)
    r = np.random.default_rng(7)
    masks = [S.tree(20, r), S.tree(7, r)]
    qc, qt = r.standard_normal((3, 4 * 64)).astype(np.float32), r.standard_normal((27, 8 * 128)).astype(np.float32)
    x, u, settings = (r.standard_normal((4, 20000)) * 3).astype(np.float32), r.random(4).astype(np.float32), S.settings([(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05)])
    qcd, qtd, xd, ud, sd, md = (be.upload(a) for a in (qc, qt, x, u, settings, np.concatenate([m.reshape(-1) for m in masks])))
    oc, ot, ids, probs = be.empty(qc.size), be.empty(qt.size), be.upload(np.zeros(4, np.int32)), be.empty(4)

    def calls():
        be.attn_tree(oc, qcd, c.table, 4, 2, 64, 0.125)
        be.attn_tree(ot, qtd, t.table, 8, 2, 128, 0.09, tree_mask=md)
        be.sample(ids, probs, xd, 20000, 4, sd, ud)

    def results():
        return [oc.numpy(np.uint32), ot.numpy(np.uint32), ids.numpy(np.int32), probs.numpy(np.uint32)]

    stream = torch.cuda.ExternalStream(be.L.ps_cuda_stream(be.h))
    g = torch.cuda.CUDAGraph()
    with pytest.raises(capi.PsCudaError, match="workspace"):    # (the first call would have to ask for memory)
        with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
            be.attn_tree(ot, qtd, t.table, 8, 2, 128, 0.09, tree_mask=md)
    calls()
    want = results()
    w0 = c.weights(0).copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream, capture_error_mode="thread_local"):
        calls()
    for _ in range(3):
        for b, n in ((oc, qc.size), (ot, qt.size), (ids, 4), (probs, 4)):
            be._ck(be.L.ps_cuda_memcpy_h2d(be.h, b.ptr, np.zeros(n, np.float32).ctypes.data, 4 * n))
        with torch.cuda.stream(stream):
            g.replay()
        for a, b in zip(results(), want):
            assert np.array_equal(a, b)
    assert np.allclose(c.weights(0) - w0, 3 * (w0 - c.w[0]), atol=1e-5)      # every replay has gathered once more
    # a larger call in between takes other memory; the graph's stays its own
    big = S.Caches(be, [6000], [30], 2, 128, seed=8, weight=True)
    qb = be.upload(r.standard_normal((30, 8 * 128)).astype(np.float32))
    ob = be.empty(30 * 8 * 128)
    be.attn_tree(ob, qb, big.table, 8, 2, 128, 0.09)
    with torch.cuda.stream(stream):
        g.replay()
    for a, b in zip(results(), want):
        assert np.array_equal(a, b)
    del g
    be.sync()
    be.close()


def test_threads_and_contexts_at_once():
    """two contexts, each in a thread of its own: every call's result is what it is alone"""
    import torch
    torch.zeros(1, device="cuda")
    bes, bad = [backend(), backend()], []
    r = np.random.default_rng(9)
    x, u = (r.standard_normal((3, 9000)) * 3).astype(np.float32), r.random(3).astype(np.float32)
    rows = [(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0)]
    want_ids = [S.sample(x[i], *rows[i], float(u[i]))[0] for i in range(3)]

    def work(be, seed):
        try:
            for k in range(12):
                c = S.Caches(be, [400 + 50 * seed, 30], [9, 2], 2, 64 if k % 2 else 128, seed=seed, weight=True)
                q = np.random.default_rng(seed).standard_normal((11, 8 * c.D)).astype(np.float32)
                qd, od = be.upload(q), be.empty(q.size)
                be.attn_tree(od, qd, c.table, 8, 2, c.D, S.scale_of(c.D))
                xd, ud, sd, idd = be.upload(x), be.upload(u), be.upload(S.settings(rows)), be.upload(np.zeros(3, np.int32))
                be.sample(idd, None, xd, 9000, 3, sd, ud)
                want, _, bound, _ = S.attention(q, c, 8, S.scale_of(c.D))
                if not (np.abs(od.numpy(np.float32, q.shape) - want).max(-1) <= bound).all() or list(idd.numpy(np.int32)) != want_ids:
                    bad.append((seed, k))
                for b in (qd, od, xd, ud, sd, idd):
                    b.free()
                c.free()
        except Exception as e:      # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(bes[i % 2], i)) for i in range(2)]     # (a context serves one caller at a time: its buffers are not for two)
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    for b in bes:
        b.close()


@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("tok", [1, 12])
def test_offsets_beyond_32_bits(D, tok):
    """a cache of more than 2^32 bytes (and, in elements of both arrays, of more than 2^31): all keys equal, so that an output is the values' mean"""
    import torch
    be = backend()
    G, n_ctx = 8, 2 ** 31 // (8 * D) + 4096
    k = torch.zeros(n_ctx, G * D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(G * D, n_ctx, dtype=torch.bfloat16, device="cuda")
    n = n_ctx - 5
    v[:, n - 1000:n] = 1.0
    v[-1, :] = 2.0
    w, pos = torch.zeros(G, n_ctx, device="cuda"), torch.arange(n_ctx, device="cuda", dtype=torch.int32).repeat(G, 1)
    q, out = torch.ones(tok, 2 * G * D, device="cuda"), torch.zeros(tok, 2 * G * D, device="cuda")
    mask = torch.ones(tok, tok, dtype=torch.uint8, device="cuda")
    t = np.zeros(1, capi.CACHE)
    t[0] = (k.data_ptr(), v.data_ptr(), w.data_ptr(), w.data_ptr(), pos.data_ptr(), pos.data_ptr(), 0, n_ctx, n, tok, n - 3)
    torch.cuda.synchronize()
    be.attn_tree(out, q, t, 2 * G, G, D, 1.0, tree_mask=mask, cache_type=capi.BF16)
    be.sync()
    o = out.double().cpu().numpy().reshape(tok, 2 * G, D)
    tol = S.EPS * (n + 64)      # sums of n terms
    assert np.abs(o[:, :, :-1] * n / 1000 - 1).max() <= tol and np.abs(o[:, -1, -1] / 2 - 1).max() <= tol
    assert np.abs(w[:, :n].double().cpu().numpy() * n / (2 * tok) - 1).max() <= tol and float(w[:, n:].abs().max()) == 0
    k[n - 3:n] = 7.0            # three slots go, all weights equal: the last ones stay for their position and move into the slots that go
    w[:, [5, 17, 40000]] = 0.0
    w[:, n - 3:n] = 1.0
    torch.cuda.synchronize()
    be.kv_evict(t, G, D, n_recent=3, cache_type=capi.BF16)
    be.sync()
    assert bool((k[[5, 17, 40000]] == 7.0).all()) and bool((v[:-1][:, [5, 17, 40000]] == 1.0).all())
    assert pos[0, [5, 17, 40000]].tolist() == [n - 3, n - 2, n - 1]
    be.close()
