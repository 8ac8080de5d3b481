"""The serving operators in company: the same bits with other, larger calls in between; several threads on one context; a layer-list model's context; and, against 64 bits,
caches of tens of thousands of slots and channels whose magnitudes lie far apart."""
import threading

import numpy as np
import pytest
import torch

from powerserve_b200 import arch, arch_synth, capi
from tests import _serve as S
from tests import test_gpu_serve_attention as A
from tests import test_gpu_serve_evict as E
from tests import test_gpu_serve_sample as P
from tests.test_gpu_serve_attention import be  # noqa: F401

pytestmark = pytest.mark.gpu


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


@pytest.mark.parametrize("D", [64, 128, 96])
def test_the_same_bits_with_others_in_between(be, D):  # noqa: F811
    """one token, a few and a tree, each with a call that needs more memory, an eviction and a sampling before it comes again"""
    r = np.random.default_rng(D)
    x = torch.from_numpy((r.standard_normal((3, 50000)) * 3).astype(np.float32)).cuda()
    u, ids, probs = torch.rand(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    settings = torch.from_numpy(S.settings([(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.02)]).view(np.float32).reshape(3, 4).copy()).cuda()

    def draw():
        be.sample(ids, probs, x, 50000, 3, settings, u)
        return ids.cpu().numpy(), bits(probs.cpu().numpy())

    first = draw()
    for k, (lens, toks) in enumerate((([700, 90], [1, 1]), ([700, 90], [12, 3]), ([5000, 64], [40, 2]))):
        c = S.Caches(be, lens, toks, 2, D, seed=12, weight=True)
        _, a = A.run(be, c, 8)
        w = [c.weights(i) - c.w[i] for i in range(2)]
        other = S.Caches(be, [9000 + 4000 * k, 300], [30 + 10 * k, 1], 2, D, seed=13, weight=True)
        A.run(be, other, 8)
        E.check(be, [3000], [1000], 2, 64, n_sink=1, n_recent=30)
        again = draw()
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
        for i in range(2):      # (the weights begin where they began)
            be._ck(be.L.ps_cuda_memcpy_h2d(be.h, c.bufs[4 * i + 2].ptr, c.w[i].ctypes.data, c.w[i].nbytes))
        _, b = A.run(be, c, 8)
        assert np.array_equal(bits(a), bits(b))
        for i in range(2):
            assert np.array_equal(bits(c.weights(i) - c.w[i]), bits(w[i]))
        c.free()
        other.free()


@pytest.mark.parametrize("D,H,G,toks", [(128, 8, 2, [1, 1]), (64, 8, 2, [2, 1]), (128, 8, 2, [32, 5]), (64, 14, 2, [12, 1]), (96, 4, 2, [3, 1])])
def test_tens_of_thousands_of_slots(be, D, H, G, toks):  # noqa: F811
    c = S.Caches(be, [32700, 20001], toks, G, D, seed=9, weight=True)
    q, out = A.run(be, c, H)
    want, w, _, _ = S.attention(q, c, H, S.scale_of(D))
    # sums over the slots are taken in parts (tiles, warps, splits) whose roundings go either way: a few steps of the whole, not one for each slot
    assert np.linalg.norm(out - want) <= 64 * S.EPS * np.linalg.norm(want)
    assert np.abs(out - want).max() <= 256 * S.EPS * np.abs(want).max()
    for i, n in enumerate(c.lens):
        got = c.weights(i)[:, :n].astype(np.float64)
        exp = c.w[i][:, :n] + w[i]
        assert np.linalg.norm(got - exp) <= 64 * S.EPS * np.linalg.norm(exp)
        assert (np.abs(got - exp) <= 4 * S.EPS * exp + 256 * S.EPS * w[i].max()).all()
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96])
@pytest.mark.parametrize("toks", [[1, 2], [20, 3]])
@pytest.mark.parametrize("least", [-16, -30])
def test_channels_of_magnitudes_far_apart(be, dtype, D, toks, least):  # noqa: F811
    """values whose channels lie up to 2^16 apart keep their precision, channel by channel; further apart the small ones are held to 2^-39 of the largest beside them.
    Keys by channel, and the queries the other way, so that all products count: up to 2^16 apart"""
    H, G = 8, 2
    c = S.Caches(be, [300, 90], toks, G, D, dtype=dtype, seed=D)
    r = np.random.default_rng(1)
    fv, fk = np.exp2(r.integers(least, 1, G * D)).astype(np.float32), np.exp2(r.integers(-16, 1, D)).astype(np.float32)
    n = sum(toks)
    q = r.standard_normal((n, H * D)).astype(np.float32)
    want, _, bound, _ = S.attention(q, c, H, S.scale_of(D))
    most = max(np.abs(c.v[i][:, :l]).max() for i, l in enumerate(c.lens))
    bufs = []
    for i in range(2):      # (powers of two: the same products, and outputs times fv)
        k, v = c.k[i] * np.tile(fk, G), c.v[i] * fv[:, None]
        if dtype == "bf16":
            k, v = S.bf16(k)[0], S.bf16(v)[0]
        bufs += [be.upload(k), be.upload(v)]
        c.table["k"][i], c.table["v"][i] = bufs[-2].ptr, bufs[-1].ptr
    x = q / np.tile(fk, H)
    qd, od = be.upload(x), be.empty(n * H * D)
    be.attn_tree(od, qd, c.table, H, G, D, S.scale_of(D), cache_type=c.type)
    f = np.repeat(fv.reshape(G, D), H // G, 0).reshape(-1)
    got = od.numpy(np.float32, (n, H * D)) / f
    assert (np.abs(got - want) <= bound[:, None] + 2.0 ** -38 * most / f).all()
    for b in bufs + [qd, od]:
        b.free()
    c.free()


def test_threads_on_one_context(be):  # noqa: F811
    """each with arrays and a stream of its own"""
    r = np.random.default_rng(9)
    rows = [(1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.02)]
    x, u = (r.standard_normal((3, 9000)) * 3).astype(np.float32), r.random(3).astype(np.float32)
    ids = [S.sample(x[i], *(float(np.float32(f)) if isinstance(f, float) else f for f in rows[i]), float(u[i]))[0] for i in range(3)]
    caches = [S.Caches(be, [400 + 300 * s, 30], [9, 2] if s % 2 else [1, 1], 2, 64 if s < 2 else 128, seed=s) for s in range(4)]
    bad = []

    def work(s):
        try:
            c = caches[s]
            n = sum(c.toks)
            q = np.random.default_rng(s).standard_normal((n, 8 * c.D)).astype(np.float32)
            want, _, bound, _ = S.attention(q, c, 8, S.scale_of(c.D))
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                xd, ud = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
                sd = torch.from_numpy(S.settings(rows).view(np.float32).reshape(3, 4).copy()).cuda()
                for k in range(40):
                    qd, out, idd = torch.from_numpy(q).cuda(), torch.zeros(n, 8 * c.D, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
                    be.attn_tree(out, qd, c.table, 8, 2, c.D, S.scale_of(c.D))
                    qd.zero_()
                    be.sample(idd, None, xd, 9000, 3, sd, ud)
                    if not (np.abs(out.cpu().numpy() - want).max(-1) <= bound).all() or idd.cpu().tolist() != ids:
                        bad.append((s, k))
        except Exception as e:      # noqa: BLE001
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    for c in caches:
        c.free()


def test_a_layer_list_model_s_context(tmp_path):
    layer = arch_synth.nufusun_layer
    cfg = arch_synth.nufusun_config(64, 500, [layer(2, 1, 16, 16, bias_max=9.0)], eps=1e-5, embed_scale=0.5)
    arch_synth.write_model_dir(str(tmp_path), cfg, arch_synth.nufusun_weights(cfg, seed=3, rel_rows=8))
    m = arch.load_model(str(tmp_path), dtype="float32", max_batch=8, n_ctx=64)
    want = m.forward([1, 2, 3])
    r = np.random.default_rng(1)
    for toks in ([1, 1], [20, 3]):
        A.check(m.be, S.Caches(m.be, [700, 90], toks, 2, 64, hidden=True, weight=True, seed=3), 8, weight=True)
    E.check(m.be, [1025, 3000], [1024, 900], 2, 64, n_sink=1, n_recent=30)
    E.check(m.be, [1025], [1024], 2, 64, dtype="bf16", n_recent=30)
    x = (r.standard_normal((len(P.FILTERS), 9000)) * 2.5).astype(np.float32)
    P.check(m.be, x, P.FILTERS, r.random(len(x)))
    m.reset()
    assert np.array_equal(bits(m.forward([1, 2, 3])), bits(want))       # and the model's own passes are what they were
    m.close()
