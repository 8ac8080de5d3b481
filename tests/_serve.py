"""Plain 64-bit forms of the serving operators (ps_cuda_attn_tree, ps_cuda_kv_evict, ps_cuda_sample) and the caches that their tests bring."""
import math

import numpy as np

from powerserve_b200 import capi

EPS = 2.0 ** -24    # half a step of float32, relative


def bf16(a):
    """float32 rounded to bfloat16: (bit patterns, the values they stand for)"""
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(a), np.uint16(0x7FC0), r)
    return r, (r.astype(np.uint32) << 16).view(np.float32)


class Caches:
    """Host copies and device arrays of one cache per sequence.  What no token may see is filled with NaN and infinities."""

    def __init__(self, be, lens, toks, G, D, n_ctx=None, dtype="f32", hidden=False, weight=False, seed=0, scale=1.0, odd=0):
        r = np.random.default_rng(seed)
        self.be, self.lens, self.toks, self.G, self.D, self.dtype = be, list(lens), list(toks), G, D, dtype
        self.type = capi.F32 if dtype == "f32" else capi.BF16
        self.k, self.v, self.w, self.hid, self.bufs = [], [], [], [], []
        self.table = np.zeros(len(self.lens), capi.CACHE)
        for i, (n, t) in enumerate(zip(self.lens, self.toks)):
            c = n_ctx or n + 3 + odd
            k, v = (r.standard_normal((c, G * D)) * scale).astype(np.float32), (r.standard_normal((G * D, c)) * scale).astype(np.float32)
            h = np.zeros(c, np.uint8)
            if hidden:
                h[:n - t] = r.random(n - t) < 0.2
            off = h.astype(bool) | (np.arange(c) >= n)
            k[off] = np.where(r.random((int(off.sum()), G * D)) < 0.5, np.nan, np.inf)
            v[:, off] = np.where(r.random((G * D, int(off.sum()))) < 0.5, np.nan, -np.inf)
            w = r.random((G, c)).astype(np.float32)
            if dtype == "f32":
                kd, vd = be.upload(k), be.upload(v)
            else:
                kb, k = bf16(k)
                vb, v = bf16(v)
                kd, vd = be.upload(kb), be.upload(vb)
            wd, hd = be.upload(w), be.upload(h)
            self.bufs += [kd, vd, wd, hd]
            self.k.append(k); self.v.append(v); self.w.append(w); self.hid.append(h)
            self.table[i] = (kd.ptr, vd.ptr, wd.ptr if weight else 0, 0, 0, 0, hd.ptr if hidden else 0, c, n, t, 0)

    def weights(self, i):
        return self.bufs[4 * i + 2].numpy(np.float32, self.w[i].shape)

    def free(self):
        for b in self.bufs:
            b.free()


def sees(n, t, mask, hidden):
    m = np.ones((t, n), bool)
    m[:, n - t:] = np.tril(np.ones((t, t), bool)) if mask is None else mask.astype(bool)
    return m & ~hidden[None, :n].astype(bool)


def attention(q, caches, H, scale, masks=None):
    """(out [tokens][H * D], weights per cache, bound on a float32 kernel's error per output row, and on its weights' rows)

    The bound, with e = 2^-24.  A score is a sum of D products, each off by at most 5 e (its factors are held to 2 e, a product of the two low parts, 4 e at most
    of it, may be missing) and D additions: |dz| <= (D + 8) e S with S = scale sum |q k|; base-2 exponents and their scaling add 4 e |z|.  exp doubles neither: a
    weight is off by a factor 1 + 2 dz + 8 e, the sums over n slots add n e each."""
    G, D = caches.G, caches.D
    R, out, t0 = H // G, np.zeros((q.shape[0], H * D)), 0
    bound, weights, wbound = np.zeros(q.shape[0]), [], []
    for i, (n, t) in enumerate(zip(caches.lens, caches.toks)):
        k, v = caches.k[i][:n].astype(np.float64), caches.v[i][:, :n].astype(np.float64)
        vis = sees(n, t, None if masks is None else masks[i], caches.hid[i])
        dead = ~vis.any(0)
        k, v = np.where(dead[:, None], 0.0, k), np.where(dead[None], 0.0, v)
        w, wb = np.zeros((G, n)), 0.0
        for h in range(H if t else 0):
            g = h // R
            qh = q[t0:t0 + t, h * D:(h + 1) * D].astype(np.float64) * scale
            z = np.where(vis, qh @ k[:, g * D:(g + 1) * D].T, -np.inf)
            S = np.where(vis, np.abs(qh) @ np.abs(k[:, g * D:(g + 1) * D]).T, 0.0).max(-1)
            top = np.where(vis.any(-1), z.max(-1, initial=-np.inf), 0.0)
            p = np.where(vis, np.exp(z - top[:, None]), 0.0)
            p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
            out[t0:t0 + t, h * D:(h + 1) * D] = p @ v[g * D:(g + 1) * D].T
            rel = EPS * (2 * (D + 16) * S + 2 * n + 32)
            bound[t0:t0 + t] = np.maximum(bound[t0:t0 + t], rel * np.abs(v).max(initial=0.0))
            w[g] += p.sum(0)
            wb = max(wb, float((rel[:, None] * p).sum(0).max(initial=0.0)) * R)
        weights.append(w)
        wbound.append(wb)
        t0 += t
    return out, weights, bound, wbound


def tree(n, r):
    m = np.zeros((n, n), np.uint8)
    for i in range(n):
        if i:
            m[i] = m[int(r.integers(max(0, i - 3), i))]
        m[i, i] = 1
    return m


def evict(weight, pos, n, keep, n_sink, n_recent):
    """(sources, destinations) of one kv head's moves"""
    w = weight[:n].astype(np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    none = np.isnan(weight[:n])         # after -inf itself
    safe = np.zeros(n, bool) if pos is None else (pos[:n] < n_sink) | (pos[:n].astype(np.int64) > int(pos[:n].max(initial=0)) - n_recent)
    kept = np.zeros(n, bool)
    kept[np.lexsort((np.arange(n), none, -w, ~safe))[:keep]] = True
    return np.flatnonzero(kept & (np.arange(n) >= keep)), np.flatnonzero(~kept & (np.arange(n) < keep))


def sample(x, temperature, top_k, top_p, min_p, u):
    """(token, probability) of one row"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    best = np.argsort(-x, kind="stable")
    best = best[x[best] > -np.inf]
    top = x[best[0]]
    if 0 < top_k < len(x):
        best = best[:top_k]
    w = np.where(x[best] == top, 1.0, np.exp(np.where(x[best] == top, 0.0, x[best] - top) / temperature))
    if top_p < 1:
        before = np.cumsum(w) - w
        ok = before < max(top_p, 0.0) * w.sum()
        ok[0] = True
        best, w = best[ok], w[ok]
    if min_p > 0:
        ok = w >= min(min_p, 1.0)
        best, w = best[ok], w[ok]
    order = np.argsort(best)
    best, w = best[order], w[order]
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    some = np.flatnonzero(w > 2.0 ** -45)
    at = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), int(some[-1]))
    return int(best[at]), float(w[at] / w.sum())


def settings(rows):
    return np.array([tuple(r) for r in rows], capi.SAMPLER)


def scale_of(D):
    return 1.0 / math.sqrt(D)
