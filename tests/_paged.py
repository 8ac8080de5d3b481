"""Plain forms, in 64 bits or in whole numbers, of the operators on caches in 8 bits and in pages, and of the verification of drafted tokens; and the caches that their tests bring."""
import numpy as np

from powerserve_b200 import capi
from tests import _serve as S

BLOCK = 16


def slot_index(P, D):
    """[K, V][slot][channel]: where a page's code lies"""
    t, d = np.arange(P)[:, None], np.arange(D)[None]
    return np.stack([((t // 8) * (D // 16) + d // 16) * 128 + (t % 8) * 16 + d % 16, ((t // 16) * D + d) * 16 + t % 16])


class Cache:
    """Host copies and device arrays of a paged cache with random codes; tables of random pages. What lies outside the filled slots is -128, no-number scales where no slot is filled."""

    def __init__(self, be, lens, G, D, P=16, layers=1, spare=2, room=0, seed=0, junk=True):
        r = np.random.default_rng(seed)
        self.be, self.G, self.D, self.P, self.lens = be, G, D, P, list(lens)
        need = [-(-n // P) for n in lens]
        self.n_pages = sum(need) + spare
        order = r.permutation(self.n_pages)
        self.codes = r.integers(-127, 128, (layers, self.n_pages, G, 2, P * D)).astype(np.int8)
        self.scales = (r.random((layers, self.n_pages, G, 2, P // BLOCK)) * 0.05 + 1e-3).astype(np.float32)
        self.tables, at = [], 0
        self.refs = np.zeros(self.n_pages, np.int32)
        for n in need:
            t = np.full(max(1, n + room), -1, np.int32)
            t[:n] = order[at:at + n]
            self.refs[t[:n]] += 1
            at += n
            self.tables.append(t)
        self.index = slot_index(P, D)
        if junk:
            used = np.zeros((self.n_pages, P // BLOCK), bool)
            for n, t in zip(lens, self.tables):
                for b in range(-(-n // BLOCK)):
                    used[t[b * BLOCK // P], b % (P // BLOCK)] = True
            self.scales[:, ~used.reshape(self.n_pages, 1, 1, -1).repeat(G, 1).repeat(2, 2)] = np.nan
        self.cache = capi.PagedCache(be, layers, self.n_pages, P, G, D, codes=be.upload(self.codes), scales=be.upload(self.scales), refs=be.upload(self.refs))
        self.dev = [be.upload(t) for t in self.tables]

    def seqs(self, toks, hidden=None):
        t = np.zeros(len(self.lens), capi.PAGED_SEQ)
        t["table"], t["n_kv"], t["n_tok"], t["n_table"] = [d.ptr for d in self.dev], self.lens, toks, [len(x) for x in self.tables]
        if hidden is not None:
            t["hidden"] = [h.ptr for h in hidden]
        return t

    def values(self, i, kv, layer=0, n=None, dtype=np.float64):
        """[slots][G][D] of sequence i"""
        n = self.lens[i] if n is None else n
        j = np.arange(n)
        p = self.tables[i][j // self.P]
        c = self.codes[layer, p, :, kv][np.arange(n)[:, None, None], np.arange(self.G)[None, :, None], self.index[kv][j % self.P][:, None, :]]
        return c.astype(dtype) * self.scales[layer, p, :, kv][np.arange(n)[:, None], np.arange(self.G)[None], (j % self.P // BLOCK)[:, None]][..., None].astype(dtype)

    def read(self):
        """(codes, scales, refs) of the device"""
        c = self.cache
        return c.codes.numpy(np.int8, self.codes.shape), c.scales.numpy(np.float32, self.scales.shape), c.refs.numpy(np.int32, self.refs.shape)

    def free(self):
        self.cache.free()
        for d in self.dev:
            d.free()


def store(c, layer, k, v, toks):
    """the cache's host copies after rows k, v [tokens][G * D] (float32) went into the last slots"""
    t0, f = 0, np.float32
    for i, (n, t) in enumerate(zip(c.lens, toks)):
        for b in range((n - t) // BLOCK, -(-n // BLOCK) if t else 0):
            lo, hi = max(b * BLOCK, n - t), min((b + 1) * BLOCK, n)
            page, o = c.tables[i][b * BLOCK // c.P], b * BLOCK % c.P
            for kv, x in enumerate((k, v)):
                rows = x[t0 + lo - (n - t):t0 + hi - (n - t)].reshape(-1, c.G, c.D).astype(f)
                for g in range(c.G):
                    old = c.scales[layer, page, g, kv, o // BLOCK] if lo > b * BLOCK else f(0)
                    now = max(old, np.abs(rows[:, g]).max() / f(127))
                    for j in range(b * BLOCK, lo):
                        at = c.index[kv][j % c.P]
                        was = c.codes[layer, page, g, kv, at].astype(f)
                        c.codes[layer, page, g, kv, at] = np.rint(was * (old / now)).astype(np.int8) if now > 0 else 0
                    for j in range(lo, hi):
                        q = rows[j - lo, g] / now if now > 0 else np.zeros(c.D, f)
                        c.codes[layer, page, g, kv, c.index[kv][j % c.P]] = np.clip(np.rint(q), -127, 127).astype(np.int8)
                    c.scales[layer, page, g, kv, o // BLOCK] = now
        t0 += t


def attention(q, c, toks, H, scale, masks=None, hidden=None, layer=0):
    """(out [tokens][H * D], bound on a float32 kernel's error per output row)

    The bound, with e = 2^-24.  A query's number is off by at most 2 e of its row's largest, so its products with n-bit codes, summed over D channels, by 2 e D max|q| max|k| scale, and the exact sum's
    rounding, scaling and base-2 exponent by 6 e |z|: |dz| <= e (2 D M + 6 |z|).  The weight is off by a factor 1 + 2 dz + 8 e, and by 2 e of the row's largest weight where it is rounded to 23 bits; sums over n
    slots of weights, split any way, add n e each: with sum p = 1 and every term at most max|v|, e (2 (2 D M + 6 Z) + 8 + 4 n + 8) max|v|."""
    G, D = c.G, c.D
    R, out, t0 = H // G, np.zeros((q.shape[0], H * D)), 0
    bound = np.zeros(q.shape[0])
    for i, (n, t) in enumerate(zip(c.lens, toks)):
        if not t:
            continue
        k, v = c.values(i, 0, layer), c.values(i, 1, layer)
        vis = S.sees(n, t, None if masks is None else masks[i], np.zeros(n, np.uint8) if hidden is None else hidden[i])
        for h in range(H):
            qh = q[t0:t0 + t, h * D:(h + 1) * D].astype(np.float64) * scale
            z = np.where(vis, qh @ k[:, h // R].T, -np.inf)
            top = np.where(vis.any(-1), z.max(-1, initial=-np.inf), 0.0)
            p = np.where(vis, np.exp(z - top[:, None]), 0.0)
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1.0)
            out[t0:t0 + t, h * D:(h + 1) * D] = p @ v[:, h // R]
            M = np.abs(qh).max(-1) * np.abs(k[:, h // R]).max(initial=0.0)
            Z = np.where(vis, np.abs(z), 0.0).max(-1, initial=0.0)
            bound[t0:t0 + t] = np.maximum(bound[t0:t0 + t], S.EPS * (2 * (2 * D * M + 6 * Z) + 16 + 4 * n) * np.abs(v[:, h // R]).max(initial=0.0))
        t0 += t
    return out, bound


def edit(refs, P, edits):
    """edits one phase after another: (table, from or None, n_old, n_new), tables are host arrays that change; (held, copies [(source, destination, blocks)])"""
    begun = [None if f is None else f.copy() for _, f, _, _ in edits]
    up = lambda n: -(-n // P)   # noqa: E731
    for (t, f, old, _), b in zip(edits, begun):
        if f is not None:
            t[:up(old)] = b[:up(old)]
            np.add.at(refs, t[:up(old)], 1)
    for t, f, old, new in edits:
        np.subtract.at(refs, t[up(new):up(old)], 1)
    free = list(np.flatnonzero(refs == 0))
    held, copies, spent, growers = [], [], 0, {}
    now = refs.copy()
    for t, f, old, new in edits:
        if new <= old:
            held.append(new)
            continue
        last = int(t[up(old) - 1]) if old % P else -1
        rank = growers.get(last, 0)
        if last >= 0:
            growers[last] = rank + 1
        copy = last >= 0 and now[last] - rank > 1
        need = int(copy) + up(new) - up(old)
        spent += need
        if not (spent <= len(free) or (need == 0 and rank == 0)):
            held.append(old)
            continue
        mine = free[spent - need:spent]
        if copy:
            copies.append((last, mine[0], -(-(old % P) // BLOCK)))
            refs[last] -= 1
            t[up(old) - 1] = mine[0]
        t[up(old):up(new)] = mine[int(copy):]
        refs[mine] = 1
        held.append(new)
    return held, copies


def compact(c, i, first, keep):
    """the cache's host copies after sequence i's slots first + keep moved to first, first + 1, ..."""
    if not len(keep):
        return
    f = np.float32
    was, scales = c.codes.copy(), c.scales.copy()
    src = list(range(first // BLOCK * BLOCK, first)) + [first + k for k in keep]
    for b in range(0, len(src), BLOCK):
        to = first // BLOCK * BLOCK + b
        page, o = c.tables[i][to // c.P], to % c.P // BLOCK
        at = [(c.tables[i][j // c.P], j % c.P) for j in src[b:b + BLOCK]]
        for kv in range(2):
            s = np.stack([scales[:, p, :, kv, j // BLOCK] for p, j in at])           # [slots][L][G]
            now = s.max(0)
            c.scales[:, page, :, kv, o] = now
            for e, (p, j) in enumerate(at):
                x = was[:, p, :, kv][:, :, c.index[kv][j]].astype(f)
                ratio = np.divide(s[e], now, out=np.zeros_like(now), where=now > 0)
                c.codes[:, page, :, kv][..., c.index[kv][(to + e) % c.P]] = np.rint(x * ratio[..., None]).astype(np.int8)


def distribution(x, temperature, top_k, top_p, min_p):
    """what the settings leave of a row of logits, normalised"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    w = np.zeros(len(x))
    if not (x > -np.inf).any():
        return w
    if not temperature > 0:
        w[int(np.argmax(x))] = 1.0
        return w
    best = np.argsort(-x, kind="stable")
    best = best[x[best] > -np.inf]
    top = x[best[0]]
    if 0 < top_k < len(x):
        best = best[:top_k]
    e = np.where(x[best] == top, 1.0, np.exp(np.where(x[best] == top, 0.0, x[best] - top) / temperature))
    ok = np.ones(len(e), bool)
    if top_p < 1:
        ok = np.cumsum(e) - e < max(top_p, 0.0) * e.sum()
        ok[0] = True
    if min_p > 0:
        ok &= e >= min(min_p, 1.0)
    w[best[ok]] = e[ok]
    return w / w.sum()


def verify(parents, tokens, u, logits, settings, draft=None, draft_settings=None):
    """(path, next token) of one sequence, by the definition: a distribution is written down after every rejection"""
    cur, path, V = 0, [0], logits.shape[1]
    p = distribution(logits[0], *settings[0])
    for i in range(1, len(parents)):
        c = int(tokens[i])
        if parents[i] != cur or not 0 <= c < V:
            continue
        q = np.zeros(V)
        if draft is None:
            q[c] = 1.0
        else:
            q = distribution(draft[cur], *draft_settings[cur])
        if float(u[i]) * q[c] < p[c]:
            cur = i
            path.append(i)
            p = distribution(logits[i], *settings[i])
            continue
        left = np.maximum(p - q, 0.0)
        if left.sum() > 0:
            p = left / left.sum()
    if not p.sum() > 0:
        return path, -1
    run = np.cumsum(p)
    some = np.flatnonzero(p > 2.0 ** -45)
    return path, min(int(np.searchsorted(run, float(u[0]) * run[-1], side="right")), int(some[-1]))
