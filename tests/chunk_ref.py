"""The operators on batches of chunks in 64 bits, straight from their definitions
(include/tlkv.h), for the tests: numpy, session by session, head by head."""
import numpy as np

U24 = 2.0 ** -24          # rounding to f32, relative


class Batch:
    """Sessions with paged caches in one pool, and their new rows.  sizes: (pos, n) of each."""

    def __init__(self, seed, shape, sizes, page=16, q8=False, pad=0, tail=2, spare=3, gap=0):
        H, KV, D = shape
        self.H, self.KV, self.D, self.q8, self.page, self.pad = H, KV, D, q8, page, pad
        self.sizes = sizes
        r = self.rng = np.random.default_rng(seed)
        per = [-(-(p + n) // page) for p, n in sizes]
        total = sum(per) + spare
        self.cap = total * page
        deal = r.permutation(total).astype(np.uint32)
        self.tables, at = [], 0
        for k in per:
            self.tables.append(deal[at:at + k].copy())
            at += k
        self.row, rows = [], 0
        for _, n in sizes:
            self.row.append(rows)
            rows += n + gap
        self.rows = rows + tail
        self.q_stride, self.kv_stride = H * D + pad, KV * D + pad
        self.q = r.standard_normal((self.rows, self.q_stride)).astype(np.float32)
        self.kin = r.standard_normal((self.rows, self.kv_stride)).astype(np.float32)
        self.vin = r.standard_normal((self.rows, self.kv_stride)).astype(np.float32)
        x = r.standard_normal((2, KV, self.cap, D)).astype(np.float32)
        if q8:
            (self.k, self.ks), (self.v, self.vs) = quantize(x[0]), quantize(x[1])
        else:
            self.k, self.v = x[0].astype(np.float16), x[1].astype(np.float16)
        self.live = [i for i, (_, n) in enumerate(sizes) if n]

    def phys(self, i, p):
        p = np.asarray(p)
        if self.tables[i] is None:
            return p.astype(np.int64)
        return self.tables[i][p // self.page].astype(np.int64) * self.page + p % self.page

    def cached(self, x, kv, rows):
        """f64 rows of K ('k') or V ('v') of a kv head; rows outside the pool: NaN."""
        ok = rows < self.cap
        at = np.where(ok, rows, 0)
        v = getattr(self, x)[kv, at].astype(np.float64)
        if self.q8:
            s = getattr(self, x + "s")[kv, at].astype(np.float64)
            v = (v.reshape(*s.shape, 32) * s[..., None]).reshape(v.shape)
        v[~ok] = np.nan
        return v


def quantize(x):
    """Q8_0 of f32 x[..., D]: int8 values and f16 scales, in f32 arithmetic as the cache does."""
    b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    d = (np.abs(b).max(-1) / np.float32(127)).astype(np.float32)
    inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), 0).astype(np.float32)
    return np.rint(b * inv[..., None]).astype(np.int8).reshape(x.shape), d.astype(np.float16)


def sees(B, i, prefix=0, window=0, first=None):
    """[n, end] which keys the session's rows see (pages outside the pool: none)."""
    pos, n = B.sizes[i]
    p = np.arange(pos, pos + n)[:, None]
    j = np.arange(pos + n)[None, :]
    s = j <= p
    if window:
        s &= p - j < window
    s |= j < prefix
    if first is not None:
        s &= j >= first[B.row[i]:B.row[i] + n].astype(np.int64)[:, None]
    return s & (B.phys(i, np.arange(pos + n)) < B.cap)[None, :]


def probs(B, i, h, scale, prefix=0, window=0, first=None, softcap=0.0, slopes=None):
    """(probabilities [n, end], log sums [n], visible, largest |score| bound) of one head."""
    pos, n = B.sizes[i]
    end = pos + n
    kv = h // (B.H // B.KV)
    K = B.cached("k", kv, B.phys(i, np.arange(end)))
    q = B.q[B.row[i]:B.row[i] + n, h * B.D:(h + 1) * B.D].astype(np.float64)
    see = sees(B, i, prefix, window, first)
    used = see.any(0)
    K = np.where(used[:, None], K, 0.0)
    with np.errstate(all="ignore"):
        x = q @ K.T * scale
        big = np.linalg.norm(q, axis=1).max() * np.linalg.norm(K, axis=1).max() * scale
        if softcap:
            x = softcap * np.tanh(x / softcap)
            big += softcap
        if slopes is not None:
            x = x - float(slopes[h]) * np.abs(np.arange(pos, end)[:, None] - np.arange(end)[None, :])
        x = np.where(see, x, -np.inf)
        top = x.max(1)
        top0 = np.where(np.isfinite(top), top, 0.0)
        e = np.where(see, np.exp(x - top0[:, None]), 0.0)
        tot = e.sum(1)
        lse = np.where(tot > 0, top0 + np.log(tot), -np.inf)
        p = e / np.where(tot > 0, tot, 1)[:, None]
    return p, lse, see, big


def attn(B, scale, prefix=None, **kw):
    """(dst, lse, relative 2-norm tolerance).

    A score differs from its exact value by the roundings of q as a pair of f16
    (22 bits), of the matrix unit's f32 sums and of the factors after them, all
    relative to |q||k| scale (and the cap): a few units of 2^-24 of it, 4 taken;
    its probability differs relatively by as much and by the exponential's and
    the pair's rounding (8 units).  The output is an average under those
    probabilities: 4 times their sum covers numerator and denominator."""
    dst = np.zeros((B.rows, B.H * B.D))
    lse = np.zeros((B.rows, B.H))
    top = 0.0
    for i in B.live:
        pos, n = B.sizes[i]
        r = slice(B.row[i], B.row[i] + n)
        phys = B.phys(i, np.arange(pos + n))
        for h in range(B.H):
            p, s, see, big = probs(B, i, h, scale, prefix=prefix[i] if prefix else 0, **kw)
            V = B.cached("v", h // (B.H // B.KV), phys)
            used = see.any(0)
            # unseen values have no part, whatever they hold
            for t in range(n):
                dst[r.start + t, h * B.D:(h + 1) * B.D] = p[t, see[t]] @ V[see[t]] if see[t].any() else 0
            lse[r, h] = s
            top = max(top, big if used.any() else 0)
    return dst, lse, 4 * (4 * top + 8) * U24


def weight(B, lse, scale, prefix=None, **kw):
    """Per session: sum over rows and heads of exp(s - lse) with the given f32 lse, and a tolerance."""
    out, top = [], 0.0
    for i in range(len(B.sizes)):
        pos, n = B.sizes[i]
        w = np.zeros(pos + n)
        for h in range(B.H if n else 0):
            p, s, see, big = probs(B, i, h, scale, prefix=prefix[i] if prefix else 0, **kw)
            given = lse[B.row[i]:B.row[i] + n, h].astype(np.float64)
            with np.errstate(all="ignore"):
                f = np.where(np.isfinite(given), np.exp(s - given), 0.0)
            w += (p * f[:, None]).sum(0)
            top = max(top, big)
        out.append(w)
    return out, 4 * (4 * top + 8) * U24


def normed(x, w, eps):
    x = x.astype(np.float64)
    y = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w.astype(np.float64)


def rotated(x, pos, rdim, theta, neox):
    """x[n, heads, D] f64 rotated at pos[n]."""
    y = x.copy()
    for j in range(rdim // 2):
        a, b = (j, j + rdim // 2) if neox else (2 * j, 2 * j + 1)
        ang = pos.astype(np.float64) * float(np.float32(theta)) ** (-2.0 * j / rdim)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def evict(w, len_, keep, sink, recent):
    """(kept, evicted) positions of one session, rising."""
    v = np.where(np.isnan(w[:len_]), -np.inf, w[:len_].astype(np.float64))
    nan = np.isnan(w[:len_])
    order = sorted(range(len_), key=lambda j: (sink <= j < len_ - recent, nan[j], -v[j], j))
    return np.array(sorted(order[:keep])), np.array(sorted(order[keep:]), dtype=np.int64)
