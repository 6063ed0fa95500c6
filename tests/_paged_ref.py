"""The paged cache of kv_append, kv_read and attn_paged on the host: inputs of a
case, and what the formulas give in 64 bits (numpy), with the roundings that the
operators make counted beside them."""
import numpy as np

import _oracle as O

DT_F16, DT_BF16 = 11, 12
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
HALF = {DT_BF16: 2.0 ** -8, DT_F16: 2.0 ** -11}      # half a step of the 16-bit type, relative
TINY = {DT_BF16: 0.0, DT_F16: 2.0 ** -25}            # and below fp16's normal numbers
F32 = 2.0 ** -24


def quantise(y, dt):
    """y f32 [..., hd] -> codes [..., hd] (0..15), scale bytes [..., hd/32]."""
    g = y.reshape(y.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(g).all(-1)
    amax = np.where(bad, 0, np.abs(np.where(np.isfinite(g), g, 0)).max(-1)).astype(np.float64)
    m, e = np.frexp(amax)
    lo, hi = (-126, 125) if dt == DT_BF16 else (-23, 13)
    e = np.clip(np.where(amax > 0, e - 3 + (m > 0.75), lo), lo, hi)
    w = np.abs(np.where(np.isfinite(g), g, 0)).astype(np.float64) / 2.0 ** e[..., None]
    code = (w > .25).astype(int) + (w >= .75) + (w > 1.25) + (w >= 1.75) + (w > 2.5) + (w >= 3.5) + (w > 5)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(g))
    return code.reshape(y.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    """What codes and scale bytes stand for, in 64 bits."""
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return E2M1[codes] * np.repeat(s, 32, -1)


class Paged:
    """A pool and the sequences of one call.  `seqs` is a list of (new rows,
    cache rows with them); `extra` rows behind the last sequence."""

    def __init__(self, seqs, dt=DT_BF16, bits=16, H=4, Hkv=2, hd=64, page=16, seed=0, extra=0, holes=(), spare=2,
                 ragged=None):
        self.rng = np.random.default_rng([seed, H, Hkv, hd, page, bits, dt])
        self.seqs, self.dt, self.bits, self.H, self.Hkv, self.hd, self.page = seqs, dt, bits, H, Hkv, hd, page
        self.b, self.n = len(seqs), sum(r for r, _ in seqs) + extra
        need = [-(-t // page) for _, t in seqs]
        self.maxpages, self.npages = max(need + [1]) + 1, sum(need) + spare
        ids = self.rng.permutation(self.npages)
        self.table = np.full((self.b, self.maxpages), -1, np.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = ids[at:at + k]
            at += k
        for s, p, v in holes:                      # pages that are none
            self.table[s, p] = v
        self.len = np.array([t for _, t in seqs], np.int32)
        self.rows = np.cumsum([0] + [r for r, _ in seqs]).astype(np.int32)
        even = len({r for r, _ in seqs}) == 1 and extra == 0
        self.ragged = (not even) if ragged is None else ragged
        self.rb = hd * 2 if bits == 16 else hd // 2 + hd // 32

    # ---- pools ----
    def stale(self):
        """A pool whose every slot holds NaN."""
        if self.bits == 16:
            return np.full((self.npages, self.Hkv, self.page * self.rb), 0xFF, np.uint8)
        a = np.full((self.npages, self.Hkv, self.page * self.rb), 0x77, np.uint8)
        a[..., self.page * self.hd // 2:] = 255
        return a

    def put(self, pool, page, slot, y):
        """Store y [Hkv][hd] (f32, rounded here) at a slot of a page."""
        ps, hd = self.page, self.hd
        if self.bits == 16:
            pool[page, :, slot * hd * 2:(slot + 1) * hd * 2] = O.encode(y.astype(np.float32), self.dt).view(np.uint8)
        else:
            c, s = quantise(y.astype(np.float32), self.dt)
            pool[page, :, slot * hd // 2:(slot + 1) * hd // 2] = c[..., 0::2] | c[..., 1::2] << 4
            at = ps * hd // 2 + slot * hd // 32
            pool[page, :, at:at + hd // 32] = s

    def get(self, pool, page, slot):
        """The values [Hkv][hd] held there, in 64 bits."""
        ps, hd = self.page, self.hd
        if self.bits == 16:
            return O.decode(np.ascontiguousarray(pool[page, :, slot * hd * 2:(slot + 1) * hd * 2]).view(np.uint16),
                            self.dt).astype(np.float64).reshape(self.Hkv, hd)
        b = pool[page, :, slot * hd // 2:(slot + 1) * hd // 2]
        at = ps * hd // 2 + slot * hd // 32
        return values(np.stack((b & 15, b >> 4), -1).reshape(self.Hkv, hd), pool[page, :, at:at + hd // 32])

    def held(self, pool):
        """All values of a pool, [npages][Hkv][page][hd] in 64 bits."""
        ps, hd = self.page, self.hd
        if self.bits == 16:
            return O.decode(pool.view(np.uint16), self.dt).astype(np.float64).reshape(self.npages, self.Hkv, ps, hd)
        b = pool[..., :ps * hd // 2].reshape(self.npages, self.Hkv, ps, hd // 2)
        return values(np.stack((b & 15, b >> 4), -1).reshape(self.npages, self.Hkv, ps, hd),
                      pool[..., ps * hd // 2:].reshape(self.npages, self.Hkv, ps, hd // 32))

    def where(self, s, pos):
        """(page, slot) of a position, or None."""
        if pos < 0 or pos >= self.maxpages * self.page:
            return None
        p = self.table[s, pos // self.page]
        return (p, pos % self.page) if 0 <= p < self.npages else None

    def filled(self, upto=None, scale=1.0):
        """A pool whose sequences' rows hold normal values, NaN elsewhere."""
        pool = self.stale()
        for s, (r, t) in enumerate(self.seqs):
            for pos in range(min(t, self.maxpages * self.page) if upto is None else upto[s]):
                at = self.where(s, pos)
                if at:
                    self.put(pool, *at, scale * self.rng.standard_normal((self.Hkv, self.hd)))
        return pool

    def each_row(self):
        """(row, sequence, position)."""
        for s, (r, t) in enumerate(self.seqs):
            for i in range(r):
                yield int(self.rows[s]) + i, s, t - r + i

    # ---- kv_append ----
    def make_x(self, ldx=None, scale=1.0):
        ldx = ldx or (self.H + 2 * self.Hkv) * self.hd
        return O.encode((scale * self.rng.standard_normal((self.n, ldx))).astype(np.float32), self.dt)

    def tables(self, base=10000.0):
        f = base ** (-np.arange(0, self.hd, 2) / self.hd)
        a = np.arange(self.maxpages * self.page)[:, None] * f
        return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)

    def project(self, x, row, pos, kind, rope=0, norm=None, eps=0.0, cos=None, sin=None):
        """q, k, v of a row before they are rounded, and a bound of what f32 adds
        to each (kind float64); kind float32: the operator's own steps in its own
        roundings, which is what a 4-bit code is made from."""
        H, K, hd = self.H, self.Hkv, self.hd
        y = O.decode(x[row, :(H + 2 * K) * hd], self.dt).astype(kind).reshape(H + 2 * K, hd)
        err = np.zeros(y.shape)
        if norm is not None:
            g = np.concatenate((np.repeat(norm[0][None], H, 0), np.repeat(norm[1][None], K, 0))).astype(kind)
            z = y[:H + K]
            ss = (z.astype(np.float64) ** 2).sum(-1, keepdims=True) / hd + float(np.float32(eps))
            y[:H + K] = (z * (1.0 / np.sqrt(ss)).astype(kind)) * g
            err[:H + K] = 3 * F32 * np.abs(y[:H + K])               # inv, and two products
        if rope and 0 <= pos < self.maxpages * self.page:
            c, s = cos[pos].astype(kind), sin[pos].astype(kind)
            ix = (np.arange(0, hd, 2), np.arange(1, hd, 2)) if rope == 1 else (np.arange(hd // 2), np.arange(hd // 2) + hd // 2)
            a, b = y[:H + K, ix[0]], y[:H + K, ix[1]]
            ea, eb = err[:H + K, ix[0]].copy(), err[:H + K, ix[1]].copy()
            y[:H + K, ix[0]], y[:H + K, ix[1]] = a * c - b * s, b * c + a * s
            # the inputs' errors, and two roundings of either product's size
            err[:H + K, ix[0]] = ea * np.abs(c) + eb * np.abs(s) + 2 * F32 * (np.abs(a * c) + np.abs(b * s))
            err[:H + K, ix[1]] = eb * np.abs(c) + ea * np.abs(s) + 2 * F32 * (np.abs(b * c) + np.abs(a * s))
        return y[:H], y[H:H + K], y[H + K:], err[:H], err[H:H + K]

    # ---- attn_paged ----
    def attend(self, q, kheld, vheld, row, s, pos, scale):
        """Output [H][hd] of a row in 64 bits over the held() values of the pools,
        and how far the operator may be off before its last rounding.  p is rounded once to the 16-bit type and its
        sum is taken over f32 values: numerator and denominator are each off by
        half a step of p at most; the scores by (hd + 4) roundings of f32 over sum
        |q k|; exp2 and the running maximum's factors by 2^-20; the sums by a
        rounding a row."""
        H, K, hd = self.H, self.Hkv, self.hd
        at = [w for w in (self.where(s, p) for p in range(max(pos + 1, 0))) if w]
        out, tol = np.zeros((H, hd)), np.zeros((H, hd))
        if not at:
            return out, tol
        pages, slots = np.array(at).T
        kk, vv = kheld[pages, :, slots], vheld[pages, :, slots]
        qf = O.decode(q[row], self.dt).astype(np.float64).reshape(H, hd)
        for h in range(H):
            k, v = kk[:, h // (H // K)], vv[:, h // (H // K)]
            with np.errstate(invalid="ignore"):
                sc = k @ qf[h] * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[h] = p @ v
                tol[h] = p @ np.abs(v) * (2 * HALF[self.dt] + 2 * ((hd + 4) * F32 * (np.abs(k) @ np.abs(qf[h])).max() *
                                          abs(scale) + 2.0 ** -20 + len(at) * F32))
        return out, tol

    def spec(self, **kw):
        d = dict(n=self.n, b=self.b, hkv=self.Hkv, hd=self.hd, page=self.page, maxpages=self.maxpages,
                 npages=self.npages, dt=self.dt, bits=self.bits)
        if self.ragged:
            d["ragged"] = 1
        return {**d, **kw}


def near(got, want, tol, dt):
    """got within tol and one rounding to dt of want; NaN and infinities alike."""
    fine = np.isfinite(want)
    if not np.array_equal(np.isnan(got), np.isnan(want)) or not np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]):
        return False
    g, w, t = got[fine], want[fine], tol[fine]
    return bool(np.all(np.abs(g - w) <= t + HALF[dt] * (np.abs(w) + t) + TINY[dt]))
