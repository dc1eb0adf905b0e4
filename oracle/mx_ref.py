"""The microscaled formats and the 8-bit key/value cache in 64 bits -- TEST INFRASTRUCTURE ONLY.

Only ``tests/`` and ``__graft_entry__.smoke()`` may import it, as the checker.  All of it is
numpy in float64 from the formats' definitions:

* MXFP4 (OCP Microscaling Formats v1.0): blocks of 32 along the last axis, scale byte b for
  2^(b - 127) (255: NaN), e2m1 codes, element 2i in the low nibble.
* e4m3 (OCP 8-bit floating point): 4 exponent bits of bias 7, 3 mantissa bits, no infinity,
  0x7F / 0xFF NaN, 448 the largest.
"""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def scale_value(byte):
    b = np.asarray(byte, dtype=np.int64)
    return np.where(b == 255, np.nan, np.ldexp(1.0, np.minimum(b, 254) - 127))


def _nearest_even(v, grid):
    """Index of the grid value nearest to v >= 0, ties to the even index, saturated."""
    hi = np.clip(np.searchsorted(grid, v), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = v - grid[lo], grid[hi] - v
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    return np.where((v <= grid[hi]) & take_lo, lo, hi)


def quantize_mxfp4(x):
    """[..., K] -> packed [..., K/2], scales [..., K/32]."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(b).all(-1)
    amax = np.where(finite, np.where(np.isfinite(b), np.abs(b), 0).max(-1), 0)
    e = np.where(amax > 0, np.frexp(np.where(amax > 0, amax, 1))[1] - 1 - 2, -127)
    byte = np.where(finite, np.clip(e + 127, 0, 254), 255).astype(np.uint8)
    safe = np.where(finite[..., None], b, 0.0)
    code = _nearest_even(np.abs(safe) / scale_value(np.where(finite, byte, 127))[..., None], E2M1)
    code = code | (np.signbit(safe).astype(np.int64) << 3)
    code = code.reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def dequantize_mxfp4(packed, scales):
    code = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    return (v.reshape(*scales.shape, 32) * scale_value(scales)[..., None]).reshape(code.shape)


def _e4m3_table():
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, np.ldexp(m / 8.0, -6), np.ldexp(1 + m / 8.0, e - 7))
    v[127] = np.nan
    return v


E4M3 = _e4m3_table()


def e4m3_decode(code):
    code = np.asarray(code)
    return E4M3[code & 127] * np.where(code & 128, -1.0, 1.0)


def e4m3_encode(v):
    """Nearest, ties to even; what is not finite becomes NaN.  No finite value is above 448."""
    v = np.asarray(v, dtype=np.float64)
    fin = np.isfinite(v)
    code = _nearest_even(np.where(fin, np.abs(v), 0), E4M3[:127])
    code = np.where(fin, code, 127) | (np.signbit(v).astype(np.int64) << 7)
    return code.astype(np.uint8)


def kv8_byte(amax):
    """Byte of the smallest power of two, 2^-126 at least, with amax <= 448 of it."""
    if amax == 0:
        return 1
    e = int(np.frexp(amax)[1]) - 1 - 8
    if amax > np.ldexp(448.0, e):
        e += 1
    return max(e + 127, 1)


class Cache:
    """k, v codes [P, H, page, D] (both token by token here) and scale bytes [P, H]."""

    def __init__(self, k, v, ks, vs):
        self.codes, self.bytes = [k.copy(), v.copy()], [ks.copy(), vs.copy()]
        self.P, self.H, self.page, self.D = k.shape

    def _id(self, table, b, j):
        if j >= table.shape[1] or not 0 <= table[b, j] < self.P:
            return None
        return int(table[b, j])

    def append(self, which, x, table, start, cu):
        for b in range(len(start)):
            s, n = int(start[b]), int(cu[b + 1] - cu[b])
            for p0 in range(s // self.page * self.page, s + n, self.page):
                lo, hi = max(s, p0), min(s + n, p0 + self.page)
                pid = self._id(table, b, p0 // self.page)
                if pid is None or hi <= lo:
                    continue
                tok = x[cu[b] + lo - s:cu[b] + hi - s].astype(np.float64)
                for h in range(self.H):
                    t = tok[:, h]
                    byte = kv8_byte(np.abs(np.where(np.isfinite(t), t, 0)).max())
                    codes = self.codes[which][pid, h]
                    if lo > p0:
                        was = int(self.bytes[which][pid, h])
                        if was < byte:
                            codes[:lo - p0] = e4m3_encode(e4m3_decode(codes[:lo - p0]) * np.ldexp(1.0, was - byte))
                        byte = max(was, byte)
                    self.bytes[which][pid, h] = byte
                    codes[lo - p0:hi - p0] = e4m3_encode(t * np.ldexp(1.0, 127 - byte))

    def values(self, which, table, b, L):
        """[L, H, D] of sequence b, NaN-free zeros where a page is missing, and which tokens are there."""
        out, here = np.zeros((L, self.H, self.D)), np.zeros(L, dtype=bool)
        for p0 in range(0, L, self.page):
            pid = self._id(table, b, p0 // self.page)
            if pid is None:
                continue
            n = min(self.page, L - p0)
            v = e4m3_decode(self.codes[which][pid, :, :n]) * scale_value(self.bytes[which][pid])[:, None, None]
            out[p0:p0 + n], here[p0:p0 + n] = v.transpose(1, 0, 2), True
        return out, here


def attention(q, cache, table, context, cu, scale, causal=True, window=0):
    """(out, lse, bound): bound holds per output the terms of the error of a 16-bit computation
    as multiples, see below: sum of weights times |v| (``av``), the largest |v|, and the
    largest error weight of a row's scores, sum |q||k| scale."""
    T, heads, D = q.shape
    G = heads // cache.H
    out, lse = np.zeros((T, heads, D)), np.full((T, heads), -np.inf)
    av, vmax, sabs = np.zeros((T, heads, D)), np.zeros((T, heads, 1)), np.zeros((T, heads, 1))
    for b in range(len(context)):
        n = int(cu[b + 1] - cu[b])
        L = int(min(max(context[b], 0), table.shape[1] * cache.page))
        if n == 0 or L == 0:
            continue
        k, here = cache.values(0, table, b, L)
        v, _ = cache.values(1, table, b, L)
        key = np.arange(L)
        for i in range(n):
            pos = L - n + i
            see = here.copy()
            if causal:
                see &= key <= pos
            if window:
                see &= key > pos - window
            t = cu[b] + i
            if not see.any():
                continue
            for hq in range(heads):
                kk, vv, qq = k[see, hq // G], v[see, hq // G], q[t, hq].astype(np.float64)
                s = kk @ qq * scale
                m = s.max()
                p = np.exp(s - m)
                out[t, hq] = p @ vv / p.sum()
                lse[t, hq] = m + np.log(p.sum())
                av[t, hq] = p @ np.abs(vv) / p.sum()
                vmax[t, hq] = np.abs(vv).max()
                sabs[t, hq] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
    return out, lse, {"av": av, "vmax": vmax, "sabs": sabs}
