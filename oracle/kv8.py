"""The 8-bit K/V pool's operators in 64 bits, in numpy: the oracle of the mkv_kv8_* calls.

TEST INFRASTRUCTURE ONLY, as oracle.py. Rows are float64 arrays holding the values of
the f32 / bf16 inputs; tiles are e4m3 values (float64) and exponents.
"""
from __future__ import annotations

import numpy as np

PAGE = 16
MIN_EXP = -100
# What e4m3 holds, from 0 to 448 (byte 0 .. 126): subnormals of 2^-9, then 3 bits of mantissa.
GRID = np.array([(m / 8 + (x > 0)) * 2.0 ** (max(x, 1) - 7) for x in range(16) for m in range(8)][:127])


def to_e4m3(x):
    """Nearest e4m3 value, ties to the even byte; NaN and infinities become NaN. |x| <= 448 otherwise."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    assert a.size == 0 or a.max() <= 448.0
    hi = np.clip(np.searchsorted(GRID, a), 1, 126)
    lo = hi - 1
    up, down = GRID[hi] - a, a - GRID[lo]
    y = np.where((up < down) | ((up == down) & (hi % 2 == 0)), GRID[hi], GRID[lo])
    return np.where(np.isfinite(x), np.copysign(y, x), np.nan)


def from_bytes(b):
    """The values of e4m3 bytes."""
    b = np.asarray(b, np.uint8)
    m = b & 0x7F
    y = np.where(m == 127, np.nan, GRID[np.minimum(m, 126)])
    return np.where(b & 0x80, -y, y)


def exponent(amax):
    """Least e >= MIN_EXP with amax <= 448 * 2^e."""
    e = MIN_EXP
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def tile_index(kv, d):
    """[16][d]: where row t, dim i of a K (kv = 0) or V tile stands in its 16 * d bytes."""
    t, i = np.arange(PAGE)[:, None], np.arange(d)[None]
    if kv == 0:
        return ((i // 16) * PAGE + t) * 16 + i % 16
    return (((i // 64) * 4 + t // 4) * 16 + i % 64 // 4) * 16 + i % 4 * 4 + t % 4


class Kv8:
    """One layer of a pool: val [2][blocks][Hkv][16][d] as held (times 2^exp)."""

    def __init__(self, blocks, hkv, d):
        self.hkv, self.d = hkv, d
        self.val = np.zeros((2, blocks, hkv, PAGE, d))
        self.exp = np.zeros((2, blocks, hkv), np.int64)

    @classmethod
    def read(cls, tiles, exps):
        """From the pool's bytes [2][blocks][Hkv][16 * d] and exponents."""
        o = cls(tiles.shape[1], tiles.shape[2], tiles.shape[3] // PAGE)
        for kv in range(2):
            o.val[kv] = from_bytes(tiles[kv][..., tile_index(kv, o.d).ravel()]).reshape(o.val[kv].shape)
        o.exp[:] = exps
        return o

    def append(self, k, v, new, ctx, tables):
        """tables: a list of block ids per sequence."""
        at = 0
        for n, c, table in zip(new, ctx, tables):
            pos = c - n
            while pos < c:
                end = min(c, pos - pos % PAGE + PAGE)
                blk, r0 = table[pos // PAGE], pos % PAGE
                for kv, x in enumerate((k, v)):
                    rows = x[at: at + end - pos]
                    for h in range(self.hkv):
                        y = rows[:, h]
                        amax = np.abs(y[np.isfinite(y)]).max(initial=0.0)
                        e = exponent(amax)
                        if r0 == 0:
                            self.val[kv, blk, h] = 0.0
                        else:
                            e = max(e, self.exp[kv, blk, h])
                            old = self.val[kv, blk, h] * 2.0 ** (self.exp[kv, blk, h] - e)
                            self.val[kv, blk, h] = to_e4m3(old)
                        self.exp[kv, blk, h] = e
                        self.val[kv, blk, h, r0: r0 + end - pos] = to_e4m3(y * 2.0 ** -e)
                at += end - pos
                pos = end

    def rows(self, kv, table, ctx):
        """[Hkv][ctx][d] of one sequence."""
        if ctx == 0:
            return np.zeros((self.hkv, 0, self.d))
        ids = list(table[: -(-ctx // PAGE)])
        x = self.val[kv][ids] * 2.0 ** self.exp[kv][ids][..., None, None]
        return x.transpose(1, 0, 2, 3).reshape(self.hkv, -1, self.d)[:, :ctx]

    def attend(self, q, new, ctx, tables, scale, zero_sink=False):
        """(o, a, s, f): a = sum p |v| / sum p, which errors of weights are relative to, s a bound
        on the error of a score's sum in f32 (log2 units), and f one on what f16 weights
        drop: the greatest weight times its tile's scale is held as 2^7 or more, and f16 ends
        at 2^-25, so each key loses at most 2^-32 of that, times 448. Padding rows are 0."""
        g = q.shape[1] // self.hkv
        o, a = np.zeros(q.shape), np.zeros(q.shape)
        s, f = np.zeros(q.shape[:2] + (1,)), np.zeros(q.shape[:2] + (1,))
        at = 0
        for n, c, table in zip(new, ctx, tables):
            if n == 0:
                continue
            if c == 0:
                at += n
                continue
            k, v = self.rows(0, table, c), self.rows(1, table, c)
            hide = np.arange(c)[None] > np.arange(c - n, c)[:, None]
            for h in range(q.shape[1]):
                kh, vh, qh = k[h // g], v[h // g], q[at: at + n, h]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = qh @ kh.T * scale
                    size = np.where(hide, 0.0, np.abs(qh) @ np.abs(kh).T * scale)
                    x = np.where(hide, -np.inf, x)
                    m = np.max(x, 1, keepdims=True, initial=0.0 if zero_sink else -np.inf)
                    p = np.exp(x - m)
                    total = p.sum(1, keepdims=True) + (np.exp(-m) if zero_sink else 0.0)
                    # (A NaN of a hidden key is not seen.)
                    odd = np.isnan(vh).any()
                    for t in range(n) if odd else ():
                        seen = c - n + t + 1
                        o[at + t, h] = p[t, :seen] @ vh[:seen] / total[t]
                        a[at + t, h] = p[t, :seen] @ np.abs(vh[:seen]) / total[t]
                    if not odd:
                        o[at: at + n, h] = p @ vh / total
                        a[at: at + n, h] = p @ np.abs(vh) / total
                    d = self.d
                    top = (p * 2.0 ** self.exp[1][list(table[: -(-c // PAGE)]), h // g].repeat(PAGE)[:c]).max(1)
                    f[at: at + n, h, 0] = c * 2.0 ** -32 * 448 * top / total[:, 0]
                    s[at: at + n, h, 0] = 1.45 * 2.0 ** -24 * (d * size.max(1) + 2 * np.abs(np.where(hide, 0, x)).max(1) + 32)
            at += n
        return o, a, s, f


def norm_rope(x, w, eps, inv_freq, pos, factor, interleaved):
    """RMSNorm(1 + w) (w None: none) and rotary positions of rows [n][heads][d]."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * (1.0 + w.astype(np.float64))
    half = len(inv_freq)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = pos.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle) * factor, np.sin(angle) * factor
    z = y.copy()
    z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    return z
