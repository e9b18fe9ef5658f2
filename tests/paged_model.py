"""A plain 64-bit model of the paged 8-bit cache: what it holds, and attention over it."""
from __future__ import annotations

import numpy as np

BLOCK = 16
TOP = {"int8": 127.0, "e4m3": 448.0}


def cache_value(x):
    """float32 values as the cache takes them: NaN is 0, magnitudes are cut at 2^62."""
    return np.clip(np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=np.inf, neginf=-np.inf),
                   -2.0 ** 62, 2.0 ** 62)


def exponent(amax, dtype):
    """Smallest k in [-40, 56] with amax <= TOP 2^k."""
    k = -40
    while k < 56 and amax > TOP[dtype] * 2.0 ** k:
        k += 1
    return k


def nearest_code(y, dtype):
    """The code nearest to y, ties to even, as a number."""
    if dtype == "int8":
        return np.rint(y)
    e = np.floor(np.log2(np.maximum(np.abs(y), 1e-300)))
    step = np.exp2(np.maximum(e, -6) - 3)
    return np.rint(y / step) * step


def rotate(x, pos, rope_dim, base, neox, factors=None, yarn=1.0):
    """x [n, heads, HD] float32 at positions pos: angles in 64 bits, each operation's result an
    fp32 number."""
    hd = x.shape[-1]
    rd = min(hd, rope_dim) // 2 * 2
    out = x.astype(np.float32).copy()
    if rd == 0:
        return out
    freq = np.float64(np.float32(base)) ** (-2.0 * np.arange(rd // 2) / rd) / max(1e-4, np.float64(np.float32(yarn)))
    if factors is not None:
        freq = freq / np.asarray(factors, np.float64)[: rd // 2]
    ang = np.asarray(pos, np.float64)[:, None] * freq
    c, s = (f(ang).astype(np.float32)[:, None] for f in (np.cos, np.sin))
    i = np.arange(rd // 2)
    u, v = (i, i + rd // 2) if neox else (2 * i, 2 * i + 1)
    a, b = out[..., u].copy(), out[..., v].copy()
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., u] = a * c - b * s
        out[..., v] = a * s + b * c
    return out


class Model:
    def __init__(self, n_seqs, n_layers, cap, n_kv, hd, dtype):
        self.dtype, self.L, self.HK, self.HD = dtype, n_layers, n_kv, hd
        nb = -(-cap // BLOCK)
        self.code = np.zeros((n_seqs, n_layers, 2, nb * BLOCK, n_kv, hd))
        self.k = np.full((n_seqs, n_layers, 2, nb, n_kv), -40, int)
        self.rows = [0] * n_seqs

    def write(self, s, l, w, pos0, x):
        """Rows x [n, HK, HD] (fp32) written from pos0 on in one call."""
        x = cache_value(x)
        n = len(x)
        for b in range(pos0 // BLOCK, (pos0 + n - 1) // BLOCK + 1):
            t = np.arange(b * BLOCK, (b + 1) * BLOCK)
            new, old = (t >= pos0) & (t < pos0 + n), t < pos0
            for h in range(self.HK):
                k = exponent(np.abs(x[t[new] - pos0, h]).max(), self.dtype)
                if old.any():
                    k0 = self.k[s, l, w, b, h]
                    k = max(k, k0)
                    c = self.code[s, l, w, t[old], h] * 2.0 ** (k0 - k)
                    self.code[s, l, w, t[old], h] = nearest_code(c, self.dtype)
                self.code[s, l, w, t[new], h] = nearest_code(x[t[new] - pos0, h] / 2.0 ** k, self.dtype)
                self.k[s, l, w, b, h] = k

    def values(self, s, l, w, lo, hi):
        t = np.arange(lo, hi)
        return self.code[s, l, w, lo:hi] * np.exp2(self.k[s, l, w, t // BLOCK])[..., None]

    def fork(self, src, dst, n=None):
        self.code[dst], self.k[dst] = self.code[src], self.k[src]
        self.rows[dst] = self.rows[src] if n is None else n

    def keep(self, s, rows):
        """Rows kept, scaled and rounded anew; leading pages that stay in place are untouched."""
        rows = list(rows)
        same = 0
        while same < len(rows) and rows[same] == same:
            same += 1
        first = same // 32 * 32 if same < len(rows) else same
        for l in range(self.L):
            for w in range(2):
                v = self.values(s, l, w, 0, self.rows[s])[rows]
                if first < len(rows):
                    self.write(s, l, w, first, v[first:])
        self.rows[s] = len(rows)

    def step(self, s, l, pos0, q, k, v, H, scale, softcap=0.0, window=0, append=True, src=None,
             **rope):
        """Tokens pos0 .. of one sequence and layer: q [n, H*HD], k and v [n, HK*HD] (fp32).
        Returns out [n, H*HD] and a bound of what a 32-bit evaluation may be off."""
        n, HK, HD, src = len(q), self.HK, self.HD, l if src is None else src
        pos = np.arange(pos0, pos0 + n)
        if append:
            self.write(s, src, 0, pos0, rotate(k.reshape(n, HK, HD), pos, **rope))
            self.write(s, src, 1, pos0, v.reshape(n, HK, HD))
        qr = rotate(q.reshape(n, H, HD), pos, **rope).astype(np.float64)
        K, V = (self.values(s, src, w, 0, pos0 + n) for w in range(2))
        out, tol = np.zeros((n, H, HD)), np.zeros((n, H, 1))
        for h in range(H):
            g = h // (H // HK)
            for i in range(n):
                lo = max(0, pos[i] - window + 1) if window else 0
                Kr, Vr = K[lo:pos[i] + 1, g], V[lo:pos[i] + 1, g]
                e = Kr @ qr[i, h] * scale
                size = (np.abs(Kr) @ np.abs(qr[i, h])).max() * scale
                if softcap > 0:
                    e = softcap * np.tanh(e / softcap)
                p = np.exp(e - e.max())
                out[i, h] = p @ Vr / p.sum()
                # A score in 32 bits: q split into two fp16 parts (2^-22), its rotation three
                # roundings (3 * 2^-24), one fp32 addition per 16 products and a few more
                # operations ((HD/16 + 5) * 2^-23 of the sum of magnitudes).  A weight: twice
                # the score's error (its own and the maximum's) and exp2's 2^-22; as parts of
                # 16 bits 2^-22, or 2^-25 of the largest where it is small.  The sums over rows:
                # one rounding (2^-23) per 16 rows.
                ds = size * ((HD / 16 + 5) * 2.0 ** -23 + 2.0 ** -22 + 3 * 2.0 ** -24) + 2.0 ** -22
                tol[i, h] = np.abs(Vr).max() * (4 * ds + 2.0 ** -21 + (len(p) / 16 + 4) * 2.0 ** -23
                                              + len(p) * 2.0 ** -25)
        return out.reshape(n, H * HD), np.broadcast_to(tol, (n, H, HD)).reshape(n, H * HD)
