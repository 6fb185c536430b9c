"""The 8-bit paged cache in 64-bit numpy, from its definition: what the
tests of grx_kv8_* compare with."""

from __future__ import annotations

import numpy as np

TORCH = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
EPS2 = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # half a step of each type


def rope_table(positions, d, base=10000.0):
    f = base ** (-np.arange(0, d, 2) / d)
    a = np.arange(positions)[:, None] * f
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def rotate(x, pos, table, mode):
    """x [rows][heads][d] (float64) at positions pos [rows]."""
    if mode == "none":
        return x
    c, s = (table[pos].astype(np.float64)[:, None, :, j] for j in (0, 1))
    half = x.shape[-1] // 2
    y = np.empty_like(x)
    if mode == "pairs":
        a, b = x[..., 0::2], x[..., 1::2]
        y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:]
        y[..., :half], y[..., half:] = a * c - b * s, a * s + b * c
    return y


class Cache:
    """k, v [pages][heads][page][d] int8, scale [pages][heads][2] float32."""

    def __init__(self, pages, heads, page, d, rng=None):
        self.page, self.d, self.heads = page, d, heads
        if rng is None:
            self.k = np.zeros((pages, heads, page, d), np.int8)
            self.v = np.zeros_like(self.k)
            self.scale = np.zeros((pages, heads, 2), np.float32)
        else:
            self.k = rng.integers(-127, 128, (pages, heads, page, d)).astype(np.int8)
            self.v = rng.integers(-127, 128, (pages, heads, page, d)).astype(np.int8)
            self.scale = ((0.5 + rng.random((pages, heads, 2))) / 73).astype(np.float32)

    def append(self, pages, length, k, v, table=None, mode="none"):
        """The last len(k) of a sequence's `length` tokens; pages: its row of the page table."""
        t = len(k)
        pos = np.arange(length - t, length)
        x = (rotate(k.astype(np.float64), pos, table, mode), v.astype(np.float64))
        for b in range((length - t) // self.page, -(-length // self.page)):
            lo, hi = max(length - t, b * self.page), min(length, (b + 1) * self.page)
            held = lo - b * self.page
            for j, pool in enumerate((self.k, self.v)):
                new = x[j][lo - (length - t):hi - (length - t)].transpose(1, 0, 2)  # [heads][tokens][d]
                for h in range(self.heads):
                    old = self.scale[pages[b], h, j] if held else np.float32(0)
                    y = new[h]
                    if np.isnan(old) or not np.isfinite(y).all():
                        s = np.float32(np.nan)
                        q = np.zeros_like(y)
                    else:
                        s = max(old, np.float32(np.abs(y).max() / 127.0))
                        if s > old and held:
                            p = pool[pages[b], h, :held].astype(np.float64)
                            pool[pages[b], h, :held] = np.rint(p * float(old) / float(s)).astype(np.int8)
                        q = np.clip(np.rint(y / float(s)), -127, 127) if s > 0 else np.zeros_like(y)
                    pool[pages[b], h, held:held + hi - lo] = q.astype(np.int8)
                    self.scale[pages[b], h, j] = s

    def values(self, pages, length, j):
        """[heads][length][d] float64."""
        pool = (self.k, self.v)[j]
        n = -(-length // self.page)
        x = pool[list(pages[:n])].astype(np.float64) * self.scale[list(pages[:n])][..., j][..., None, None]
        return x.transpose(1, 0, 2, 3).reshape(self.heads, -1, self.d)[:, :length]


def attend(cache, pages, length, q, table=None, mode="none", scale=None, window=0, first=0, half=False):
    """q [t][heads][d] of the last t tokens → out [t][heads][d], lse, and a
    bound on a float32 kernel's error of out (see below)."""
    t, heads, d = q.shape
    scale = d**-0.5 if scale is None else scale
    pos = np.arange(length - t, length)
    out, lse, tol = np.zeros((t, heads, d)), np.full((t, heads), -np.inf), np.zeros((t, heads))
    if length == 0:
        return out, lse, tol
    k, v = cache.values(pages, length, 0), cache.values(pages, length, 1)
    x = rotate(q.astype(np.float64), pos, table, mode)
    group = heads // cache.heads
    for r in range(t):
        lo, hi = max(first, pos[r] - window + 1 if window else 0, 0), pos[r] + 1
        if lo >= hi:
            continue
        for h in range(heads):
            kk, vv = k[h // group, lo:hi], v[h // group, lo:hi]
            with np.errstate(invalid="ignore"):
                s = kk @ x[r, h] * scale
                m = s.max()
                e = np.exp(s - m)
                out[r, h] = e @ vv / e.sum()
                lse[r, h] = m + np.log(e.sum())
                # A score is off by what the query's 22 bits below its largest
                # value leave (2^-23 each, and as much for the rotation) on
                # every product, and by four roundings of the score itself; a
                # weight by that, by ex2's 2^-22 and by its 24 bits; the sums
                # by a step (2^-23) for each of n/16 products and of the joins.
                ds = (2.0**-22 * np.abs(x[r, h]).max() * np.abs(kk).sum(1).max() * abs(scale)
                      + 4 * 2.0**-24 * np.abs(s).max())
                tol[r, h] = np.abs(vv).max() * (2 * ds + 2.0**-21 + ((hi - lo) / 16 + 32) * 2.0**-23)
                # The weights of 16-bit outputs are float16 (half a step 2^-11
                # of each, or 2^-25 of the reference below its smallest normal
                # number; the reference is at most 2·3 times a page's scale
                # where the scales are in 0.5..1.5, and counts 1 in the sum).
                if half:
                    tol[r, h] += np.abs(vv).max() * (2.0**-11 + (hi - lo) * 6 * 2.0**-25)
    return out, lse, tol
