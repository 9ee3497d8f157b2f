"""Plain 64-bit restatement of the key/value cache in codes of 8 bits, token by token, and of what reads it."""
import math

import numpy as np

LOWEST = -120


def exponent(top):
    """Of the scale that a largest magnitude asks for: floor(log2(top)) - 6, at least -120."""
    return LOWEST if top == 0.0 else max(math.frexp(float(top))[1] - 7, LOWEST)


class Page:
    """One page of one kv head: rows of codes and an exponent, begun anew by a token at row 0."""

    def __init__(self, rows, hd, codes=None, e=None):
        self.q = np.zeros((rows, hd), dtype=np.int64) if codes is None else codes.astype(np.int64) - 128
        self.e = e

    def add(self, row, x):
        need = exponent(np.abs(x).max())
        if row == 0:
            self.e = need
        elif need > self.e:
            self.q[:row] = np.floor(self.q[:row] / 2.0 ** (need - self.e)).astype(np.int64)
            self.e = need
        self.q[row] = np.floor(np.asarray(x, dtype=np.float64) * 2.0 ** (-self.e)).astype(np.int64)

    @property
    def codes(self):
        return self.q + 128

    @property
    def scale(self):
        return 2.0 ** self.e

    def values(self):
        return (self.q + 0.5) * 2.0 ** self.e


def coded(x, page):
    """[tokens, heads, hd] from position 0 as the values that the cache keeps of them once all are in."""
    out = np.empty(x.shape, dtype=np.float64)
    for lo in range(0, x.shape[0], page):
        part = x[lo:lo + page]
        for h in range(x.shape[1]):
            pg = Page(page, x.shape[2])
            for i, row in enumerate(part[:, h]):
                pg.add(i, row)
            out[lo:lo + page, h] = pg.values()[:len(part)]
    return out


def rotate(x, pos, turns, interleaved, amplitude):
    """One head's vector ``x`` at position ``pos``: the first 2 len(turns) dims turned in pairs."""
    y, n = np.array(x, dtype=np.float64), len(turns)
    for j in range(n):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
        angle = 2.0 * math.pi * math.fmod(pos * float(turns[j]), 1.0)
        c, s = amplitude * math.cos(angle), amplitude * math.sin(angle)
        y[a], y[b] = x[a] * c - x[b] * s, x[a] * s + x[b] * c
    return y


def attend(q, k, v, multiplier, cap, lo, hi):
    """One query over the keys [lo, hi) of ``k``, ``v`` [keys, hd]."""
    s = (k[lo:hi] @ q) * multiplier
    if cap:
        s = cap * np.tanh(s / cap)
    w = np.exp(s - s.max())
    return (w / w.sum()) @ v[lo:hi]
