"""Rotary positions, the 8-bit key/value cache and attention over it, in 64 bits, token by token."""
import math

import numpy as np


def rotary(x, positions, frequencies, part, layout, axes, factor=1.0, inverse=False):
    """x (tokens, heads, dim) fp64, positions (tokens, axes) integers, frequencies per pair of a section."""
    y = np.array(x, dtype=np.float64)
    n = part // axes
    for ax in range(axes):
        for p, f in enumerate(frequencies):
            i, j = (p, p + n // 2) if layout == 'half' else (2 * p, 2 * p + 1)
            i, j = i + ax * n, j + ax * n
            # the angle modulo 2 pi in extended precision: positions may be large
            t = np.array([_angle(int(v), f) for v in positions[:, ax]])[:, None]
            t = -t if inverse else t
            a, b = x[:, :, i], x[:, :, j]
            y[:, :, i] = factor * (a * np.cos(t) - b * np.sin(t))
            y[:, :, j] = factor * (a * np.sin(t) + b * np.cos(t))
    return y


def _angle(position, f):
    turns = round(f / (2 * math.pi) * 2.0 ** 64)            # whole numbers of 2^-64 turns wrap without error
    return (position * turns % (1 << 64)) / 2.0 ** 64 * 2 * math.pi


def fit(amax, bits):
    """Factor of a block whose largest new value is amax (an fp32 number)."""
    if not math.isfinite(amax):
        return math.nan
    if bits == 'int8':
        f = max(float(np.float32(np.float64(amax) / 127.0)), 2.0 ** -60)
    else:
        e = -60
        while 448.0 * 2.0 ** e < amax:
            e += 1
        f = 2.0 ** e
    return f if f <= 2.0 ** 60 else math.nan


def nearest_code(x, bits):
    """x rounded to the nearest code, ties to even: whole numbers, or e4m3's steps of 2^(e - 3) (2^-9 below 2^-6)."""
    if bits == 'int8':
        return np.clip(np.rint(x), -127, 127)
    _, e = np.frexp(np.maximum(np.abs(x), 2.0 ** -6))
    step = np.exp2(e - 4.0)
    return np.rint(x / step) * step


class Cache:
    """codes k, v (blocks, heads, 64, dim) as the numbers they stand for, scales (blocks, heads, 2)."""

    def __init__(self, k, v, scales, bits):
        self.k, self.v, self.scales, self.bits = np.array(k, np.float64), np.array(v, np.float64), np.array(scales, np.float64), bits

    def append(self, k, v, pages, lengths, counts):
        """k, v (tokens, heads, dim) fp32 values, the rows of one sequence after the other."""
        row = 0
        for s, (start, n) in enumerate(zip(lengths, counts)):
            done = 0
            while done < n:
                at = (start + done) % 64
                m = min(64 - at, n - done)
                slot = (start + done) // 64
                page = pages[s][slot] if slot < len(pages[s]) else -1
                if 0 <= page < len(self.k):
                    for codes, src, w in ((self.k, k, 0), (self.v, v, 1)):
                        for h in range(self.k.shape[1]):
                            self._block(codes[page, h], page, h, w, at, np.asarray(src[row + done:row + done + m, h], np.float64))
                done += m
            row += n

    def _block(self, codes, page, h, w, at, x):
        with np.errstate(invalid='ignore'):
            amax = float(np.max(np.abs(x))) if np.all(np.isfinite(x)) else math.inf
        f = fit(amax, self.bits)
        old = float(self.scales[page, h, w])
        if at:
            if math.isnan(f) or math.isnan(old):
                f = math.nan
            elif old >= f:
                f = old
            else:
                ratio = np.float64(np.float32(old / f))
                codes[:at] = nearest_code(np.float64(np.float32(codes[:at] * ratio)), self.bits)
        self.scales[page, h, w] = f
        if math.isnan(f):
            codes[at:at + len(x)] = 0.0
            return
        inv = np.float64(np.float32(1.0 / f))
        codes[at:at + len(x)] = nearest_code(np.float64(np.float32(x * inv)), self.bits)

    def values(self, page, i):
        """Keys and values (heads, dim) of place i of a block."""
        return self.k[page, :, i] * self.scales[page, :, 0:1], self.v[page, :, i] * self.scales[page, :, 1:2]

    def sequence(self, pages, length):
        """Keys, values (tokens, heads, dim) and whether each is there."""
        H, D = self.k.shape[1], self.k.shape[3]
        k, v, there = np.zeros((length, H, D)), np.zeros((length, H, D)), np.zeros(length, bool)
        for b in range((length + 63) // 64):
            n = min(64, length - 64 * b)
            if b < len(pages) and 0 <= pages[b] < len(self.k):
                p = pages[b]
                k[64 * b:64 * b + n] = (self.k[p, :, :n] * self.scales[p, :, 0][:, None, None]).transpose(1, 0, 2)
                v[64 * b:64 * b + n] = (self.v[p, :, :n] * self.scales[p, :, 1][:, None, None]).transpose(1, 0, 2)
                there[64 * b:64 * b + n] = True
        return k, v, there


def attend(cache, q, pages, lengths, counts, scale, causal=True, window=None):
    """(o, lse, sum of p |v|) of rows q (tokens, q_heads, dim).  A NaN key or value among those that a row sees makes both
    its result and its lse NaN."""
    o, a, lse = np.zeros(q.shape), np.zeros(q.shape), np.full(q.shape[:2], -math.inf)
    group, row = q.shape[1] // cache.k.shape[1], 0
    for s, (length, n) in enumerate(zip(lengths, counts)):
        k, v, there = cache.sequence(pages[s], length)
        j = np.arange(length)
        for i in range(n):
            at = length - n + i
            seen = there & ((j <= at) if causal else True) & ((j > at - window) if window else True)
            if np.any(seen):
                for h in range(q.shape[1]):
                    z = scale * (k[seen, h // group] @ q[row + i, h])
                    p = np.exp(z - np.max(z))
                    vs = v[seen, h // group]
                    o[row + i, h] = p @ vs / p.sum()
                    a[row + i, h] = p @ np.abs(vs) / p.sum()
                    lse[row + i, h] = np.max(z) + math.log(p.sum()) if np.isfinite(p.sum()) and not np.isnan(vs).any() else math.nan
        row += n
    return o, lse, a
