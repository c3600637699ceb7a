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
            if b < len(pages) and 0 <= block(pages[b]) < len(self.k):
                p = block(pages[b])
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


def attend_formed(cache, q, pages, lengths, counts, scale, causal=True, window=None, cap=None, slopes=None, prefix=None,
                  since=None, until=None):
    """``attend`` with formed scores and masks: cap tanh(z / cap), less slopes[h] |p - j|; a row sees the tokens below its
    sequence's prefix, and of the others those from since[row] on and below until[row], causal and in the window."""
    o, a, lse = np.zeros(q.shape), np.zeros(q.shape), np.full(q.shape[:2], -math.inf)
    group, row = q.shape[1] // cache.k.shape[1], 0
    for s, (length, n) in enumerate(zip(lengths, counts)):
        k, v, there = cache.sequence(pages[s], max(0, length))
        j = np.arange(max(0, length))
        for i in range(n):
            at = length - n + i
            seen = ((j <= at) if causal else True) & ((j > at - window) if window else True) & (j >= 0)
            if since is not None:
                seen = seen & (j >= since[row + i])
            if until is not None:
                seen = seen & (j < until[row + i])
            if prefix is not None:
                seen = seen | (j < prefix[s])
            seen = seen & there
            if np.any(seen):
                for h in range(q.shape[1]):
                    z = scale * (k[seen, h // group] @ q[row + i, h])
                    if cap:
                        z = cap * np.tanh(z / cap)
                    if slopes is not None:
                        z = z - float(slopes[h]) * np.abs(at - j[seen])
                    p = np.exp(z - np.max(z))
                    vs = v[seen, h // group]
                    o[row + i, h] = p @ vs / p.sum()
                    a[row + i, h] = p @ np.abs(vs) / p.sum()
                    lse[row + i, h] = np.max(z) + math.log(p.sum()) if np.isfinite(p.sum()) and not np.isnan(vs).any() else math.nan
        row += n
    return o, lse, a


KEPT = 1 << 30       # added to the number of a block that a list holds and must not write to


def block(entry):
    return int(entry) - KEPT if entry >= KEPT else int(entry)


class Pool:
    """Which lists hold which of n blocks, call by call and list by list."""

    def __init__(self, n):
        self.counts, self.missing = [0] * n, 0

    def _held(self, b):
        return 0 <= b < len(self.counts)

    def count(self, *tables):
        self.counts = [0] * len(self.counts)
        for t in tables:
            for b in np.asarray(t).flatten().tolist():
                if self._held(block(b)):
                    self.counts[block(b)] += 1

    def grow(self, pages, lengths, new):
        """The copies to be made, as [(src, dst)]; pages is changed."""
        past = []                        # blocks past the tokens of lists that grow, which other lists hold too
        for row, length, n in zip(pages, lengths, new):
            length, n = max(0, int(length)), max(0, int(n))
            for b in range((length + 63) // 64, min(len(row), (length + n + 63) // 64)) if n else ():
                if self._held(block(row[b])):
                    row[b] = row[b] if self.counts[block(row[b])] > 1 else block(row[b])
                    past += [(row, b)] if self.counts[block(row[b])] > 1 else []
        for row, b in past:
            self.counts[block(row[b])] -= 1
            row[b] = -1
        free = [b for b, c in enumerate(self.counts) if c == 0][::-1]
        moves, self.missing = [], 0
        left = dict()                    # holders of an open block that have not been asked to part with it
        stay = []                        # lists whose open block is the one that it was

        def take():
            if free:
                self.counts[free[-1]] = 1
                return free.pop()
            self.missing += 1
            return -1

        for row, length, n in zip(pages, lengths, new):
            length, n, width = max(0, int(length)), max(0, int(n)), len(row)
            at = length // 64
            if n and length % 64 and at < width and self._held(block(row[at])):
                old = block(row[at])
                got = -1
                if left.setdefault(old, self.counts[old]) > 1:
                    left[old] -= 1
                    got = take()
                if got >= 0:
                    self.counts[old] -= 1
                    row[at] = got
                    moves.append((old, got))
                else:
                    stay.append((row, at))
            for b in range((length + 63) // 64, min(width, (length + n + 63) // 64)):
                if row[b] < 0:
                    row[b] = take()
        for row, at in stay:
            b = block(row[at])
            row[at] = b + KEPT if self.counts[b] > 1 else b
        return moves

    def drop(self, row, keep=lambda b: False):
        for b in range(len(row)):
            if row[b] >= 0 and not keep(b):
                old = block(row[b])
                if self._held(old) and self.counts[old] > 0:
                    self.counts[old] -= 1
                row[b] = -1

    def fork(self, pages, lengths, parents, children, to, to_lengths):
        same = to is pages
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < len(pages) and 0 <= c < len(to)) or c in children[i + 1:] or same and c in parents:
                continue
            row = [int(b) if self._held(block(b)) and 64 * x < lengths[p] else -1 for x, b in enumerate(pages[p])]
            for b in row:
                if b >= 0:
                    self.counts[block(b)] += 1
            for b in to[c]:
                if self._held(block(b)) and self.counts[block(b)] > 0:
                    self.counts[block(b)] -= 1
            to[c] = row + [-1] * (len(to[c]) - len(row))
            to_lengths[c] = lengths[p]

    def compact(self, tables, most):
        free = [b for b, c in enumerate(self.counts) if c == 0]
        used = [b for b, c in enumerate(self.counts) if c > 0][::-1]
        moves = [(a, b) for a, b in zip(used, free) if b < a][:most]
        for a, b in moves:
            self.counts[b], self.counts[a] = self.counts[a], 0
        for t in tables:
            old = t.copy()
            for a, b in moves:
                t[old == a] = b
                t[old == a + KEPT] = b + KEPT
        return moves
