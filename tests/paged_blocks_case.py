"""Plain 64-bit forms of the operators around a paged cache: head norms with rotation, block means, block selection, pages."""
from __future__ import annotations

import numpy as np

from paged_case import bf16_values


def norm_rope(bits, weight, positions, inv_freq, eps, offset, interleaved):
    """Heads [N, heads, D] (BF16 bits) normalised and rotated in 64 bits, and the largest error of a result.

    FP32: the sum of squares of 8 values a lane and 4 or 5 steps over the lanes is off by 13 2^-24 of itself, its root by half of
    that; the mean, root, quotient, two products and the weight's sum add 2^-24 each; sine and cosine two units and an argument off by pi
    2^-24; the rotation's products and sum three more: below 32 2^-24 = 2^-19 of |a| + |b| in all. The result is rounded to BF16: 2^-8 of
    itself, 2^-134 at least."""
    x = bf16_values(bits).astype(np.float64)
    D = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    y = y * ((weight.astype(np.float64) if weight is not None else np.ones(D)) + np.float64(np.float32(offset)))
    out, size = y.copy(), np.abs(y)
    if inv_freq is not None:
        half = len(inv_freq)
        angle = np.asarray(positions, np.float64)[:, None, None] * inv_freq.astype(np.float64)
        c, s = np.cos(angle), np.sin(angle)
        ia, ib = (np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if interleaved else (np.arange(half), np.arange(half, 2 * half))
        a, b = y[..., ia], y[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    return out, 2.0**-8 * np.abs(out) + 2.0**-19 * size + 2.0**-134


def mean_codes(total, rows):
    """INT8 codes and FP32 scale of 64-bit sums [..., D] over `rows` rows."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        amax = np.where(np.isfinite(total).all(-1), np.abs(total).max(-1), np.inf)
        step = amax * (1.0 / 127.0)
        tell = (amax > 0) & np.isfinite(amax)
        inv = np.where(tell, 1.0 / step, 0.0)
        codes = np.where(tell[..., None], np.clip(np.rint(np.where(np.isfinite(total), total, 0) * inv[..., None]), -127, 127), 0)
        return codes.astype(np.int8), (step / rows).astype(np.float32)


def block_means(case, block):
    """{(sequence, block): (codes [Hkv, D], scales [Hkv])} of the blocks that the case's new rows touch and whose page is there."""
    out = {}
    for b, (t, h) in enumerate(case.seqs):
        if t == 0:
            continue
        K = case.stored(b)[0]
        for blk in range(h // block, (h + t - 1) // block + 1):
            rows = K[blk * block:min((blk + 1) * block, h + t)]
            if case.present(b, np.array([blk * block]))[0]:
                with np.errstate(invalid="ignore"):
                    out[b, blk] = mean_codes(rows.sum(0), len(rows))
    return out


def select(q, codes, scales, there, pos, block, first, local, top):
    """The list of one token and KV head: q [G, D] 64-bit query heads, codes [blocks, D], scales and `there` [blocks]."""
    own = pos // block
    u = mean_codes(q.sum(0), 1)[0].astype(np.int64)
    dots = codes.astype(np.int64) @ u
    with np.errstate(invalid="ignore", over="ignore"):
        score = np.where(np.isinf(scales), np.float32(np.inf), scales * dots.astype(np.float32)).astype(np.float32)
    middle = [c for c in range(first, own - local + 1) if there[c]]
    middle.sort(key=lambda c: (-score[c], c))
    chosen = sorted(set(range(min(first, own + 1))) | set(middle[:top]) | set(range(max(0, own - local + 1), own + 1)))
    return np.array(chosen + [-1] * (first + local + top - len(chosen)), np.int32)


class Pages:
    """The table and the counts, kept one entry at a time."""

    def __init__(self, table, refs, page):
        self.table, self.refs, self.page = table.copy(), refs.copy(), page
        self.B, self.width = table.shape

    def held(self, e):
        return 0 <= e < len(self.refs)

    def free(self):
        return [int(p) for p in np.flatnonzero(self.refs == 0)]

    def reserve(self, starts, history):
        free = self.free()
        granted = np.zeros(self.B, np.int32)
        for b in range(self.B):
            t, h = int(starts[b + 1]) - int(starts[b]), int(history[b])
            if starts[b] < 0 or t <= 0 or h < 0:
                continue
            end = self.width * self.page
            for e in range(h // self.page, min((h + t - 1) // self.page + 1, self.width)):
                if not self.held(self.table[b, e]):
                    if free:
                        self.table[b, e] = free.pop(0)
                        self.refs[self.table[b, e]] = 1
                    else:
                        end = min(end, e * self.page)
            granted[b] = max(0, min(t, end - h))
        return granted

    def drop(self, b, e):
        if self.held(self.table[b, e]):
            self.refs[self.table[b, e]] -= 1
        self.table[b, e] = -1

    def release(self, sequences, keep):
        for b, rows in zip(sequences, keep):
            if 0 <= b < self.B and rows >= 0:
                for e in range(-(-int(rows) // self.page), self.width):
                    self.drop(b, e)

    def fork(self, parents, children, history):
        history = history.copy()
        free = self.free()
        src, dst = (np.full(len(parents), -1, np.int32) for _ in range(2))
        work = []
        for i, (p, c) in enumerate(zip(parents, children)):
            if 0 <= p < self.B and 0 <= c < self.B and c not in parents and c not in children[:i]:
                rows = max(0, int(history[p]))
                whole = min(rows // self.page, self.width)
                if rows % self.page and whole < self.width and self.held(self.table[p, whole]) and free:
                    src[i], dst[i] = self.table[p, whole], free.pop(0)
                else:
                    rows = whole * self.page
                work.append((i, p, c, rows, whole))
        for i, p, c, rows, whole in work:
            for e in range(self.width):
                self.drop(c, e)
                entry = self.table[p, e] if e < whole else dst[i] if e == whole else -1
                self.table[c, e] = entry
                if self.held(entry):
                    self.refs[entry] += 1
            history[c] = rows
        return history, src, dst

    def compact(self, n):
        src, dst = (np.full(n, -1, np.int32) for _ in range(2))
        moved = 0
        used, free = [int(p) for p in np.flatnonzero(self.refs != 0)][::-1], self.free()
        for a, b in list(zip(used, free))[:n]:
            if b > a:
                break
            src[moved], dst[moved] = a, b
            moved += 1
        for a, b in zip(src[:moved], dst[:moved]):
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        return src, dst, moved
