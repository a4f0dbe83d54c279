"""64-bit results of chosen tokens of a paged-cache problem, with an error bound per element that counts every key by its
own weight: a key without weight loosens nothing."""
from __future__ import annotations

import numpy as np

from paged_case import bf16_bits, bf16_values


def bound(case, tokens=None, kv_heads=None, dropped=()):
    """(packed token, KV head, out [G, D], tol [G, D]) of every chosen one. `dropped`: rows of the sequences that the
    result is computed without (a planted mistake).

    Scores are off by d_j: 2^-11 of sum |q k| scale where an INT8 key is rounded to FP16 (BF16 keys are exact), 2^-16 of
    it for FP32 sums of up to 256 products, 2^-22 of the scores for the exponent's argument, 2^-11 for P in FP16 and 2^-20
    for the exponential. With weights p' = p e^delta, |delta_j| <= d_j, the output moves by
    sum p_j (e^delta_j - 1) (v_j - o) / sum p_j e^delta_j; the same with every delta_j less the heaviest key's, whose term
    is then zero; and by 2 max |v| at most. Values: 2^-11 of p_j |v_j| where INT8 rows are rounded; FP32 sums 2^-24 for each 32 keys and 64 more.
    FP16's steps: p is held to 2^-33 of the heaviest, an INT8 weight p_j s_j to 2^-32 of the largest, a BF16 value to 2^-19 of
    the largest of its eight, seen keys only. The result is rounded to BF16, 2^-8 of itself at most."""
    i8 = case.kv == "i8"
    G = case.Hq // case.Hkv
    stored = {}
    for n in (range(case.N) if tokens is None else tokens):
        b = int(np.searchsorted(case.starts, n, side="right")) - 1
        if not 0 <= b < case.B or n >= case.starts[b + 1]:
            continue
        t, h = case.seqs[b]
        if b not in stored:
            stored[b] = case.stored(b)
        K, V = stored[b]
        pos = h + n - int(case.starts[b])
        rows = np.arange(pos + 1)
        see = case.present(b, rows)
        if case.window:
            see &= (pos - rows < case.window) | (rows < case.sinks)
        see &= ~np.isin(rows, list(dropped))
        rows = rows[see]
        q = bf16_values(case.q[n]).astype(np.float64).reshape(case.Hkv, G, case.D)
        for hh in (range(case.Hkv) if kv_heads is None else kv_heads):
            if len(rows) == 0:
                yield n, hh, np.zeros((G, case.D)), np.zeros((G, case.D))
                continue
            k, v = K[rows, hh], V[rows, hh]
            av = np.abs(v)
            s = (q[hh] @ k.T) * case.scale  # [G, rows]
            size = (np.abs(q[hh]) @ np.abs(k).T) * case.scale
            top = s.max(-1, keepdims=True)
            heaviest = s.argmax(-1)
            d = size * ((2.0**-11 if i8 else 0.0) + 2.0**-16) + 2.0**-22 * (np.abs(s) + np.abs(top)) + 2.0**-11 + 2.0**-20
            log_p = s - top
            log_p -= np.log(np.exp(log_p).sum(-1, keepdims=True))
            p = np.exp(log_p)
            out = p @ v

            def moved(d):
                # p (e^d - 1) without p underflowing before e^d grows; |v - o| <= |v| + |o|
                up = np.where(d < 1, p * np.expm1(np.minimum(d, 1)), np.exp(np.minimum(log_p + d, 300)))
                return (up @ av + up.sum(-1, keepdims=True) * np.abs(out)) / np.maximum((p * np.exp(-d)).sum(-1, keepdims=True), 1e-100)
            each = np.arange(G)
            far = d + d[each, heaviest][:, None]
            far[each, heaviest] = 0
            weight = p @ av
            fp16 = p.max(-1, keepdims=True) * 2.0**-33 * av.sum(0)
            if i8:
                amax = av.reshape(len(rows), -1, 64).max(-1)  # [rows, groups]
                largest = np.stack([(x[:, None] * amax).max(0) for x in p])
                fp16 = fp16 + 2.0**-32 * len(rows) * np.repeat(largest, 64, -1)
            else:
                fp16 = fp16 + 2.0**-19 * np.repeat(p @ av.reshape(len(rows), -1, 8).max(-1), 8, -1)
            move = np.minimum(np.minimum(moved(d), moved(far)), 2 * av.max(0))
            tol = 2.0**-8 * np.abs(out) + move + fp16 + 1e-38
            tol += weight * ((2.0**-11 if i8 else 0.0) + 2.0**-24 * (len(rows) / 32 + 64))
            yield n, hh, out, tol


def check_bound(case, bits, tokens=None, kv_heads=None):
    """The chosen elements within their bounds, every token of a sequence written, all others untouched."""
    own = np.zeros(case.N, bool)
    own[case.starts[0]:case.starts[-1]] = True
    assert (bits[~own] == 0xCDCD).all(), "rows of no sequence were written"
    got = bf16_values(bits).astype(np.float64)
    assert np.isfinite(got[own]).all(), f"{(~np.isfinite(got[own])).sum()} results are not finite"
    G = case.Hq // case.Hkv
    worst = 0.0
    for n, hh, o, tol in bound(case, tokens, kv_heads):
        err = np.abs(got[n, hh * G:(hh + 1) * G] - o)
        bad = ~(err <= tol)
        assert not bad.any(), f"token {n}, KV head {hh}: {bad.sum()} of {bad.size} outside, worst {(err / tol).max():.3g} of the bound"
        worst = max(worst, float((err / np.maximum(tol, 1e-300)).max()))
    print(f"worst {worst:.3f} of the bound", flush=True)


def needles(c, b, rows, gain=13.0):
    """The sequence's rows `rows` stand `gain` above its others in every score."""
    rows = [r for r in set(rows) if 0 <= r < c.k[b].shape[0]]
    c.q[c.starts[b]:c.starts[b + 1], :, 1] = bf16_bits(np.float32(8.0))
    c.k[b][:, :, 1] = 0
    c.k[b][rows, :, 1] = bf16_bits(np.float32(gain / (8.0 * c.scale)))


def borders(t, h):
    """Rows where a chunk, a unit, a key tile, the history or the sequence begins or ends."""
    n = t + h
    r = [0, 31, 32, 63, 127, 128, 500, 511, 512, n // 2 // 128 * 128 - 1, n // 2 // 128 * 128, n // 3, h - 1, h, n - 2, n - 1]
    return r
