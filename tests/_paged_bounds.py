"""How far each output element of the paged attention may be off, from the
terms of its own query (tests/_paged.py's `attention_bound` takes the largest
of a whole sequence), and what a kernel with a mistake in it would give.

With x = q·log2 e/√hd, s_i = x·k_i and the softmax's p_i, an output is off by
    sum_i p_i (v_i - out) e_i  +  what the sums and the parts of p add.
 - Each element of x has three roundings of 2^-24 (the constant, its product, the
   sum of its parts) beside half a step of the high part and half of the low
   part, 2^-11 each, and a low part that ends at f16's step of 2^-24: half of it is
   2^-25 (2^-39 of the largest element where a power of two brings it there).
 - s_i is a sum of hd exact products in f32, then meets the key's scale, the
   reference and, where the reference moves, the way that it goes.  The
   reference itself is the same for all keys of a row and cancels.
 - p_i = 2^(s_i - m) takes 2^-22, its parts 2^-22 and, below f16's normal numbers,
   2^-25 where the row's largest product with a value scale is 2^8 or more.
`hard` adds all of it up with every rounding at its largest and is never
passed.  `rms` takes roundings as independent of each other, each at its
largest, and holds the root of the mean square over a batch."""
from __future__ import annotations

import numpy as np

from _paged import Batch, Pool, random_rows

LN2 = float(np.log(2.0))
STEP = 2.0 ** -24  # half a step of f32, relative


def terms(q, k, v, past):
    """(outputs, hard, rms) [tokens, heads, hd] for q over the positions k, v [positions, kv, hd], in float64."""
    tokens, heads, hd = q.shape
    want, hard, rms = np.empty(q.shape), np.empty(q.shape), np.empty(q.shape)
    for t in range(tokens):
        n = past + t + 1
        for h in range(heads):
            kk, vv = k[:n, h * k.shape[1] // heads], v[:n, h * k.shape[1] // heads]
            x = q[t, h].astype(np.float64) / (LN2 * np.sqrt(hd))
            top = np.abs(x).max()
            low = 2.0 ** -25 if 0.0625 <= top <= 32768 else top * 2.0 ** -39
            s = kk @ x
            p = np.exp2(s - s.max())
            p /= p.sum()
            out = p @ vv
            size = np.abs(vv).max(1)  # of a value row: its scale times the format's largest
            logs = np.log2(size[size > 0])
            room = 14 + (logs.max() - logs.min() if logs.size else 0)
            seen = STEP * (2 * np.abs(s) + 2 * (s.max() - s + room))  # the score's places and the exponent's, twice each
            apart, lost = vv - out, 2.0 ** -33 * (p * size).max()
            off = np.abs(kk) @ np.abs(x) * (2.0 ** -22 + (hd + 3) * STEP) + low * np.abs(kk).sum(1) + seen
            mass = p @ np.abs(vv) + np.abs(out)
            hard[t, h] = 1.01 * ((p * (LN2 * off + 2.0 ** -22)) @ np.abs(apart) + mass * (2.0 ** -22 + (n + 8) * STEP) + n * lost)
            query = np.hypot(x * 2.0 ** -22, low)  # of each element, the same for all keys
            keys = p * np.hypot(LN2 * np.hypot(np.sqrt(hd * (kk * kk @ (x * x))) * 2 * STEP, seen), 2.0 ** -22)
            walk = np.sqrt((p * p) @ (vv * vv))
            rms[t, h] = np.sqrt(LN2 ** 2 * (query * query) @ ((kk * p[:, None]).T @ apart) ** 2 + (keys * keys) @ (apart * apart)
                                + (walk * 2.0 ** -22) ** 2 + (walk + np.abs(out)) ** 2 * (n + 16) * STEP ** 2 + n * lost * lost)
            want[t, h] = out
    return want, hard, rms


def excess(got, want, hard, rms):
    """(largest error over `hard`, root mean square over that of `rms`): both at most 1 for a sound kernel."""
    d = np.abs(got - want)
    return float((d / hard).max()), float(np.sqrt((d * d).mean() / (rms * rms).mean()))


def case(rng, fmt, heads, kv, hd, page, seqs):
    """A filled cache of random rows, its batch, and queries [tokens, heads, hd]."""
    batch = Batch(rng, seqs, page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    batch.fill(rng, pool)
    batch.put(pool, *np.stack([random_rows(rng, kv, hd) for _ in range(batch.tokens)], 1))
    return pool, batch, (1.5 * rng.standard_normal((batch.tokens, heads, hd))).astype(np.float32)


def restated(q, k, v, past, *, query_parts=2, p_parts=2, drop=None, peak=8.0):
    """The kernels' arithmetic, with as many f16 parts of queries and probabilities as given and without the key that
    `drop` names (0 the first, -1 the newest that a query sees), sums in float64."""
    out = np.empty(q.shape)
    f16 = lambda a: a.astype(np.float16).astype(np.float64)  # noqa: E731
    for t in range(q.shape[0]):
        n = past + t + 1
        for h in range(q.shape[1]):
            kk, vv = k[:n, h * k.shape[1] // q.shape[1]], v[:n, h * k.shape[1] // q.shape[1]]
            x = (q[t, h] * np.float32(1 / (LN2 * np.sqrt(q.shape[2])))).astype(np.float64)
            parts = f16(x) + (f16(x - f16(x)) if query_parts == 2 else 0.0)
            s = kk @ parts
            if drop is not None:
                s[drop] = -np.inf
            b = np.abs(vv).max(1) / 127
            b = np.where(b > 0, b, 1.0)
            pb = np.exp2(s + np.log2(b) - (s + np.log2(b)).max() + peak)
            kept = f16(pb) + (f16(pb - f16(pb)) if p_parts == 2 else 0.0)
            out[t, h] = kept @ (vv / b[:, None]) / (pb / b).sum()
    return out
