"""Plain restatements of the paged cache for its tests: the quantiser, the
blocks' layout element by element, and attention in float64."""
from __future__ import annotations

import numpy as np

TOP = {"i8": np.float32(127), "f8": np.float32(448)}
SIZE = {"f16": 2, "i8": 1, "f8": 1}


def e4m3_table() -> np.ndarray:
    """The value of every e4m3 byte: 1 sign, 4 exponent (bias 7), 3 mantissa bits, 0x7f and 0xff NaN."""
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b & 128, -v, v)


E4M3 = e4m3_table()


def to_e4m3(y: np.ndarray) -> np.ndarray:
    """The bytes nearest to y (|y| <= 448), ties to the even byte."""
    grid = E4M3[:127]
    a = np.abs(y.astype(np.float64))
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def quantise(x: np.ndarray, fmt: str):
    """(bit patterns, scales or None) of float32 rows x [..., hd]."""
    if fmt == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16), None
    fine = np.isfinite(x).all(-1)
    with np.errstate(invalid="ignore", over="ignore"):
        largest = np.abs(x).max(-1)
        scale = np.clip(largest * (np.float32(1) / TOP[fmt]), np.float32(2.0 ** -40), np.float32(2.0 ** 60)).astype(np.float32)
        y = np.clip(x / scale[..., None], -TOP[fmt], TOP[fmt])
    y = np.where(fine[..., None], y, np.float32(0))
    bits = np.rint(y).astype(np.int8).view(np.uint8) if fmt == "i8" else to_e4m3(y)
    return bits, np.where(fine, scale, np.float32(np.nan))


def dequantise(bits: np.ndarray, scale, fmt: str) -> np.ndarray:
    if fmt == "f16":
        return bits.view(np.float16).astype(np.float64)
    v = bits.view(np.int8).astype(np.float64) if fmt == "i8" else E4M3[bits]
    return v * scale.astype(np.float64)[..., None]


def block_bytes(fmt: str, hd: int) -> int:
    return 32 * hd * SIZE[fmt] + (0 if fmt == "f16" else 128)


class Pool:
    """A cache's bytes on the host, addressed position by position."""

    def __init__(self, fmt, kv, hd, page, n_pages, fill=0xFF):
        self.fmt, self.kv, self.hd, self.page, self.n_pages = fmt, kv, hd, page, n_pages
        self.bytes = np.full((n_pages, kv, page // 16, block_bytes(fmt, hd)), fill, np.uint8)
        size, d = SIZE[fmt], np.arange(hd)
        e, m = 16 // size, 4 // size
        i = np.arange(16)[:, None]
        self.key_at = (d // e * 16 + i) * e + d % e  # [position, element]
        self.value_at = ((d // (16 * m) * 4 + i // 4) * 16 + d % 16) * m * 4 + d // 16 % m * 4 + i % 4

    def put(self, page, at, k, v):
        """Rows k and v [kv, hd] (float32) at position `at` of `page`."""
        b, i, n = at // 16, at % 16, 16 * self.hd * SIZE[self.fmt]
        for part, (x, where) in enumerate(((k, self.key_at), (v, self.value_at))):
            bits, scale = quantise(x, self.fmt)
            for h in range(self.kv):
                block = self.bytes[page, h, b]
                block[part * n:(part + 1) * n].view(bits.dtype)[where[i]] = bits[h]
                if scale is not None:
                    block[2 * n:].view(np.float32)[16 * part + i] = scale[h]

    def get(self, page, at):
        """The rows (k, v) [kv, hd] that position `at` of `page` holds, in float64."""
        b, i, n = at // 16, at % 16, 16 * self.hd * SIZE[self.fmt]
        out = []
        for part, where in enumerate((self.key_at, self.value_at)):
            raw = self.bytes[page, :, b, part * n:(part + 1) * n].copy().view(np.uint16 if self.fmt == "f16" else np.uint8)
            scale = None if self.fmt == "f16" else self.bytes[page, :, b, 2 * n:].copy().view(np.float32)[:, 16 * part + i]
            out.append(dequantise(raw[:, where[i]].copy(), scale, self.fmt))
        return out


class Batch:
    """Sequences of (past, new) positions with their pages, drawn out of order from a cache of `spare` more pages."""

    def __init__(self, rng, seqs, page, spare=3):
        self.past, self.new = [p for p, _ in seqs], [n for _, n in seqs]
        need = [-(-(p + n) // page) for p, n in seqs]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages).tolist()
        self.pages = [[order.pop() for _ in range(n)] for n in need]
        self.page, self.tokens = page, sum(self.new)
        self.rows = [(s, p + i) for s, (p, n) in enumerate(seqs) for i in range(n)]  # of each token

    def fill(self, rng, pool: Pool, scale=1.0):
        """Random rows at every past position."""
        for s, n in enumerate(self.past):
            for at in range(n):
                pool.put(self.pages[s][at // self.page], at % self.page, *random_rows(rng, pool.kv, pool.hd, scale))

    def put(self, pool: Pool, k, v):
        for t, (s, at) in enumerate(self.rows):
            pool.put(self.pages[s][at // self.page], at % self.page, k[t], v[t])

    def gather(self, pool: Pool, s: int):
        """(k, v) [positions, kv, hd] of sequence s, in float64."""
        got = [pool.get(self.pages[s][at // self.page], at % self.page) for at in range(self.past[s] + self.new[s])]
        return np.stack([g[0] for g in got]), np.stack([g[1] for g in got])


def random_rows(rng, kv, hd, scale=1.0):
    size = np.exp(0.5 * rng.standard_normal((2, kv, 1)))
    return (scale * size * rng.standard_normal((2, kv, hd))).astype(np.float32)


def attention(q, k, v, past):
    """q [tokens, heads, hd] over k, v [positions, kv, hd], in float64: what a query does not see is left out."""
    heads, kv = q.shape[1], k.shape[1]
    out = np.empty(q.shape)
    for t in range(q.shape[0]):
        n = past + t + 1
        for h in range(heads):
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[:n, h * kv // heads] @ q[t, h].astype(np.float64) / np.sqrt(q.shape[2])
                p = np.exp(s - s.max())
                out[t, h] = p @ v[:n, h * kv // heads] / p.sum()
    return out


def attention_bound(q, k, v):
    """How far an output may be off.  The parts of a query are off by 2^-22 of its elements (two f16 roundings of half a
    step, 2^-11 each) and its products with a key are summed in f32, so a score by A·(2^-22 + hd·2^-24) with
    A = sum |q||k| / sqrt(hd); the probabilities follow it, once in the sum and once in the quotient, and are themselves
    kept to 2^-22 with a few f32 roundings (exponential, scales, quotient: 16·2^-24 in all); the sums over n keys are
    off by n·2^-24 at most."""
    n, hd = k.shape[0], q.shape[2]
    size = np.abs(q).max(1).max(0).astype(np.float64) @ np.abs(k).max(1).max(0) / np.sqrt(hd)
    return np.abs(v).max() * (2 * size * (2.0 ** -22 + hd * 2.0 ** -24) + 2.0 ** -22 + (16 + 2 * n) * 2.0 ** -24)
