"""Attention of trees whose kernels other tests do not reach: wide tiles of every format and head size, and batches of which
one part takes narrow tiles and another wide ones.  Bounds and caches as in tests/test_gpu_attn_tree.py."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import ancestors, chain, random_tree
from _paged import Batch, Pool, attention_bound, random_rows
from test_gpu_attn_tree import check, decoded, plan_of, setup
from test_gpu_paged import attend

pytestmark = pytest.mark.gpu

FORMATS = [(fmt, hd) for fmt in ("f16", "i8", "f8") for hd in (64, 128, 256)]


@pytest.mark.parametrize("fmt,hd", FORMATS)
def test_more_rows_than_narrow_tiles_take(hip, fmt, hd):
    """More than 512 packed rows of a sequence are wide in any batch: pasts within, at and behind a tile's keys."""
    rng = np.random.default_rng(hd)
    for past, n in ((0, 70), (64, 65), (100, 90), (129, 67)):
        print("wide", fmt, hd, past, n, flush=True)
        trees = [random_tree(rng, n, width=3)]
        batch, pool, q = setup(rng, fmt, 1, hd, 32, [past], trees, 8)
        q[::3] *= np.float32(2.0 ** -9)  # queries that get a factor, beside others that do not
        check(hip, pool, batch, 8, q, trees)


@pytest.mark.parametrize("fmt,hd", FORMATS)
def test_small_trees_beside_a_prompt(hip, fmt, hd):
    """Of one plan a prompt of 520 rows and a tree of 516 in wide tiles, trees, a single token and nothing in narrow ones."""
    rng = np.random.default_rng(hd + 1)
    trees = [random_tree(rng, 9, width=3), chain(130), random_tree(rng, 4), chain(0), chain(1), random_tree(rng, 129, width=3),
             random_tree(rng, 14, width=4), chain(5)]
    past = [40, 20, 0, 7, 100, 33, 63, 31]
    batch, pool, q = setup(rng, fmt, 2, hd, 48, past, trees, 8)
    check(hip, pool, batch, 8, q, trees, extra=(4, 8))


@pytest.mark.parametrize("fmt,hd", FORMATS)
def test_values_that_are_not_finite_beside_a_prompt(hip, fmt, hd):
    """One row of each sequence holds an infinite value: in f16 only the queries that see it get NaN, and only in that element; in
    8 bits the whole row is NaN."""
    rng = np.random.default_rng(hd + 2)
    trees = [random_tree(rng, 9, width=3), chain(130), random_tree(rng, 129, width=3), random_tree(rng, 3)]
    past = [40, 20, 33, 5]
    batch, pool, q = setup(rng, fmt, 1, hd, 32, past, trees, 4)
    plan = plan_of(hip, pool, batch, 4, trees)
    clean, at = attend(hip, pool, batch, 4, q, plan=plan), [4, 77, 60, 1]
    for s, a in enumerate(at):
        k, v = random_rows(rng, 1, hd)
        v[0, 3] = np.inf
        pool.put(batch.pages[s][(past[s] + a) // 32], (past[s] + a) % 32, k, v)
    got, row = attend(hip, pool, batch, 4, q, plan=plan), 0
    for s, t in enumerate(trees):
        sees = ancestors(t)[:, at[s]]
        for i in range(len(t)):
            x = got[row + i]
            if not sees[i]:
                assert np.array_equal(x, clean[row + i]), (s, i)
            elif fmt == "f16":
                assert np.isnan(x[:, 3]).all() and np.isfinite(np.delete(x, 3, 1)).all(), (s, i)
            else:
                assert np.isnan(x).all(), (s, i)
        row += len(t)


@pytest.mark.parametrize("fmt,hd,kv,heads,seqs,new,past", [
    ("f16", 64, 8, 32, 12, 64, 2500), ("f16", 128, 8, 32, 12, 64, 2500), ("f16", 256, 2, 8, 40, 44, 2500),
    ("i8", 64, 8, 32, 12, 128, 2000), ("i8", 128, 8, 32, 12, 96, 2000), ("f8", 128, 8, 32, 12, 96, 2000),
    ("i8", 256, 2, 16, 24, 56, 3000), ("f8", 256, 2, 16, 24, 56, 3000)])
def test_few_rows_beside_wide_trees(hip, fmt, hd, kv, heads, seqs, new, past):
    """Batches whose trees are wide by their work, with sequences of up to 16 rows, which stay narrow."""
    print("wide by work", fmt, hd, flush=True)
    rng = np.random.default_rng(hd + new)
    group = heads // kv
    few = 16 // group
    trees = [random_tree(rng, new, width=4) for _ in range(seqs)]
    trees[1:1] = [chain(1), random_tree(rng, few, width=2), chain(few)]
    trees.append(chain(1))
    pasts = [int(n) for n in rng.integers(past // 2, past, len(trees))]
    batch = Batch(rng, [(p, len(t)) for p, t in zip(pasts, trees)], 64)
    pool = Pool(fmt, kv, hd, 64, batch.n_pages)
    part = 16 * hd * (2 if fmt == "f16" else 1)
    if fmt == "f16":
        pool.bytes[:] = rng.standard_normal(pool.bytes.size // 2, np.float32).astype(np.float16).view(np.uint8).reshape(pool.bytes.shape)
    else:
        pool.bytes[..., :2 * part] = rng.integers(0, 256, pool.bytes[..., :2 * part].shape, np.uint8)
        if fmt == "f8":
            pool.bytes[..., :2 * part] &= 0xBF  # (below 2, and no NaN)
        scales = np.exp(0.4 * rng.standard_normal(pool.bytes[..., 2 * part:].shape[:-1] + (32,))) / (64 if fmt == "i8" else 1)
        pool.bytes[..., 2 * part:] = np.ascontiguousarray(scales.astype(np.float32)).view(np.uint8)
    q = rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32)
    got, row = attend(hip, pool, batch, heads, q, plan=plan_of(hip, pool, batch, heads, trees)), 0
    for s, t in enumerate(trees):
        n = len(t)
        if s < 5 or s == len(trees) - 1:
            k, v = decoded(pool, batch.pages[s], pasts[s] + n)
            seen = np.concatenate([np.ones((n, pasts[s]), bool), ancestors(t)], 1)
            qs = q[row:row + n].astype(np.float64).reshape(n, kv, group, hd)
            for h in range(kv):
                a = qs[:, h].reshape(n * group, hd) @ k[:, h].T / np.sqrt(hd)
                a = np.where(np.repeat(seen, group, 0), a, -np.inf)
                p = np.exp(a - a.max(1, keepdims=True))
                want = ((p / p.sum(1, keepdims=True)) @ v[:, h]).reshape(n, group, hd)
                mine = got[row:row + n, h * group:(h + 1) * group]
                bound = attention_bound(q[row:row + n, h * group:(h + 1) * group], k[:, h:h + 1], v[:, h:h + 1])
                assert np.abs(mine - want).max() <= bound, (s, h)
        row += n
