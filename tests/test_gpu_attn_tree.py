"""GPU parity of bch_attention_paged on plans with trees against attention along each token's own path in float64, inside the
bounds of tests/_paged.py.  Free places of the caches hold NaN in every format."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import ancestors, as_given, chain, random_tree, tree_attention
from _paged import Batch, Pool, attention_bound, dequantise, random_rows
from bobcat_amd.backend import Hip
from test_gpu_paged import attend

pytestmark = pytest.mark.gpu


def setup(rng, fmt, kv, hd, page, past, trees, heads, scale=1.0):
    batch = Batch(rng, [(p, len(t)) for p, t in zip(past, trees)], page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    batch.fill(rng, pool, scale)
    batch.put(pool, *np.stack([random_rows(rng, kv, hd, scale) for _ in range(batch.tokens)], 1))
    return batch, pool, rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32)


def plan_of(hip, pool, batch, heads, trees, given=None):
    plan = hip.kv_plan(pool.fmt, pool.kv, pool.hd, pool.page, pool.n_pages, heads)
    plan.set(batch.past, batch.new, batch.pages, parents=as_given(trees) if given is None else given)
    return plan


def check(hip, pool, batch, heads, q, trees, plan=None, extra=(0, 0)):
    got = attend(hip, pool, batch, heads, q, plan=plan or plan_of(hip, pool, batch, heads, trees), extra=extra)
    row = 0
    for s, t in enumerate(trees):
        n = len(t)
        if n:
            k, v = batch.gather(pool, s)
            want = tree_attention(q[row:row + n], k, v, batch.past[s], t)
            off = np.abs(got[row:row + n] - want).max()
            assert off <= attention_bound(q[row:row + n], k, v), (s, off)
        row += n
    return got


def mixed(rng, sizes, roots=1):
    return [random_tree(rng, n, roots=roots) for n in sizes]


# Past positions around words of 32 and pages, trees of one token to several words, roots of their own, chains beside trees.
CASES = {
    "small": ([5, 31, 32, 33, 0], lambda r: mixed(r, [7, 2, 9, 1, 5]), 16),
    "forests": ([0, 63, 40], lambda r: mixed(r, [6, 11, 3], roots=3), 32),
    "wide trees": ([90, 17], lambda r: mixed(r, [70, 45]), 48),
    "beside chains": ([20, 100, 7, 64], lambda r: [chain(5), random_tree(r, 12), chain(40), chain(0)], 16),
    "long past": ([700, 333], lambda r: mixed(r, [3, 33]), 64),
}


@pytest.mark.parametrize("fmt", ["f16", "i8", "f8"])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (3, 3, 64), (4, 1, 128), (8, 2, 256)])
@pytest.mark.parametrize("name", CASES)
def test_trees(hip, fmt, heads, kv, hd, name):
    print("tree", fmt, heads, kv, hd, name, flush=True)
    rng = np.random.default_rng(len(name) + hd)
    past, trees, page = CASES[name]
    trees = trees(rng)
    batch, pool, q = setup(rng, fmt, kv, hd, page, past, trees, heads)
    check(hip, pool, batch, heads, q, trees, extra=(4, 8))


@pytest.mark.parametrize("fmt,hd,heads", [("f16", 64, 32), ("i8", 128, 8), ("f8", 256, 2), ("f8", 64, 8)])
def test_one_tree_in_wide_tiles(hip, fmt, hd, heads):
    """More than 128 packed rows: the tiles that share their keys, whole steps, masked ones and the ends of both."""
    rng = np.random.default_rng(hd)
    for past, n in ((0, 150), (64, 150), (100, 131), (129, 33 if heads > 8 else 140)):
        print("wide", fmt, hd, past, n, flush=True)
        trees = [random_tree(rng, n, width=3)]
        batch, pool, q = setup(rng, fmt, 1, hd, 32, [past], trees, heads)
        check(hip, pool, batch, heads, q, trees)


def test_the_largest_tree(hip):
    rng = np.random.default_rng(4)
    trees = [random_tree(rng, 1024, width=3)]
    batch, pool, q = setup(rng, "i8", 1, 64, 64, [45], trees, 1)
    check(hip, pool, batch, 1, q, trees)


@pytest.mark.parametrize("fmt", ["f16", "i8", "f8"])
@pytest.mark.parametrize("hd,n,heads", [(64, 6, 4), (128, 20, 8), (64, 70, 4), (256, 70, 4)])
def test_rows_that_are_not_finite_reach_only_their_descendants(hip, fmt, hd, n, heads):
    rng = np.random.default_rng(n)
    trees = [random_tree(rng, n, width=3), chain(4)]
    batch, pool, q = setup(rng, fmt, 1, hd, 16, [37, 3], trees, heads)
    clean = attend(hip, pool, batch, heads, q, plan=plan_of(hip, pool, batch, heads, trees))
    seen = ancestors(trees[0])
    for what, at in (("value", n // 2), ("key", n // 3), ("value", n - 1)):
        other = Pool(fmt, 1, hd, 16, batch.n_pages)
        other.bytes[:] = pool.bytes
        k, v = random_rows(rng, 1, hd)
        (v if what == "value" else k)[0, 3] = np.nan if what == "key" else np.inf
        pos = 37 + at
        other.put(batch.pages[0][pos // 16], pos % 16, k, v)
        got = attend(hip, other, batch, heads, q, plan=plan_of(hip, other, batch, heads, trees))
        for t in range(n):
            if not seen[t, at]:
                assert np.array_equal(got[t], clean[t]), (what, at, t)
            elif what == "key" or fmt != "f16":
                assert np.isnan(got[t]).all(), (what, at, t)
            else:
                assert np.isnan(got[t][:, 3]).all() and np.isfinite(np.delete(got[t], 3, 1)).all(), (what, at, t)
        assert np.array_equal(got[n:], clean[n:])


def test_chains_as_parents_are_chains(hip):
    """Lists of parents that make chains of all sequences give the bits of a plan without."""
    rng = np.random.default_rng(8)
    trees = [chain(3), chain(60), chain(1)]
    batch, pool, q = setup(rng, "i8", 2, 64, 16, [40, 0, 7], trees, 8)
    plain = hip.kv_plan("i8", 2, 64, 16, pool.n_pages, 8)
    plain.set(batch.past, batch.new, batch.pages)
    want = attend(hip, pool, batch, 8, q, plan=plain)
    for given in ([None] * 3, as_given(trees)):
        got = attend(hip, pool, batch, 8, q, plan=plan_of(hip, pool, batch, 8, trees, given))
        assert np.array_equal(got, want)


def test_a_plan_with_trees_becomes_one_without(hip):
    rng = np.random.default_rng(9)
    trees = [random_tree(rng, 9), random_tree(rng, 14)]
    batch, pool, q = setup(rng, "f16", 2, 64, 16, [40, 5], trees, 8)
    plan = plan_of(hip, pool, batch, 8, trees)
    check(hip, pool, batch, 8, q, trees, plan=plan)
    plan.set(batch.past, batch.new, batch.pages)
    check(hip, pool, batch, 8, q, [chain(9), chain(14)], plan=plan)
    plan.set(batch.past, batch.new, batch.pages, parents=as_given(trees))
    check(hip, pool, batch, 8, q, trees, plan=plan)


# --- batches with work for tiles of more blocks, and for wide ones -----------------------

def decoded(pool, page_list, n):
    """A sequence's first n positions' (k, v) [n, kv, hd] in float64, all at once."""
    size = 2 if pool.fmt == "f16" else 1
    raw, part = pool.bytes[page_list], 16 * pool.hd * size  # [page, kv, block, bytes]
    out = []
    for i, where in enumerate((pool.key_at, pool.value_at)):
        bits = np.ascontiguousarray(raw[..., i * part:(i + 1) * part]).view(np.uint16 if size == 2 else np.uint8)[..., where]
        scale = None if size == 2 else np.ascontiguousarray(raw[..., 2 * part:]).view(np.float32)[..., 16 * i:16 * i + 16]
        x = dequantise(bits, scale, pool.fmt)  # [page, kv, block, 16, hd]
        out.append(x.transpose(0, 2, 3, 1, 4).reshape(-1, pool.kv, pool.hd)[:n])
    return out


def large(rng, fmt, hd, kv, heads, seqs, new, past):
    """A batch of trees (and a chain) with random caches: (batch, pool, queries, trees, past positions)."""
    trees = [random_tree(rng, int(n), width=4) for n in rng.integers(new // 2, new + 1, seqs - 1)] + [chain(new)]
    pasts = [past] + [int(n) for n in rng.integers(past // 2, past, seqs - 1)]
    batch = Batch(rng, [(p, len(t)) for p, t in zip(pasts, trees)], 64)
    pool = Pool(fmt, kv, hd, 64, batch.n_pages)
    part = 16 * hd * (2 if fmt == "f16" else 1)
    if fmt == "f16":
        values = rng.standard_normal(pool.bytes.size // 2, np.float32).astype(np.float16)
        pool.bytes[:] = values.view(np.uint8).reshape(pool.bytes.shape)
    else:
        pool.bytes[..., :2 * part] = rng.integers(0, 256, pool.bytes[..., :2 * part].shape, np.uint8)
        if fmt == "f8":
            pool.bytes[..., :2 * part] &= 0xBF  # (below 2, and no NaN)
        scales = np.exp(0.4 * rng.standard_normal(pool.bytes[..., 2 * part:].shape[:-1] + (32,))) / (64 if fmt == "i8" else 1)
        pool.bytes[..., 2 * part:] = np.ascontiguousarray(scales.astype(np.float32)).view(np.uint8)
    return batch, pool, rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32), trees, pasts


@pytest.mark.parametrize("fmt,hd,kv,heads,seqs,new,past", [
    ("i8", 64, 8, 32, 40, 24, 3000),    # 64 steps for each wave and more: three blocks
    ("i8", 64, 8, 32, 16, 18, 2500),    # two
    ("f8", 64, 8, 24, 40, 30, 3000), ("i8", 128, 8, 32, 24, 20, 2500), ("f8", 128, 4, 32, 24, 12, 3500),
    ("f16", 64, 8, 16, 40, 16, 3500),   # two blocks of an unquantised cache
    ("f16", 128, 8, 32, 24, 12, 4000),  # two, of a workgroup that has its CU to itself
    ("f16", 128, 8, 32, 16, 40, 2500),  # wide ones
    ("i8", 64, 8, 32, 12, 96, 2000), ("f8", 256, 2, 16, 24, 40, 3000), ("f16", 256, 2, 8, 40, 40, 2500)])
def test_tiles_by_the_batchs_work(hip, fmt, hd, kv, heads, seqs, new, past):
    print("work", fmt, hd, kv, heads, seqs, new, past, flush=True)
    rng = np.random.default_rng(hd + new)
    batch, pool, q, trees, pasts = large(rng, fmt, hd, kv, heads, seqs, new, past)
    if new % 8:
        q[::3] *= np.float32(2.0 ** -9)  # queries that get a factor, beside others that do not
    got, row = attend(hip, pool, batch, heads, q, plan=plan_of(hip, pool, batch, heads, trees)), 0
    group = heads // kv
    for s, t in enumerate(trees):
        n = len(t)
        if s % 5 == 0 or s == seqs - 1:
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


@pytest.mark.parametrize("fmt,hd,kv,heads,seqs,new,past", [
    ("i8", 64, 8, 32, 40, 24, 3000), ("i8", 128, 8, 32, 24, 20, 2500), ("f16", 64, 8, 16, 40, 16, 3500),
    ("f16", 128, 8, 32, 16, 40, 2500), ("f16", 128, 8, 32, 24, 12, 4000), ("i8", 64, 8, 32, 12, 96, 2000)])
def test_rows_that_are_not_finite_in_larger_tiles(hip, fmt, hd, kv, heads, seqs, new, past):
    rng = np.random.default_rng(new)
    batch, pool, q, trees, pasts = large(rng, fmt, hd, kv, heads, seqs, new, past)
    clean = attend(hip, pool, batch, heads, q, plan=plan_of(hip, pool, batch, heads, trees))
    hit, row = [], 0
    for s, t in enumerate(trees):
        n, at = len(t), int(rng.integers(len(t)))
        k, v = random_rows(rng, kv, hd)
        (v if s % 2 else k)[:, 5] = np.inf if s % 2 else np.nan
        pos = pasts[s] + at
        pool.put(batch.pages[s][pos // 64], pos % 64, k, v)
        sees = ancestors(t)[:, at]
        hit += [(row + i, bool(sees[i]), s % 2) for i in range(n)]
        row += n
    got = attend(hip, pool, batch, heads, q, plan=plan_of(hip, pool, batch, heads, trees))
    for i, sees, value in hit:
        if not sees:
            assert np.array_equal(got[i], clean[i]), i
        elif value and fmt == "f16":
            assert np.isnan(got[i][:, 5]).all() and np.isfinite(np.delete(got[i], 5, 1)).all(), i
        else:
            assert np.isnan(got[i]).all(), i
