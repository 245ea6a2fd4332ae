"""GPU parity of bch_kv_keep: the cache's bytes equal those of moving each row by itself, in the order of the path."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import Batch, Pool
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS
from bobcat_amd.backend import Hip

pytestmark = pytest.mark.gpu


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


def moved(pool, batch, bytes_, s, path):
    """Rows of a path moved one after the other in a copy of a cache's bytes."""
    out, n = bytes_.copy(), 16 * pool.hd * (2 if pool.fmt == "f16" else 1)
    size = 2 if pool.fmt == "f16" else 1
    kind = np.uint16 if size == 2 else np.uint8

    def row(raw, at):
        p = batch.past[s] + at
        page, b, i = batch.pages[s][p // pool.page], p % pool.page // 16, p % 16
        parts = []
        for h in range(pool.kv):
            block = raw[page, h, b]
            parts += [(block[:n].view(kind), pool.key_at[i]), (block[n:2 * n].view(kind), pool.value_at[i])]
            if size == 1:
                parts.append((block[2 * n:].view(np.float32), np.array([i, 16 + i])))
        return parts

    for j, a in enumerate(path):
        for (to, at), (of, where) in zip(row(out, j), row(out, a)):
            to[at] = of[where].copy()
    return out


def path_of(rng, new):
    """Places that go up, the first among them, some of them neighbours."""
    if not new:
        return []
    return sorted(set([0, *rng.choice(new, rng.integers(1, new + 1), replace=False).tolist()]))


@pytest.mark.parametrize("fmt", ["f16", "i8", "f8"])
@pytest.mark.parametrize("kv,hd,page", [(1, 64, 16), (3, 128, 48), (2, 256, 32)])
@pytest.mark.parametrize("layers", [1, 3])
def test_rows_of_the_path(hip, fmt, kv, hd, page, layers):
    print("kv_keep", fmt, kv, hd, page, layers, flush=True)
    rng = np.random.default_rng(hd + layers)
    batch = Batch(rng, [(0, 9), (15, 2), (33, 0), (100, 24), (31, 40), (7, 1), (16, 17)], page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    caches = rng.integers(0, 128, (layers, *pool.bytes.shape), np.uint8)  # (no NaN among the scales)
    caches.view(np.uint32)[...] &= 0x7f7fffff if fmt != "f16" else 0xffffffff
    apart = pool.bytes.nbytes + 64
    given = np.full(layers * apart, 0x5a, np.uint8)
    for i in range(layers):
        given[i * apart:i * apart + pool.bytes.nbytes] = caches[i].reshape(-1)
    for first, n in ((0, 7), (2, 3), (3, 1), (7, 0)):
        paths = [path_of(rng, m) for m in batch.new]
        paths[4] = list(range(40))  # all, in place
        plan = hip.kv_plan(fmt, kv, hd, page, batch.n_pages, kv)
        plan.set(batch.past, batch.new, batch.pages)
        kept = np.array([len(p) for p in paths], np.uint32)
        path = np.concatenate([p + [0xFFFFFFFF] * (m - len(p)) for p, m in zip(paths, batch.new)]).astype(np.uint32)
        row, rows = sum(batch.new[:first]), sum(batch.new[first:first + n])
        kb = hip.buffer_from(np.append(kept[first:first + n], np.uint32(9)))
        pb = hip.buffer_from(np.append(path[row:row + rows], np.uint32(1)))
        cache = hip.buffer_from(given)
        run(hip, lambda: hip.kv_keep(plan, first, n, cache.at(0), layers, apart, kb.at(0), pb.at(0)))
        got = hip.read(cache.at(0), np.empty_like(given))
        want = given.copy()
        for i in range(layers):
            raw = caches[i]
            for s in range(first, first + n):
                raw = moved(pool, batch, raw, s, paths[s])
            want[i * apart:i * apart + pool.bytes.nbytes] = raw.reshape(-1)
        assert np.array_equal(got, want), (first, n)


def test_paths_that_are_none_stay_inside_the_new_tokens(hip):
    """Counts and places that no path has: only rows of the sequence's new tokens may change."""
    rng = np.random.default_rng(2)
    batch = Batch(rng, [(20, 6), (33, 5)], 16)
    pool = Pool("i8", 2, 64, 16, batch.n_pages)
    pool.bytes[:] = rng.integers(0, 64, pool.bytes.shape, np.uint8)
    plan = hip.kv_plan("i8", 2, 64, 16, batch.n_pages, 2)
    plan.set(batch.past, batch.new, batch.pages)
    for kept, path in (([0xFFFFFFFF, 200], [0, 5, 0xFFFFFFFF, 6, 2, 100, 4, 3, 2, 1, 0]), ([0, 0], [5] * 11)):
        cache = hip.buffer_from(pool.bytes)
        kb, pb = hip.buffer_from(np.array(kept, np.uint32)), hip.buffer_from(np.array(path, np.uint32))
        run(hip, lambda: hip.kv_keep(plan, 0, 2, cache.at(0), 1, 0, kb.at(0), pb.at(0)))
        after = Pool("i8", 2, 64, 16, batch.n_pages)
        after.bytes[:] = hip.read(cache.at(0), np.empty_like(pool.bytes))
        for s, (past, new) in enumerate(zip(batch.past, batch.new)):
            for at in range(len(batch.pages[s]) * 16):
                if not past <= at < past + new or kept == [0, 0]:
                    for a, b in zip(after.get(batch.pages[s][at // 16], at % 16), pool.get(batch.pages[s][at // 16], at % 16)):
                        assert np.array_equal(a, b), (s, at)


def test_refusals(hip):
    plan = hip.kv_plan("f16", 1, 64, 16, 2, 1)
    plan.set([3, 0], [5, 2], [[0], [1]])
    size = 2 * 4096
    cache, kb, pb = hip.new_buffer(3 * size), hip.new_buffer(8), hip.new_buffer(28)

    def refused(status, first=0, n=2, at=0, layers=1, apart=size, kept=kb.at(0), path=pb.at(0), plan_=plan):
        hip.begin()
        with pytest.raises(BobcatError) as e:
            hip.kv_keep(plan_, first, n, cache.at(at), layers, apart, kept, path)
        hip.discard()
        assert e.value.status == STATUS[status], str(e.value)

    with pytest.raises(BobcatError) as e:
        hip.kv_keep(plan, 0, 2, cache.at(0), 1, size, kb.at(0), pb.at(0))
    assert e.value.status == STATUS["NotRecording"]
    refused("Argument", first=1)
    refused("Argument", first=3, n=0)
    refused("Argument", first=0xFFFFFFFF, n=2)
    refused("OutOfBounds", at=2 * size + 16)
    refused("OutOfBounds", layers=4)
    refused("Argument", layers=2, apart=size - 16)
    refused("Argument", layers=2, apart=size + 8)
    refused("Argument", layers=2, apart=(1 << 64) - 16)
    refused("Argument", layers=129)
    refused("Argument", at=8)
    refused("OutOfBounds", kept=kb.at(4))
    refused("OutOfBounds", path=pb.at(4))
    refused("Argument", kept=cache.at(16))
    refused("Argument", layers=3, path=cache.at(2 * size + 64))
    odd = hip.new_buffer(64)
    refused("Argument", path=odd.at(2))
    with Hip() as other:
        refused("ForeignBuffer", kept=other.new_buffer(8).at(0))
    run(hip, lambda: hip.kv_keep(plan, 2, 0, cache.at(0), 1, 0, kb.at(8), pb.at(28)))
    run(hip, lambda: hip.kv_keep(plan, 0, 2, cache.at(0), 0, 0, kb.at(0), pb.at(0)))
