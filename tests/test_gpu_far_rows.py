"""Rows and pages behind the first 4 GiB of their buffers give the bits that the same rows give in small ones."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import as_given, random_tree
from bobcat_amd.backend import RopeRows, kv_page_bytes

pytestmark = pytest.mark.gpu

FAR = 1 << 32


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


def plan_of(hip, past, trees, pages, n_pages, heads=4):
    plan = hip.kv_plan("i8", 1, 64, 16, n_pages, heads)
    plan.set(past, [len(t) for t in trees], pages, parents=as_given(trees))
    return plan


@pytest.mark.parametrize("mode", ["drawn", "chosen"])
def test_verdicts(hip, mode):
    rng = np.random.default_rng(1)
    vocab, tree = 1 << 20, random_tree(rng, 9, width=3)
    before = FAR // (4 * vocab) + 3  # sequences of one token each, whose rows lie in front
    logits = (2 * rng.standard_normal((9, vocab))).astype(np.float32)
    logits[:, rng.integers(0, vocab, 40)] += 14
    q = np.exp(logits + 0.5 * rng.standard_normal(logits.shape) - logits.max())
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    tokens, u = rng.integers(0, vocab, 9).astype(np.uint32), rng.random(9, np.float32)
    for i, a in enumerate(tree[1:], 1):
        tokens[i] = np.argsort(-q[a])[i % 4]
    got = []
    for n in (0, before):
        rows = n + 9
        trees = [[-1]] * n + [tree]
        plan = plan_of(hip, [0] * (n + 1), trees, [[i] for i in range(n + 1)], n + 1)
        lb, db = hip.new_buffer(rows * vocab * 4), hip.new_buffer(rows * vocab * 4)
        hip.write(lb.at(n * vocab * 4), logits)
        hip.write(db.at(n * vocab * 4), q)
        all_tokens = np.concatenate([np.zeros(n, np.uint32), tokens])
        all_u = np.concatenate([np.zeros(n, np.float32), u])
        heat = np.concatenate([np.zeros(n, np.float32), np.array([0.7], np.float32)])
        tb, ub, hb = hip.buffer_from(all_tokens), hip.buffer_from(all_u), hip.buffer_from(heat)
        kept, next_, path, chance = (hip.new_buffer(4 * k) for k in (n + 1, n + 1, rows, rows))
        run(hip, lambda: hip.verify_drafts(plan, 0, n + 1, vocab, lb.at(0), tb.at(0), ub.at(0), hb.at(0), kept.at(0), path.at(0),
                                           next_.at(0), chances=chance.at(0), draft=db.at(0) if mode == "drawn" else None))
        read = lambda b, at, k: hip.read(b.at(4 * at), np.empty(k, np.uint32)).tolist()  # noqa: E731
        got.append((read(kept, n, 1), read(next_, n, 1), read(path, n, 9), read(chance, n, 9)))
        for b in (lb, db):
            b.free()
    assert got[0] == got[1]


def test_attention_of_trees_and_kept_rows(hip):
    rng = np.random.default_rng(2)
    trees, past = [random_tree(rng, 14, width=3), random_tree(rng, 21, width=4)], [21, 40]
    need = [3, 4]
    q = hip.buffer_from(rng.standard_normal((35, 4 * 64)).astype(np.float32))
    path = hip.buffer_from(np.array([0, 2, 5, 9] + [0] * 10 + [0, 1, 7, 8, 20] + [0] * 16, np.uint32))
    kept = hip.buffer_from(np.array([4, 5], np.uint32))
    contents, got = None, []
    for n_pages in (7, FAR // 2176 + 50):
        pages, at = [], n_pages
        for n in need:
            pages.append(list(range(at - 1, at - 1 - n, -1)))
            at -= n
        plan = plan_of(hip, past, trees, pages, n_pages)
        size = kv_page_bytes(plan.shape)
        assert size == 2176
        cache = hip.new_buffer(2 * n_pages * size)
        if contents is None:
            contents = rng.integers(0, 256, (2, 7, size), np.uint8)
            contents[..., 2048:] = rng.uniform(0.01, 0.02, (2, 7, 32)).astype(np.float32).view(np.uint8)
        last = [cache.at((layer * n_pages + n_pages - 7) * size) for layer in range(2)]
        for layer in range(2):
            hip.write(last[layer], contents[layer])
        out = hip.new_buffer(35 * 4 * 64 * 4)
        run(hip, lambda: (hip.attention_paged(plan, cache.at(n_pages * size), q.at(0), 256, out.at(0), 256),
                          hip.kv_keep(plan, 0, 2, cache.at(0), 2, n_pages * size, kept.at(0), path.at(0))))
        got.append((hip.read(out.at(0), np.empty(35 * 256, np.float32)),
                    [hip.read(v, np.empty((7, size), np.uint8)) for v in last]))
        cache.free()
    assert np.array_equal(got[0][0], got[1][0]) and np.isfinite(got[0][0]).all()
    assert all(np.array_equal(a, b) for a, b in zip(got[0][1], got[1][1]))
    assert not np.array_equal(got[0][1][1], contents[1])


def test_rotary_rows(hip):
    rng = np.random.default_rng(3)
    tokens, some = (1 << 10) + 40, 20
    x = rng.standard_normal((some, 128)).astype(np.float32)
    plan = hip.kv_plan("f16", 1, 64, 16, 70, 2)
    plan.set([5], [tokens], [range(67)])
    rope, got = hip.rope(64, 1e4), []
    for stride in (128, 1 << 20):
        b = hip.new_buffer(((tokens - 1) * stride + 128) * 4)
        for i in range(some):
            hip.write(b.at((tokens - some + i) * stride * 4), x[i])
        run(hip, lambda: hip.rope_paged(rope, plan, RopeRows(b.at(0), stride, b.at(0), stride, 2), None))
        got.append([hip.read(b.at((tokens - some + i) * stride * 4), np.empty(128, np.float32)) for i in range(some)])
        b.free()
    assert np.array_equal(got[0], got[1]) and not np.array_equal(got[0], x)
