"""Steps with drafted tokens as a serving loop runs them, in one recording each: rotary positions, store, attention along
the trees, rules on the logits, the verdict, the kept rows, and the next step over what was kept."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import as_given, chain, depths, random_tree, rope, verify
from _paged import Batch, Pool, attention_bound, quantise, dequantise
from _drafts import tree_attention
from bobcat_amd.backend import LOGIT_ROW, NO_MASK, NO_TOKEN, RopeRows, rope_frequencies, rope_spec

pytestmark = pytest.mark.gpu


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


@pytest.mark.parametrize("fmt,hd,mode", [("f16", 64, "chosen"), ("i8", 128, "drawn"), ("f8", 256, "distinct")])
def test_two_steps(hip, fmt, hd, mode):
    rng = np.random.default_rng(hd)
    heads, kv, page, vocab, layers = 4, 2, 16, 700, 2
    past = [37, 0, 16, 90]
    trees = [random_tree(rng, 9, width=3), random_tree(rng, 14, width=3), chain(4), random_tree(rng, 6, width=2)]
    new = [len(t) for t in trees]
    tokens = sum(new)
    room = [p + n + 20 for p, n in zip(past, new)]
    batch = Batch(rng, [(n, 0) for n in room], page)  # pages for both steps
    pools = [Pool(fmt, kv, hd, page, batch.n_pages) for _ in range(layers)]
    for pool in pools:
        for s, n in enumerate(past):
            for at in range(n):
                pool.put(batch.pages[s][at // page], at % page, *rng.standard_normal((2, kv, hd)).astype(np.float32))
    apart = pools[0].bytes.nbytes
    cache = hip.buffer_from(np.concatenate([p.bytes.reshape(-1) for p in pools]))

    def pages(lengths):
        return [p[:-(-n // page)] for p, n in zip(batch.pages, lengths)]

    plan = hip.kv_plan(fmt, kv, hd, page, batch.n_pages, heads)
    plan.set(past, new, pages([p + n for p, n in zip(past, new)]), parents=as_given(trees))
    spec = rope_spec(hd // 2, 1e6, scaling="parts", factor=4.0, n_original=64, magnitude=1.1)
    turn = hip.rope(hd // 2, 1e6, scaling="parts", factor=4.0, n_original=64, magnitude=1.1)

    def layer_rows(n):
        return rng.standard_normal((n, (heads + 2 * kv) * hd)).astype(np.float32)

    qkv = [layer_rows(tokens) for _ in range(layers)]
    width = qkv[0].shape[1]
    rows = [hip.buffer_from(x) for x in qkv]
    outs = [hip.new_buffer(tokens * heads * hd * 4) for _ in range(layers)]
    logits = (2 * rng.standard_normal((tokens, vocab))).astype(np.float32)
    heat = np.array([0.8, 1.1, 0.0, 0.6], np.float32)
    near = logits + 0.5 * rng.standard_normal(logits.shape).astype(np.float32)
    q = np.exp(near - near.max(-1, keepdims=True))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    ids, at = np.zeros(tokens, np.uint32), 0
    for t in trees:
        for i in range(len(t)):
            kids = [at + c for c, a in enumerate(t) if a == i]
            ids[kids] = np.argsort(-near[at + i])[:len(kids)] if mode == "chosen" else rng.choice(
                vocab, len(kids), replace=mode == "drawn", p=q[at + i].astype(np.float64) / q[at + i].astype(np.float64).sum())
        at += len(t)
    u = rng.random(tokens, np.float32) * np.float32(0.7)
    allowed = rng.random((tokens, vocab)) < 0.8
    words = np.zeros((tokens, -(-vocab // 32) * 32), np.uint32)
    words[:, :vocab] = allowed
    words = (words.reshape(tokens, -1, 32) << np.arange(32, dtype=np.uint32)).sum(-1).astype(np.uint32)
    rules = np.zeros(tokens, LOGIT_ROW)
    rules["mask"], rules["repeat"] = np.arange(tokens), 1
    rules["mask"][::3] = NO_MASK
    up = hip.buffer_from
    b = dict(logits=up(logits), rules=up(rules.view(np.uint8)), masks=up(words), q=up(q), ids=up(ids), u=up(u), heat=up(heat),
             kept=hip.new_buffer(16), path=hip.new_buffer(4 * tokens), next=hip.new_buffer(16), chances=hip.new_buffer(4 * tokens))

    def step():
        for i in range(layers):
            r, c = rows[i], cache.at(i * apart)
            k, v = r.floats(heads * hd), r.floats((heads + kv) * hd)
            hip.rope_paged(turn, plan, RopeRows(r.at(0), width, r.at(0), width, heads), RopeRows(k, width, k, width, kv))
            hip.kv_store(plan, c, k, width, v, width)
            hip.attention_paged(plan, c, r.at(0), width, outs[i].at(0), heads * hd)
        hip.logits_edit(b["logits"].at(0), b["logits"].at(0), tokens, vocab, b["rules"].at(0), masks=b["masks"].at(0), n_masks=tokens)
        hip.verify_drafts(plan, 0, 4, vocab, b["logits"].at(0), b["ids"].at(0), b["u"].at(0), b["heat"].at(0), b["kept"].at(0),
                          b["path"].at(0), b["next"].at(0), chances=b["chances"].at(0),
                          draft=None if mode == "chosen" else b["q"].at(0), distinct=mode == "distinct")
        hip.kv_keep(plan, 0, 4, cache.at(0), layers, apart, b["kept"].at(0), b["path"].at(0))

    run(hip, step)
    kept, path, next_ = (hip.read(b[k].at(0), np.empty(n, np.uint32)) for k, n in (("kept", 4), ("path", tokens), ("next", 4)))

    # The parts, each from what the one before it gave.
    positions = [p + d for p, t in zip(past, trees) for d in depths(t)]
    f, ends, turned = rope_frequencies(spec), np.cumsum([0] + new), []
    for i in range(layers):
        got = hip.read(rows[i].at(0), np.empty_like(qkv[i]))
        turned.append(got)
        for a, n in ((0, heads), (heads * hd, kv)):
            part = slice(a, a + n * hd)
            want, size = rope(qkv[i][:, part].reshape(tokens, n, hd), positions, f, "halves", 1.1)
            assert (np.abs(got[:, part].reshape(tokens, n, hd) - want) <= 9 * 2.0 ** -24 * size).all()
        assert np.array_equal(got[:, (heads + kv) * hd:], qkv[i][:, (heads + kv) * hd:])
        out = hip.read(outs[i].at(0), np.empty((tokens, heads, hd), np.float32))
        for s, t in enumerate(trees):
            part = slice(ends[s], ends[s + 1])
            old = [pools[i].get(batch.pages[s][p // page], p % page) for p in range(past[s])]
            x = got[part, heads * hd:].reshape(-1, 2, kv, hd)
            rest = [dequantise(*quantise(x[:, j], fmt), fmt) for j in range(2)]
            keys, values = (np.concatenate([np.array([o[j] for o in old]).reshape(-1, kv, hd), rest[j]]) for j in range(2))
            qs = got[part, :heads * hd].reshape(-1, heads, hd)
            off = np.abs(out[part] - tree_attention(qs, keys, values, past[s], t)).max()
            assert off <= attention_bound(qs, keys, values)
    edited = np.where(allowed | (np.arange(tokens) % 3 == 0)[:, None], logits, -np.inf).astype(np.float32)
    assert np.array_equal(hip.read(b["logits"].at(0), np.empty_like(logits)), edited)
    paths = []
    for s, t in enumerate(trees):
        part = slice(ends[s], ends[s + 1])
        want = verify(t, edited[part], None if mode == "chosen" else q[part], ids[part], u[part], heat[s], mode == "distinct")
        assert (kept[s], path[part].tolist(), next_[s]) == (want[0], want[1], want[2])
        assert next_[s] != NO_TOKEN
        paths.append(want[1][:want[0]])
    assert sum(map(len, paths)) > 4  # (some drafts stay, so that rows move)

    # The next step, a token each, gives the bits of one over a cache that only ever got the kept tokens.
    plain = hip.buffer_from(np.concatenate([p.bytes.reshape(-1) for p in pools]))
    after = [p + len(x) for p, x in zip(past, paths)]
    short = hip.kv_plan(fmt, kv, hd, page, batch.n_pages, heads)
    short.set(past, [len(x) for x in paths], pages(after))
    order = np.concatenate([ends[s] + np.array(x) for s, x in enumerate(paths)])
    for i in range(layers):
        kept_rows = hip.buffer_from(np.ascontiguousarray(turned[i][order]))
        run(hip, lambda: hip.kv_store(short, plain.at(i * apart), kept_rows.floats(heads * hd), width,
                                      kept_rows.floats((heads + kv) * hd), width))
    plan.set(after, [1] * 4, pages([n + 1 for n in after]))
    more = [hip.buffer_from(layer_rows(4)) for _ in range(layers)]
    results = []
    for where in (cache, plain):
        for i in range(layers):
            copy = hip.buffer_from(hip.read(more[i].at(0), np.empty((4, width), np.float32)))
            k, v, out = copy.floats(heads * hd), copy.floats((heads + kv) * hd), hip.new_buffer(4 * heads * hd * 4)

            def next_step():
                hip.rope_paged(turn, plan, RopeRows(copy.at(0), width, copy.at(0), width, heads), RopeRows(k, width, k, width, kv))
                hip.kv_store(plan, where.at(i * apart), k, width, v, width)
                hip.attention_paged(plan, where.at(i * apart), copy.at(0), width, out.at(0), heads * hd)

            run(hip, next_step)
            results.append(hip.read(out.at(0), np.empty((4, heads, hd), np.float32)))
    for i in range(layers):
        assert np.array_equal(results[i], results[layers + i]) and np.isfinite(results[i]).all()


def test_plans_are_held_by_work_that_reads_them(hip):
    """Each of the operators marks its plan as used until the recording has been waited for."""
    from bobcat_amd import BobcatError
    from bobcat_amd._lib import STATUS
    tree = [random_tree(np.random.default_rng(1), 5)]
    b, r = hip.new_buffer(1 << 16), hip.rope(64, 1e4)
    calls = [lambda p: hip.rope_paged(r, p, RopeRows(b.at(0), 64, b.at(1 << 15), 64, 1), None),
             lambda p: hip.kv_keep(p, 0, 1, b.at(0), 1, 0, b.at(1 << 15), b.at(1 << 14)),
             lambda p: hip.verify_drafts(p, 0, 1, 8, b.at(0), *(b.at(256 * i) for i in range(1, 7)))]
    for call in calls:
        plan = hip.kv_plan("i8", 1, 64, 16, 1, 1)
        give = lambda: plan.set([0], [5], [[0]], parents=as_given(tree))  # noqa: E731
        give()
        hip.begin()
        call(plan)
        with pytest.raises(BobcatError) as e:
            give()
        assert e.value.status == STATUS["Busy"]
        ticket = hip.commit()
        with pytest.raises(BobcatError) as e:
            give()
        assert e.value.status == STATUS["Busy"]
        hip.wait(ticket)
        give()
