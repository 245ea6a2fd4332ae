"""GPU parity of bch_verify_drafts with the walk by its definition (tests/_drafts.py, float64), on the same inputs: kept
tokens, paths and next tokens are equal, probabilities agree to f32.

A test or a draw can only differ from the definition's where its uniform lies within rounding of a border (the sums'
relative error, below 2^-22 here: the exponentials are off by at most |exponent| + 2 roundings of 2^-24, at most 24 of them,
with either sign, and sums are f64): of all the tests' draws together that is below one in a thousand, and their
seeds are fixed.  The probabilities are f64 of a sum with that error, rounded once: 2^-22."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import as_given, chain, random_tree, verify
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS
from bobcat_amd.backend import NO_TOKEN, Hip

pytestmark = pytest.mark.gpu


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


def plan_of(hip, trees, n_chains=False):
    plan = hip.kv_plan("i8", 1, 64, 512, max(1, sum(-(-len(t) // 512) for t in trees)), 1)
    need = [-(-len(t) // 512) for t in trees]
    ends = np.cumsum([0] + need)
    plan.set([0] * len(trees), [len(t) for t in trees], [range(a, b) for a, b in zip(ends, ends[1:])],
             parents=None if n_chains else as_given(trees))
    return plan


def verdict(hip, plan, trees, logits, draft, tokens, uniforms, temperatures, distinct=False, first=0, n=None, chances=True,
            slack=0):
    """verify_drafts of sequences first .. first + n, whose rows the arrays hold; `slack` floats before the logits."""
    n = len(trees) - first if n is None else n
    rows = sum(len(t) for t in trees[first:first + n])
    vocab = logits.shape[1]
    fill = lambda count: hip.buffer_from(np.full(count + 1, 0x77777777, np.uint32))  # noqa: E731
    kept, path, next_, chance = fill(n), fill(rows), fill(n), fill(rows)
    up = lambda x, t=np.float32: hip.buffer_from(np.ascontiguousarray(x, t))  # noqa: E731
    lb = hip.buffer_from(np.concatenate([np.full(slack, np.nan, np.float32), logits.reshape(-1)]))
    db = None if draft is None else hip.buffer_from(np.concatenate([np.full(slack, np.nan, np.float32), draft.reshape(-1)]))
    tb, ub, hb = up(tokens, np.uint32), up(uniforms), up(temperatures)
    run(hip, lambda: hip.verify_drafts(plan, first, n, vocab, lb.floats(slack), tb.at(0), ub.at(0), hb.at(0), kept.at(0),
                                       path.at(0), next_.at(0), chances=chance.at(0) if chances else None,
                                       draft=None if db is None else db.floats(slack), distinct=distinct))
    out = []
    for b, count in ((kept, n), (path, rows), (next_, n), (chance, rows)):
        got = hip.read(b.at(0), np.empty(count + 1, np.uint32))
        assert got[-1] == 0x77777777
        out.append(got[:-1])
    if not chances:
        assert (out[3] == 0x77777777).all()
    out[3] = out[3].view(np.float32)
    return out


def check(hip, trees, logits, draft, tokens, uniforms, temperatures, distinct=False, first=0, n=None, plan=None, slack=0):
    got = verdict(hip, plan or plan_of(hip, trees), trees, logits, draft, tokens, uniforms, temperatures, distinct, first, n,
                  slack=slack)
    row = 0
    for i, t in enumerate(trees[first:None if n is None else first + n]):
        m = len(t)
        if not m:
            assert got[0][i] == 0 and got[2][i] == NO_TOKEN
            continue
        part = slice(row, row + m)
        kept, path, token, chances = verify(t, logits[part], None if draft is None else draft[part], tokens[part],
                                            uniforms[part], temperatures[i], distinct)
        assert got[0][i] == kept and got[1][part].tolist() == path and got[2][i] == token, (i, t)
        np.testing.assert_allclose(got[3][part], chances, rtol=2.0 ** -22, atol=1e-37)
        row += m
    return got


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def case(rng, trees, vocab, mode, heat=None, spread=2.0):
    """Logits, a draft near the target (or none), tokens drawn from it at each parent, uniforms, temperatures."""
    rows = sum(map(len, trees))
    logits = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    temperatures = (rng.uniform(0.4, 1.5, len(trees)) if heat is None else np.full(len(trees), heat)).astype(np.float32)
    each = np.repeat(np.where(temperatures > 0, temperatures, 1), [len(t) for t in trees])[:, None]
    near = logits / each + 0.6 * rng.standard_normal(logits.shape)
    q = softmax(near)
    tokens, at = np.zeros(rows, np.uint32), 0
    for t in trees:
        for i in range(len(t)):
            kids = [c for c, a in enumerate(t) if a == i]
            if mode == "chosen":
                picks = np.argsort(-near[at + i])[:len(kids)]
            else:
                p = q[at + i].astype(np.float64)
                picks = rng.choice(vocab, len(kids), replace=mode == "drawn", p=p / p.sum())
            tokens[[at + c for c in kids]] = picks
        at += len(t)
    return logits, None if mode == "chosen" else q, tokens, rng.random(rows, np.float32), temperatures


@pytest.mark.parametrize("mode", ["drawn", "distinct", "chosen"])
@pytest.mark.parametrize("vocab", [1, 3, 63, 64, 1000, 4096, 4097, 70001])
def test_trees(hip, mode, vocab):
    print("verify", mode, vocab, flush=True)
    rng = np.random.default_rng(vocab)
    wide = min(4, vocab)
    trees = [random_tree(rng, int(n), width=wide) for n in rng.integers(1, 14, 24 if vocab < 5000 else 8)] + [chain(6), chain(1)]
    trees.insert(3, [])
    logits, q, tokens, u, heat = case(rng, trees, vocab, mode, spread=0.5 if vocab < 100 else 2.0)
    heat[::5] = [0.0, -1.0, np.nan, 0.0, 0.0, 0.0][:len(heat[::5])]
    check(hip, trees, logits, q, tokens, u, heat, mode == "distinct")


@pytest.mark.parametrize("mode", ["drawn", "chosen"])
def test_chains_without_parents(hip, mode):
    rng = np.random.default_rng(7)
    trees = [chain(int(n)) for n in rng.integers(0, 9, 40)]
    logits, q, tokens, u, heat = case(rng, trees, 517, mode)
    check(hip, trees, logits, q, tokens, u, heat, plan=plan_of(hip, trees, n_chains=True), slack=1)


@pytest.mark.parametrize("slack", [1, 2, 3])
def test_rows_at_any_alignment(hip, slack):
    rng = np.random.default_rng(slack)
    trees = [random_tree(rng, 7), chain(5)]
    logits, q, tokens, u, heat = case(rng, trees, 8191 + slack, "drawn")
    check(hip, trees, logits, q, tokens, u, heat, slack=slack)


def test_a_part_of_the_sequences(hip):
    rng = np.random.default_rng(11)
    trees = [random_tree(rng, n) for n in (5, 9, 1, 12, 4)]
    logits, q, tokens, u, heat = case(rng, trees, 300, "distinct")
    plan, ends = plan_of(hip, trees), np.cumsum([0] + [len(t) for t in trees])
    for first, n in ((0, 2), (1, 3), (4, 1), (5, 0)):
        rows = slice(ends[first], ends[first + n])
        check(hip, trees, logits[rows], q[rows], tokens[rows], u[rows], heat[first:first + n], True, first, n, plan)


def test_the_largest_tree_and_many_children(hip):
    rng = np.random.default_rng(12)
    for mode in ("chosen", "drawn"):
        star = [[-1] + [0] * (1023 if mode == "chosen" else 40)]
        logits, q, tokens, u, heat = case(rng, star, 1500, mode, heat=1.0, spread=0.1)
        u[1:] = 0.9999  # nearly all are looked at
        check(hip, star, logits, q, tokens, u, heat)
    deep = [chain(1024)]
    logits, q, tokens, u, heat = case(rng, deep, 64, "chosen", heat=0.05)
    u[1:] = 0.0
    got = check(hip, deep, logits, None, tokens, u, heat)
    assert got[0][0] == 1024 or got[0][0] > 100


def test_one_token_named_by_several_children(hip):
    rng = np.random.default_rng(13)
    trees = [[-1, 0, 0, 0, 1, 2]] * 30
    logits, q, tokens, u, heat = case(rng, trees, 20, "drawn", spread=1.0)
    tokens[:] = np.tile(np.array([0, 7, 7, 7, 3, 3], np.uint32), 30)
    check(hip, trees, logits, q, tokens, u, heat)
    check(hip, trees, logits, None, tokens, u, heat)
    tokens[1::6] = 20  # outside the vocabulary
    tokens[2::6] = 0xFFFFFFFF
    check(hip, trees, logits, q, tokens, u, heat)
    check(hip, trees, logits, None, tokens, u, heat)


def test_certain_tests(hip):
    """Tests that no rounding can turn: a draft that is the target keeps all, no probability keeps nothing."""
    rng = np.random.default_rng(14)
    trees, vocab = [chain(5)] * 8, 100
    logits, _, tokens, u, heat = case(rng, trees, vocab, "drawn", heat=1.0)
    half = softmax(logits) / 2  # u·q < p for every u below 1
    u[:] = np.nextafter(np.float32(1), np.float32(0))
    got = check(hip, trees, logits, half, tokens, u, heat)
    assert (got[0] == 5).all()
    logits[np.arange(40), np.roll(tokens, -1)] = -np.inf  # each token's child
    u[:] = 0
    got = check(hip, trees, logits, half, tokens, u, heat)
    assert (got[0] == 1).all()
    u[:] = np.nan
    logits[:] = rng.standard_normal(logits.shape)
    got = verdict(hip, plan_of(hip, trees), trees, logits, half, tokens, u, heat)
    assert (got[0] == 1).all() and (got[2] < vocab).all()


def test_logits_that_are_not_finite(hip):
    rng = np.random.default_rng(15)
    trees, vocab = [random_tree(rng, 5) for _ in range(12)], 90
    for mode in ("drawn", "chosen"):
        logits, q, tokens, u, heat = case(rng, trees, vocab, mode)
        logits[rng.random(logits.shape) < 0.3] = -np.inf
        logits[rng.random(logits.shape) < 0.1] = np.nan
        logits[::7] = -np.inf      # no token at all
        logits[3::7] = np.nan
        logits[5::7, 11] = np.inf  # nothing else counts beside it
        logits[6::7, 4:6] = np.finfo(np.float32).max
        heat[::4] = 0
        check(hip, trees, logits, q, tokens, u, heat)


@pytest.mark.parametrize("heat", [1e-45, 1e-38, 1e-6, 1e6, 1e38, np.inf])
def test_temperatures_at_the_ends(hip, heat):
    rng = np.random.default_rng(16)
    trees = [random_tree(rng, 6) for _ in range(6)]
    logits, q, tokens, u, _ = case(rng, trees, 77, "drawn", heat=1.0)
    got = verdict(hip, plan_of(hip, trees), trees, logits, q, tokens, u, np.full(6, heat, np.float32))
    if heat >= 1e6 and heat < np.inf:
        check(hip, trees, logits, q, tokens, u, np.full(6, heat, np.float32))
    if heat <= 1e-6:  # (largest logits of the rows are far enough apart)
        cold = verdict(hip, plan_of(hip, trees), trees, logits, None, tokens, u, np.zeros(6, np.float32))
        assert np.array_equal(got[2][got[0] == cold[0]], cold[2][got[0] == cold[0]])
    assert (got[2] < 77).all() and np.isfinite(got[3]).all()


def test_drafts_that_are_no_probabilities(hip):
    """Nothing of a draft's row leads out of bounds, and the next token is one that the target has."""
    rng = np.random.default_rng(17)
    trees, vocab = [random_tree(rng, 6) for _ in range(10)], 50
    logits, q, tokens, u, heat = case(rng, trees, vocab, "drawn")
    logits[:, ::3] = -np.inf
    for bad in (np.nan, np.inf, -np.inf, -3.0, 1e30):
        q[rng.random(q.shape) < 0.2] = bad
        for distinct in (False, True):
            got = verdict(hip, plan_of(hip, trees), trees, logits, q, tokens, u, heat, distinct)
            assert ((got[0] >= 1) & (got[0] <= 6)).all() and (got[2] < vocab).all() and (got[2] % 3 != 0).all()


@pytest.mark.parametrize("mode", ["drawn", "distinct", "chosen"])
def test_tokens_have_the_targets_distribution(hip, mode):
    """Over 20,000 walks the first token after the root is distributed as p, whatever the draft: each count is within five
    standard deviations of its mean (a chance of about one in 10^5 for all of them, and fixed inputs)."""
    rng = np.random.default_rng(18)
    n, vocab, tree = 20000, 12, [-1, 0, 0, 0]
    logits = np.tile(rng.standard_normal(vocab).astype(np.float32), (4 * n, 1))
    q = softmax(rng.standard_normal(vocab))
    if mode == "chosen":
        tokens = np.tile(np.array([0, 3, 8, 5], np.uint32), n)
    else:
        order = np.log(q) + rng.gumbel(size=(n, 3, vocab) if mode == "drawn" else (n, vocab))
        picks = order.argmax(-1) if mode == "drawn" else np.argsort(-order, -1)[:, :3]
        tokens = np.concatenate([np.zeros((n, 1), np.uint32), picks.astype(np.uint32)], 1).reshape(-1)
    got = verdict(hip, plan_of(hip, [tree] * n), [tree] * n, logits, None if mode == "chosen" else np.tile(q, (4 * n, 1)),
                  tokens, rng.random(4 * n, np.float32), np.ones(n, np.float32), mode == "distinct")
    path = got[1].reshape(n, 4)
    after = np.where(got[0] > 1, tokens.reshape(n, 4)[np.arange(n), np.minimum(path[:, 1], 3)], got[2])
    p = softmax(logits[0]).astype(np.float64)
    count = np.bincount(after, minlength=vocab)
    assert (np.abs(count - n * p) < 5 * np.sqrt(n * p * (1 - p))).all(), (count / n, p)
    # The share of walks that keep a draft: the children's own p, or at least what the first child alone keeps, sum min(p, q).
    share, sigma = (got[0] > 1).mean(), 5 * np.sqrt(0.25 / n)
    if mode == "chosen":
        assert abs(share - p[[3, 8, 5]].sum()) < sigma
    else:
        assert np.minimum(p, q).sum() - sigma < share < 1


def test_two_calls_in_one_recording(hip):
    """Calls in a row share the scratch memory, also where the second's is larger."""
    rng = np.random.default_rng(19)
    small, large = [chain(3)] * 3, [random_tree(rng, 20) for _ in range(10)]
    cases = [(t, case(rng, t, v, "drawn")) for t, v in ((small, 5000), (large, 9000), (small, 5000))]
    outs, plans = [], [plan_of(hip, t) for t, _ in cases]
    made = []
    for (t, (logits, q, tokens, u, heat)) in cases:
        bufs = [hip.buffer_from(np.ascontiguousarray(x)) for x in (logits, q, tokens, u, heat)]
        rows = len(tokens)
        made.append((bufs, [hip.new_buffer(4 * len(t)), hip.new_buffer(4 * rows), hip.new_buffer(4 * len(t))]))

    def both():
        for plan, (t, c), (i, o) in zip(plans, cases, made):
            hip.verify_drafts(plan, 0, len(t), c[0].shape[1], i[0].at(0), i[2].at(0), i[3].at(0), i[4].at(0), o[0].at(0),
                              o[1].at(0), o[2].at(0), draft=i[1].at(0))

    run(hip, both)
    for (t, (logits, q, tokens, u, heat)), (_, o) in zip(cases, made):
        row = 0
        kept, next_ = (hip.read(o[j].at(0), np.empty(len(t), np.uint32)) for j in (0, 2))
        for i, tree in enumerate(t):
            part = slice(row, row + len(tree))
            want = verify(tree, logits[part], q[part], tokens[part], u[part], heat[i], False)
            assert (kept[i], next_[i]) == (want[0], want[2])
            row += len(tree)


def test_refusals(hip):
    trees = [chain(3), [-1, 0, 0]]
    plan, vocab = plan_of(hip, trees), 100
    b = {k: hip.new_buffer(v) for k, v in dict(logits=2400, draft=2400, tokens=24, uniforms=24, temperatures=8, kept=8,
                                               path=24, next=8, chances=24).items()}

    def refused(status, plan_=plan, first=0, n=2, v=vocab, **change):
        at = {k: x.at(0) for k, x in b.items()} | change
        hip.begin()
        with pytest.raises(BobcatError) as e:
            hip.verify_drafts(plan_, first, n, v, *[at[k] for k in ("logits", "tokens", "uniforms", "temperatures", "kept", "path", "next")],
                              chances=at["chances"], draft=at["draft"])
        hip.discard()
        assert e.value.status == STATUS[status], str(e.value)

    with pytest.raises(BobcatError) as e:
        hip.verify_drafts(plan, 0, 2, vocab, *[b[k].at(0) for k in ("logits", "tokens", "uniforms", "temperatures", "kept", "path", "next")])
    assert e.value.status == STATUS["NotRecording"]
    refused("Argument", first=1)
    refused("Argument", v=0)
    refused("Argument", v=(1 << 30) + 1)
    refused("OutOfBounds", v=101)
    for k in b:
        refused("OutOfBounds", **{k: b[k].at(4)})
        refused("Argument" if k in ("logits", "draft") else "Argument", v=99, **{k: hip.new_buffer(4000).at(2)})
    refused("Argument", kept=b["next"].at(0))
    refused("Argument", path=b["tokens"].at(0))
    refused("Argument", chances=b["logits"].at(16))
    refused("Argument", plan_=plan_of(hip, [chain(3), [-1, -1, 0]]))
    refused("Argument", plan_=plan_of(hip, [chain(3000), chain(3)]))
    with Hip() as other:
        refused("ForeignBuffer", plan_=plan_of(other, trees))
    run(hip, lambda: hip.verify_drafts(plan_of(hip, [chain(3), [-1, -1, 0]]), 0, 1, vocab, *[
        b[k].at(0) for k in ("logits", "tokens", "uniforms", "temperatures", "kept", "path", "next")]))
