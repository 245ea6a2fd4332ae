"""GPU parity of bch_logits_edit against a float64 restatement: penalties over
whole histories, biases in list order, masks.  The largest error allowed is
that of its own f32 operations on a logit x: at most five roundings of 2^-24 of
the largest value on the way (the quotient or product, frequency·c, the sum of
the penalties, the difference) and one more for each bias."""
from __future__ import annotations

import numpy as np
import pytest

from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS, Sampling
from bobcat_amd.backend import LOGIT_ROW, NO_MASK

pytestmark = pytest.mark.gpu


def rules(histories, biases, masks=None, repeat=1.2, presence=0.3, frequency=0.1):
    """(rows, history, bias tokens, bias values) of lists per row."""
    rows = np.zeros(len(histories), LOGIT_ROW)
    rows["history_len"], rows["bias_len"] = [len(h) for h in histories], [len(b) for b in biases]
    rows["history_at"] = np.cumsum([0] + [len(h) for h in histories[:-1]])
    rows["bias_at"] = np.cumsum([0] + [len(b) for b in biases[:-1]])
    rows["mask"] = NO_MASK if masks is None else masks
    rows["repeat"], rows["presence"], rows["frequency"] = repeat, presence, frequency
    flat = [t for h in histories for t in h]
    return (rows, np.asarray(flat, np.uint32), np.asarray([t for b in biases for t, _ in b], np.uint32),
            np.asarray([v for b in biases for _, v in b], np.float32))


def words(allowed):
    """Mask words of truth values [masks, vocab]."""
    padded = np.zeros((allowed.shape[0], -(-allowed.shape[1] // 32) * 32), np.uint8)
    padded[:, :allowed.shape[1]] = allowed
    return np.packbits(padded, axis=1, bitorder="little").view(np.uint32)


def edit(hip, x, rows, history, tokens, values, masks=None, in_place=False):
    lb = hip.buffer_from(x)
    out = lb if in_place else hip.buffer_from(np.full(x.size + 1, 7.0, np.float32))
    args = dict(history=history, bias_tokens=tokens, bias_values=values, masks=masks)
    views = {k: hip.buffer_from(v).at(0) for k, v in args.items() if v is not None and v.size}
    hip.begin()
    hip.logits_edit(lb.at(0), out.at(0), *x.shape, hip.buffer_from(rows).at(0), n_history=history.size,
                    n_bias=tokens.size, n_masks=0 if masks is None else masks.shape[0], **views)
    hip.end()
    got = hip.read(out.at(0), np.empty(x.size + (not in_place), np.float32))
    if not in_place:
        assert got[-1] == 7.0 and np.array_equal(hip.read(lb.at(0), np.empty_like(x)), x, equal_nan=True)
    return got[:x.size].reshape(x.shape)


def restate(x, rows, history, tokens, values, allowed=None):
    y, most = x.astype(np.float64), np.abs(x).astype(np.float64)
    biases = np.zeros(x.shape)
    for i, r in enumerate(rows):
        h = history[r["history_at"]:r["history_at"] + r["history_len"]]
        t, c = np.unique(h[h < x.shape[1]], return_counts=True)
        rho, alpha, beta = (float(r[k]) for k in ("repeat", "presence", "frequency"))
        z = y[i, t]
        y[i, t] = np.where(z > 0, z / rho, z * rho) - (alpha + beta * c)
        most[i, t] = np.maximum(np.abs(z) * max(rho, 1 / rho), np.abs(alpha) + np.abs(beta) * c) + np.abs(y[i, t])
        for j in range(r["bias_at"], r["bias_at"] + r["bias_len"]):
            if tokens[j] < x.shape[1]:
                y[i, tokens[j]] += values[j]
                most[i, tokens[j]] += np.abs(values[j])
                biases[i, tokens[j]] += 1
        if allowed is not None and r["mask"] != NO_MASK:
            y[i, ~allowed[r["mask"]] if r["mask"] < len(allowed) else slice(None)] = -np.inf
    return y, most * (5 + biases) * 2.0 ** -24


def check(got, want, bound):
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine].astype(np.float32), equal_nan=True)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


@pytest.mark.parametrize("n_rows,vocab,history,n_bias", [(1, 1, 3, 2), (1, 31, 0, 0), (3, 33, 50, 40), (2, 1000, 600, 0),
                                                         (5, 2048, 0, 300), (7, 2049, 700, 513), (2, 65536, 5000, 8),
                                                         (33, 7777, 300, 30), (3, 151936, 2000, 300)])
def test_matches_float64(hip, n_rows, vocab, history, n_bias):
    print("logits_edit", n_rows, vocab, history, n_bias, flush=True)
    rng = np.random.default_rng(vocab + n_rows)
    x = (4 * rng.standard_normal((n_rows, vocab))).astype(np.float32)
    h = [(vocab * rng.random(rng.integers(0, history + 1) if i else history) ** 3).astype(int) for i in range(n_rows)]
    b = [[(int(t), float(v)) for t, v in zip(rng.integers(0, vocab, n), rng.standard_normal(n))]
         for n in [n_bias] + [int(rng.integers(0, n_bias + 1)) for _ in range(n_rows - 1)]]
    allowed = rng.random((3, vocab)) < np.asarray([[0.95], [0.02], [0.0]])
    lists = rules(h, b, masks=[(0, 1, 2, NO_MASK)[i % 4] for i in range(n_rows)], repeat=rng.uniform(0.8, 1.5, n_rows),
                  presence=rng.uniform(-0.5, 1, n_rows), frequency=rng.uniform(-0.2, 0.5, n_rows))
    want, bound = restate(x, *lists, allowed)
    got = edit(hip, x, *lists, words(allowed))
    check(got, want, bound)
    assert np.array_equal(edit(hip, x, *lists, words(allowed), in_place=True), got)


def test_a_token_named_often(hip):
    """Counts past a byte's, and biases of one token added in list order: the f32 sum of a loop, bit for bit."""
    rng = np.random.default_rng(4)
    x = np.asarray([[1.5, -2.0, 0.0, 3.25]], np.float32)
    values = rng.standard_normal(700).astype(np.float32) * np.float32(10) ** rng.integers(-3, 4, 700)
    values = values.astype(np.float32)
    lists = rules([[3] * 70000 + [1]], [[(2, float(v)) for v in values]], repeat=1.0, presence=0.0, frequency=0.5)
    got = edit(hip, x, *lists)
    want = np.float32(0)
    for v in values:
        want = np.float32(want + v)
    assert got[0].tolist() == [1.5, -2.5, want, np.float32(3.25 - 35000.0)]


def test_rows_that_are_not_finite_and_entries_outside_the_lists(hip):
    x = np.asarray([[np.nan, np.inf, -np.inf, 2.0, -0.0], [1.0, 2.0, 3.0, 4.0, 5.0], [1.0, 2.0, 3.0, 4.0, 5.0]], np.float32)
    rows, history, tokens, values = rules([[0, 1, 2, 4, 9, 0xFFFFFFFF], [], []], [[(7, 1.0), (0xFFFFFFFF, 2.0)], [], []],
                                          masks=[NO_MASK, 0, 5], repeat=2.0, presence=0.0, frequency=0.0)
    allowed = np.asarray([[True, False, True, False, True]])
    got = edit(hip, x, rows, history, tokens, values, words(allowed))
    inf = np.inf
    assert np.array_equal(got, np.asarray([[np.nan, inf, -inf, 2, 0], [1, -inf, 3, -inf, 5], [-inf] * 5], np.float32),
                          equal_nan=True)
    # A masked NaN is masked; lists that run past their entries end there.
    rows["mask"] = 0
    rows["history_at"], rows["history_len"] = [2, 5, 0xFFFFFFFF], [0xFFFFFFFF, 100, 0xFFFFFFFF]
    rows["bias_at"], rows["bias_len"] = [0xFFFFFFFF, 1, 2], [3, 0xFFFFFFFF, 1]
    got = edit(hip, x, rows, history, tokens, values, words(~allowed))
    assert np.array_equal(got, np.asarray([[-inf, inf, -inf, 2, -inf]] + [[-inf, 2, -inf, 4, -inf]] * 2, np.float32))


def test_refusals(hip):
    b, rows = hip.new_buffer(4096), hip.buffer_from(np.zeros(4, LOGIT_ROW))

    def refused(status, *args, **kw):
        hip.begin()
        with pytest.raises(BobcatError) as e:
            hip.logits_edit(*args, **kw)
        hip.discard()
        assert e.value.status == STATUS[status], str(e.value)

    refused("Argument", b.at(0), b.at(2048), 1, 0, rows.at(0))
    refused("Argument", b.at(0), b.at(64), 1, 100, rows.at(0))      # half over the logits
    refused("Argument", b.at(64), b.at(0), 1, 100, rows.at(0))
    refused("Argument", b.at(2), b.at(2048), 1, 100, rows.at(0))
    refused("OutOfBounds", b.at(0), b.at(2048), 3, 256, rows.at(0))
    refused("OutOfBounds", b.at(0), b.at(2048), 5, 10, rows.at(0))  # of the rows
    refused("OutOfBounds", b.at(0), b.at(2048), 1, 33, rows.at(0), masks=b.at(4092), n_masks=1)
    refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_history=4)  # a list without a view
    refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_bias=4, bias_tokens=b.at(0))
    refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_history=(1 << 30) + 1, history=b.at(0))
    refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_bias=(1 << 30) + 1, bias_tokens=b.at(0), bias_values=b.at(0))
    refused("Argument", b.at(0), b.at(0), 1 << 23, 33, rows.at(0))
    # The outputs over each of the rules.
    refused("Argument", b.at(0), rows.at(64), 1, 10, rows.at(64))
    for at in (2048, 2048 + 4 * 32):
        refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_history=4, history=b.at(at))
        refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_bias=4, bias_tokens=b.at(at), bias_values=b.at(0))
        refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_bias=4, bias_tokens=b.at(0), bias_values=b.at(at))
        refused("Argument", b.at(0), b.at(2048), 1, 33, rows.at(0), n_masks=1, masks=b.at(at))
    hip.begin()
    hip.logits_edit(b.at(0), b.at(0), 0, 33, rows.at(0))
    hip.end()


def test_a_sampled_step_of_a_batch(hip):
    """Rows edited together, then sampled one by one: greedy picks the best allowed token of each."""
    rng = np.random.default_rng(12)
    n_rows, vocab = 4, 5000
    x = rng.standard_normal((n_rows, vocab)).astype(np.float32)
    best = x.argmax(1)
    allowed = np.ones((n_rows, vocab), bool)
    allowed[1, best[1]] = False
    rows, history, tokens, values = rules([[], [], [int(best[2])] * 3, []], [[], [], [], [(17, 50.0)]],
                                          masks=[NO_MASK, 1, NO_MASK, NO_MASK], repeat=1.0, presence=1.0, frequency=5.0)
    want, _ = restate(x, rows, history, tokens, values, allowed)
    xb, out = hip.buffer_from(x), hip.new_buffer(4 * n_rows)
    state = hip.buffer_from(np.zeros(1, np.uint64))
    lists = [hip.buffer_from(a).at(0) for a in (rows, history, tokens, values, words(allowed))]
    hip.begin()
    hip.logits_edit(xb.at(0), xb.at(0), n_rows, vocab, lists[0], history=lists[1], n_history=history.size,
                    bias_tokens=lists[2], bias_values=lists[3], n_bias=tokens.size, masks=lists[4], n_masks=n_rows)
    for i in range(n_rows):
        hip.sample(xb.floats(i * vocab), vocab, xb.at(0), 0, Sampling(0.0, 0, 1.0, 0.0, 1.0), state.at(0), out.at(4 * i))
    hip.end()
    got = hip.read(out.at(0), np.empty(n_rows, np.uint32))
    assert got.tolist() == want.argmax(1).tolist()
    assert got[0] == best[0] and got[1] != best[1] and got[3] == 17
