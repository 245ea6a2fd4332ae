"""What bch_verify_drafts makes of the last that is left: of the target where all of it was drafted."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import chain, random_tree, verify
from bobcat_amd.backend import NO_TOKEN
from test_gpu_verify import case, plan_of, verdict

pytestmark = pytest.mark.gpu

BELOW_1 = np.nextafter(np.float32(1), np.float32(0))


@pytest.mark.parametrize("vocab,places", [(64, (5, 40)), (64, (40, 5)), (9000, (4100, 17)), (9000, (8999, 0, 4096)),
                                          (9000, (8000, 4095, 4097, 1))])
def test_children_that_are_all_the_target_has(hip, vocab, places):
    """Rows (as a grammar leaves them) whose few tokens are all drafted, and uniforms that reject them all but for
    roundings: where none stays nothing is left of p, and the draw is from p itself."""
    rng = np.random.default_rng(len(places) + vocab)
    n, kids = 2000, len(places)
    trees = [[-1] + [0] * kids] * n
    logits = rng.standard_normal((n, kids + 1, vocab)).astype(np.float32)
    logits[:, 0] = -np.inf
    depth = np.concatenate([np.zeros((n, 1)), rng.uniform(0.5, 14, (n, kids - 1))], 1)
    logits[:, 0, list(places)] = -depth.astype(np.float32)
    heat = rng.uniform(0.3, 2, n).astype(np.float32)
    tokens = np.tile(np.array([0, *places], np.uint32), n)
    u = np.full((n, kids + 1), BELOW_1, np.float32)
    u[:, 0] = rng.random(n, np.float32)
    got = verdict(hip, plan_of(hip, trees), trees, logits.reshape(-1, vocab), None, tokens, u.reshape(-1), heat)
    assert (got[2] != NO_TOKEN).all() and (got[2] < vocab).all()
    none = got[0] == 1
    assert none.any()
    # p of the places in token order; a draw further than 2^-20 from its borders (64 times an f32 term's roundings) is certain.
    order = np.argsort(places)
    p = np.exp(-depth.astype(np.float32).astype(np.float64) / heat[:, None].astype(np.float64))[:, order]
    up = np.cumsum(p / p.sum(1, keepdims=True), 1)
    want = np.array(places)[order][(u[:, :1] >= up[:, :-1]).sum(1)]
    sure = none & (np.abs(up[:, :-1] - u[:, :1]) > 2.0 ** -20).all(1)
    assert sure.sum() > none.sum() // 2 and (got[2][sure] == want[sure]).all()
    chances = got[3].reshape(n, kids + 1)[none, 0]
    assert (chances > 0).all()


@pytest.mark.parametrize("masses", [(0.5, 0.5), (0.75, 0.25), (0.25, 0.25, 0.125, 0.25, 0.0625, 0.0625)])
@pytest.mark.parametrize("vocab", [40, 5000])
def test_a_draft_whose_tokens_are_all_drawn(hip, masses, vocab):
    """A draft of a few tokens, drawn without replacement to the last, whose f32 probabilities sum to just over 1: the last
    one has all of the draft that is left, whatever the rounded sums of the others say.  Its row normalised in f64 is the
    definition's.  (Tests lie 0.1 and more from their borders, draws by chance: 2^-20 each, with fixed seeds.)"""
    rng = np.random.default_rng(vocab + len(masses))
    few = len(masses) + 1
    tree, n = [-1] + [0] * few, 64
    q = np.zeros((n, few + 1, vocab), np.float32)
    x = np.stack([rng.permutation(vocab)[:few] for _ in range(n)])
    logits = rng.standard_normal((n, few + 1, vocab)).astype(np.float32)
    u = np.full((n, few + 1), 0.9, np.float32)
    for i in range(n):
        q[i, 0, x[i, :-1]] = masses
        q[i, 0, x[i, -2]] = np.nextafter(np.float32(masses[-1]), np.float32(1))
        q[i, 0, x[i, -1]] = 2.0 ** -30
        q[i, 1:] = 1 / vocab
        # The target: next to nothing of the first; of the last less than c·q leaves, or half of all.
        logits[i, 0, x[i, :-1]] = -9
        others = np.delete(logits[i, 0].astype(np.float64), x[i, -1])
        logits[i, 0, x[i, -1]] = -40 if i % 2 else np.log(np.exp(others).sum())
    u[1::2, -1], u[::2, -1] = 0.0, 0.3  # the last: rejected with any uniform; kept with half of what is left
    u[:, 0] = rng.random(n, np.float32)
    tokens = np.concatenate([np.zeros((n, 1)), x], 1).astype(np.uint32).reshape(-1)
    heat = np.ones(n, np.float32)
    got = verdict(hip, plan_of(hip, [tree] * n), [tree] * n, logits.reshape(-1, vocab), q.reshape(-1, vocab), tokens, u.reshape(-1),
                  heat, True)
    for i in range(n):
        row = q[i].astype(np.float64)
        assert row[0].sum() > 1
        kept, path, token, _ = verify(tree, logits[i], row / row.sum(1, keepdims=True), tokens[i * (few + 1):][:few + 1], u[i], 1.0,
                                      True)
        assert kept == (1 if i % 2 else 2)
        assert got[0][i] == kept and got[1][i * (few + 1):][:few + 1].tolist() == path and got[2][i] == token, i


def term_errors(logits, temperature):
    """What the sum of a row's exponentials may be off by, relative to it: its terms are f32, the sum is f64.  A term 2^-a of
    the largest is off by two roundings of its exponent (the difference and the product: 2·a·ln 2·2^-24 of the term) and by two
    exponentials (to the piece's largest and from there to the row's) of at most 2^-23 each."""
    x = (logits.astype(np.float64) - logits.max()) / np.float64(temperature)
    p = np.exp(x)
    return (p * (2 * -x + 4)).sum() / p.sum() * 2.0 ** -24


@pytest.mark.parametrize("vocab", [4096, 4095, 12288, 12289])
def test_sums_of_terms_far_apart(hip, vocab):
    """Each piece has 256 tokens of weight 1 and else tokens of 0.98·2^-24, which an f32 sum of 1 and more loses: 14.7 of 15
    roundings for each of the former."""
    stride = 4 if vocab % 4 == 0 else 1  # (where rows are read four at a time, a thread's first are four apart)
    heavy = (np.arange(vocab) % 4096 < 256 * stride) & (np.arange(vocab) % stride == 0)
    row = np.where(heavy, 0, np.log(0.98 * 2.0 ** -24)).astype(np.float32)
    trees, n = [[-1, 0, 0]] * 3, 9
    logits = np.tile(row, (n, 1))
    tokens = np.tile(np.array([0, 8, 9], np.uint32), 3)
    got = verdict(hip, plan_of(hip, trees), trees, logits, None, tokens, np.full(n, 0.5, np.float32), np.ones(3, np.float32))
    p = np.exp(row.astype(np.float64))
    want = p[tokens] / p.sum()
    bound = term_errors(row, 1.0) + 2.0 ** -24  # (and the chance's own rounding)
    assert bound < 6 * 2.0 ** -24
    chances = got[3].reshape(3, 3)[:, 1:]
    assert (np.abs(chances / want.reshape(3, 3)[:, 1:] - 1) <= bound).all()


@pytest.mark.parametrize("spread", [1.0, 0.1, 0.01, 0.001, 0.0003])
@pytest.mark.parametrize("vocab,n", [(5000, 96), (70001, 24)])
def test_draws_from_what_a_rejection_leaves(hip, vocab, n, spread):
    """After a rejection the draw is from (p - q)+ / S, each term the difference of two f32 numbers: p·(1 ± E' ± s), where E'
    is a term's own error with two more roundings (of 1 / sum and of the product; term_errors has as many for the second
    exponential that these terms do not have) and s the sum's, q·2^-24 and the difference's own rounding.  So partial sums and S
    are off by e = 2·term_errors + 2·2^-24, and a place among them by 2·e / S: the token's range holds the uniform, taken
    that much wider.  S goes down to about 10^-4 here, where 2^-22 of a border would not hold."""
    rng = np.random.default_rng(vocab)
    logits = (2 * rng.standard_normal((n, 2, vocab))).astype(np.float32)
    heat = rng.uniform(0.6, 1.4, n).astype(np.float32)
    x = logits[:, 0].astype(np.float64) / heat[:, None]
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    q = p * np.exp(spread * rng.standard_normal(p.shape))
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    draft = np.zeros((n, 2, vocab), np.float32)
    draft[:, 0] = q
    child = (q / p).argmax(1)  # rejected: q is some standard deviations above p there
    tokens = np.stack([np.zeros(n), child], 1).astype(np.uint32).reshape(-1)
    u = np.stack([rng.random(n, np.float32), np.full(n, BELOW_1)], 1).astype(np.float32)
    trees = [[-1, 0]] * n
    got = verdict(hip, plan_of(hip, trees), trees, logits.reshape(-1, vocab), draft.reshape(-1, vocab), tokens, u.reshape(-1), heat)
    assert (got[0] == 1).all()
    smallest = 1.0
    for i in range(n):
        rest = np.maximum(p[i] - q[i].astype(np.float64), 0)
        s = rest.sum()
        off = 2 * (2 * term_errors(logits[i, 0], heat[i]) + 2 * 2.0 ** -24) / s
        up, t = np.cumsum(rest) / s, int(got[2][i])
        assert t < vocab and (up[t - 1] if t else 0) - off <= u[i, 0] <= up[t] + off, (i, s, off)
        assert abs(got[3][2 * i] - p[i, t]) <= (term_errors(logits[i, 0], heat[i]) + 2.0 ** -24) * p[i, t]
        smallest = min(smallest, s)
    assert smallest < spread


@pytest.mark.parametrize("mode", ["drawn", "distinct", "chosen"])
@pytest.mark.parametrize("vocab", [262144, 262145, 600001])
def test_vocabularies_of_more_pieces_than_lanes(hip, mode, vocab):
    """64 pieces of 4,096 tokens, one more, and 147: sums in several rounds, and lanes that have several pieces each.  (Logits
    spread so that some tens of tokens hold nearly all of p: a draw within 2^-20 of a border is a matter of one in 10^4.)"""
    rng = np.random.default_rng(vocab)
    trees = [random_tree(rng, 7, width=3), chain(4), [-1], random_tree(rng, 5, width=4)]
    logits, q, tokens, u, heat = case(rng, trees, vocab, mode, spread=6.0)
    heat[1] = 0.0 if mode == "chosen" else heat[1]
    got, row, beyond = verdict(hip, plan_of(hip, trees), trees, logits, q, tokens, u, heat, mode == "distinct"), 0, 0
    for i, t in enumerate(trees):
        part = slice(row, row + len(t))
        kept, path, token, chances = verify(t, logits[part], None if q is None else q[part], tokens[part], u[part], heat[i],
                                            mode == "distinct")
        assert got[0][i] == kept and got[1][part].tolist() == path and got[2][i] == token, (i, t)
        for j, a in enumerate(t):
            of = path[kept - 1] if j == 0 else a
            off = term_errors(logits[row + of], heat[i]) + 2.0 ** -24 if heat[i] > 0 else 0
            assert abs(got[3][row + j] - chances[j]) <= off * chances[j] + 1e-37, (i, j)
        beyond += token >= 64 * 4096
        row += len(t)
    assert beyond > 0 or vocab < 300000


def test_draws_in_every_piece(hip):
    """Next tokens all over a vocabulary of 600,001: of each piece two tokens hold the same mass, a uniform for each."""
    vocab, piece = 600001, 4096
    places = np.array([at + d for at in range(0, vocab, piece) for d in (0, min(piece, vocab - at) - 1)])
    row = np.full(vocab, -np.inf, np.float32)
    row[places] = 1.5
    n = 49  # (rows of 2.4 MB each)
    for first in range(0, places.size, n):
        some = np.arange(first, min(first + n, places.size))
        u = ((some + 0.5) / places.size).astype(np.float32)
        trees = [[-1]] * some.size
        got = verdict(hip, plan_of(hip, trees), trees, np.tile(row, (some.size, 1)), None, np.zeros(some.size, np.uint32), u,
                      np.ones(some.size, np.float32))
        assert np.array_equal(got[2], places[some])
