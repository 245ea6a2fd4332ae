"""GPU parity of bch_rope_paged with the definition in float64.

Bound: the angle is off by less than 2^-31 of a turn (bits left out) and two roundings of at most pi/4 (2^-24 each of it), in
all 1.0e-7; sine and cosine by their series' rest (2^-28) and four roundings; the magnitude, the product and the sum round
once each.  So an output is off by (a + b)·m·(1.7 + 4 + 3)·2^-24 < 9·2^-24·(a + b)·m of its pair.  A norm adds the sum of squares
(at most 8 + 5 roundings, half of it in the root), the root (2) and two products: 11·2^-24 more."""
from __future__ import annotations

import numpy as np
import pytest

from _drafts import as_given, chain, depths, random_tree, rope
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS
from bobcat_amd.backend import Hip, NormSpec, RopeRows, rope_frequencies, rope_spec

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


def plan_of(hip, past, new, hd, heads, kv, parents=None, page=512):
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    plan = hip.kv_plan("i8", kv, hd, page, max(1, sum(need)), heads)
    ends = np.cumsum([0] + need)
    plan.set(past, new, [range(a, b) for a, b in zip(ends, ends[1:])], parents=parents)
    return plan


def turned(hip, plan, spec, rows, norms=(None, None), frequencies=None, eps=1e-5, pad=0, gate=False):
    """rope_paged of (q, k) [tokens, heads, hd], out of and into rows with `pad` floats behind each; q with `gate` behind each
    head."""
    rope_ = hip.rope(spec.n_rot, spec.theta, layout=spec.layout, scaling=spec.scaling, factor=spec.factor,
                     n_original=spec.n_original, slow=spec.slow, fast=spec.fast, magnitude=spec.magnitude,
                     frequencies=frequencies)
    given, outs = [], []
    for x, norm, apart in zip(rows, norms, (2 if gate else 1, 1)):
        if x is None:
            given.append(None)
            outs.append(None)
            continue
        n, heads, hd = x.shape
        src = np.full((n, heads * apart * hd + pad), np.nan, np.float32)
        src[:, :heads * apart * hd].reshape(n, heads, apart * hd)[..., :hd] = x
        out = hip.buffer_from(np.full((n + 1, heads * hd + pad), 7.0, np.float32))
        weight = None if norm is None else NormSpec(hip.buffer_from(norm).at(0), eps)
        given.append(RopeRows(hip.buffer_from(src).at(0), src.shape[1], out.at(0), heads * hd + pad, heads, apart * hd, weight))
        outs.append(out)
    run(hip, lambda: hip.rope_paged(rope_, plan, *given))
    got = []
    for x, out in zip(rows, outs):
        if x is not None:
            n, heads, hd = x.shape
            y = hip.read(out.at(0), np.empty((n + 1, heads * hd + pad), np.float32))
            assert (y[-1] == 7.0).all() and (y[:, heads * hd:] == 7.0).all()  # nothing behind the rows
            got.append(y[:-1, :heads * hd].reshape(x.shape))
    return got


SPECS = [dict(n_rot=64), dict(n_rot=64, layout="pairs"), dict(n_rot=32, scaling="linear", factor=8.0), dict(n_rot=2),
         dict(n_rot=30, layout="pairs", scaling="parts", factor=16.0, n_original=4096, magnitude=1.25), dict(n_rot=12),
         dict(n_rot=20, layout="pairs"), dict(n_rot=62)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("spec", SPECS + [dict(n_rot="hd"), dict(n_rot="hd", layout="pairs"), dict(n_rot="hd - 2")])
def test_matches_the_definition(hip, hd, spec):
    rng = np.random.default_rng(hd)
    spec = dict(spec, n_rot=eval(str(spec["n_rot"]), dict(hd=hd)))
    c = rope_spec(spec.pop("n_rot"), 1e6, **spec)
    print("rope_paged", hd, spec, flush=True)
    trees = [chain(1), random_tree(rng, 19, roots=2), chain(0), chain(37), random_tree(rng, 5)]
    past, new = [0, 1000, 5, 131000, 15], [len(t) for t in trees]
    heads, kv = 6, 2
    q, k = (3 * rng.standard_normal((sum(new), h, hd)).astype(np.float32) for h in (heads, kv))
    norms = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    for parents in (None, trees):
        at = [p + d for p, t in zip(past, trees if parents else [chain(n) for n in new]) for d in depths(t)]
        plan = plan_of(hip, past, new, hd, heads, kv, parents and as_given(parents))
        for weights in ((None, None), tuple(norms), (norms[0], None)):
            got = turned(hip, plan, c, (q, k), weights, pad=4, gate=parents is None)
            for y, x, w in zip(got, (q, k), weights):
                want, size = rope(x, at, rope_frequencies(c), "pairs" if c.layout else "halves", c.magnitude, w, 1e-5)
                off = np.abs(y - want) / (size * STEP)
                assert off.max() <= (9 if w is None else 20), off.max()
                if w is None:
                    assert np.array_equal(y[..., c.n_rot:], x[..., c.n_rot:])


def test_far_positions_and_given_frequencies(hip):
    """Positions to 2^27 and frequencies of any size and sign: an angle in f32 would be off by whole turns."""
    rng, hd = np.random.default_rng(3), 64
    past, new = [(1 << 27) - 40, 99_999_991], [40, 3]
    at = [p + i for p, n in zip(past, new) for i in range(n)]
    plan = plan_of(hip, past, new, hd, 2, 1)
    q = rng.standard_normal((43, 2, hd)).astype(np.float32)
    c = rope_spec(64, 1e4)
    got, = turned(hip, plan, c, (q, None))
    # (float64 angles: t·f is off by 2^-53 of itself, 1.5e-8 radians at 2^27.)
    want, size = rope(q, at, rope_frequencies(c), "halves")
    assert (np.abs(got - want) / (size * STEP)).max() <= 9 + 0.3
    # Frequencies whose angles float64 holds exactly as parts of a turn: quarters, eighths, and whole turns.
    turns = np.array([0.0, 0.25, 0.5, 0.75, 1.0, 3.0, -0.25, 1.125, -2.0, 1 / 16] * 4)[:32]
    got, = turned(hip, plan, c, (q, None), frequencies=turns * 2 * np.pi)
    _, size = rope(q, [1], [0.0] * 32, "halves")
    for t, p in enumerate(at):
        angle = (p * turns) % 1.0 * 2 * np.pi
        a, b = q[t, :, :32].astype(np.float64), q[t, :, 32:].astype(np.float64)
        want = np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)
        own = np.tile(np.spacing(np.abs(turns) * 2 * np.pi) / 2 * p / STEP, 2)  # what a frequency's rounding makes of t·f
        assert (np.abs(got[t] - want) / (size[t] * STEP) <= 9 + own).all()


def test_in_place_and_side_by_side(hip):
    """Heads turned where they are, in rows that queries, keys and values share."""
    rng, hd, heads, kv = np.random.default_rng(5), 128, 4, 2
    past, new = [7, 300], [3, 18]
    rows = rng.standard_normal((21, (heads + 2 * kv) * hd)).astype(np.float32)
    plan, r = plan_of(hip, past, new, hd, heads, kv), hip.rope(hd, 1e4)
    width = rows.shape[1]
    b = hip.buffer_from(rows)
    at_k = b.floats(heads * hd)
    run(hip, lambda: hip.rope_paged(r, plan, RopeRows(b.at(0), width, b.at(0), width, heads), RopeRows(at_k, width, at_k, width, kv)))
    got = hip.read(b.at(0), np.empty_like(rows))
    f = rope_frequencies(rope_spec(hd, 1e4))
    at = [p + i for p, n in zip(past, new) for i in range(n)]
    for a, n in ((0, heads), (heads * hd, kv)):
        want, size = rope(rows[:, a:a + n * hd].reshape(21, n, hd), at, f, "halves")
        assert (np.abs(got[:, a:a + n * hd].reshape(21, n, hd) - want) <= 9 * STEP * size).all()
    assert np.array_equal(got[:, (heads + kv) * hd:], rows[:, (heads + kv) * hd:])


def test_what_is_not_finite_stays_in_its_pair(hip):
    rng, hd = np.random.default_rng(6), 64
    q = rng.standard_normal((2, 3, hd)).astype(np.float32)
    q[0, 1, 5], q[1, 2, 60] = np.nan, np.inf
    got, = turned(hip, plan_of(hip, [9], [2], hd, 3, 1), rope_spec(48, 1e4), (q, None))
    bad = ~np.isfinite(got)
    assert bad[0, 1, [5, 29]].all() and bad.sum() == 3 and got[1, 2, 60] == np.inf


def test_no_tokens(hip):
    plan, r = plan_of(hip, [4, 0], [0, 0], 64, 2, 1), hip.rope(64, 1e4)
    b = hip.buffer_from(np.full(64, 7.0, np.float32))
    run(hip, lambda: hip.rope_paged(r, plan, RopeRows(b.at(0), 128, b.at(0), 128, 2), None))
    run(hip, lambda: hip.rope_paged(r, plan, None, None))
    assert (hip.read(b.at(0), np.empty(64, np.float32)) == 7.0).all()


def test_refusals(hip):
    hd, plan = 64, plan_of(hip, [3], [5], 64, 2, 1)
    r, b, o = hip.rope(64, 1e4), hip.new_buffer(5 * 256 * 4), hip.new_buffer(5 * 256 * 4)
    good = RopeRows(b.at(0), 256, o.at(0), 128, 2)

    def refused(status, q=good, k=None, rope_=r, plan_=plan):
        hip.begin()
        with pytest.raises(BobcatError) as e:
            hip.rope_paged(rope_, plan_, q, k)
        hip.discard()
        assert e.value.status == STATUS[status], str(e.value)

    with pytest.raises(BobcatError) as e:
        hip.rope_paged(r, plan, good, None)
    assert e.value.status == STATUS["NotRecording"]
    refused("Argument", rope_=hip.rope(128, 1e4))                                  # more elements than a head has
    refused("Argument", RopeRows(b.at(0), 256, o.at(0), 128, 0))
    refused("Argument", RopeRows(b.at(0), 256, o.at(0), 128, 2, head_stride=60))
    refused("Argument", RopeRows(b.at(0), 256, o.at(0), 128, 2, head_stride=66))
    refused("Argument", RopeRows(b.at(0), 124, o.at(0), 128, 2))
    refused("Argument", RopeRows(b.at(0), 256, o.at(0), 126, 2))
    refused("Argument", RopeRows(b.at(8), 128, o.at(0), 128, 2))
    refused("OutOfBounds", RopeRows(b.at(0), 320, o.at(0), 128, 2))
    refused("OutOfBounds", RopeRows(b.at(0), 256, o.at(4096), 128, 2))
    refused("OutOfBounds", RopeRows(b.at(0), 256, o.at(0), 128, 2, norm=NormSpec(o.at(5 * 1024 - 16), 1e-5)))
    refused("Argument", RopeRows(b.at(0), 256, o.at(0), 128, 2, norm=NormSpec(o.at(0), 1e-5)))
    refused("Argument", RopeRows(b.at(0), 256, b.at(0), 128, 2))                   # another stride
    refused("Argument", RopeRows(b.at(0), 256, b.at(256), 256, 2))                 # half a row on
    refused("Argument", RopeRows(b.at(0), 256, b.at(0), 256, 2, head_stride=128))  # other places in a row
    refused("Argument", good, RopeRows(b.at(512), 256, o.at(256), 128, 1))         # over the queries' outputs
    refused("Argument", good, RopeRows(o.at(0), 128, b.at(512), 256, 1))           # over them while they are written
    with Hip() as other:
        refused("ForeignBuffer", rope_=other.rope(64, 1e4))
        refused("ForeignBuffer", plan_=plan_of(other, [3], [5], 64, 2, 1))
    with pytest.raises(BobcatError):
        hip.rope(4, 1e4, frequencies=[1.0, np.inf])
    with pytest.raises(BobcatError):
        hip.rope(4, 1e4, frequencies=[1.0])
    empty = hip.kv_plan("i8", 1, 64, 16, 1, 2)
    refused("Argument", plan_=empty)


def test_a_batch_that_no_l2_holds(hip):
    """More than 32 MiB of rows: they are written past the caches."""
    rng, hd, heads, kv = np.random.default_rng(8), 256, 30, 2
    past, new = [1000, 0], [600, 530]
    q, k = (rng.standard_normal((1130, h, hd)).astype(np.float32) for h in (heads, kv))
    c = rope_spec(128, 1e6)
    got = turned(hip, plan_of(hip, past, new, hd, heads, kv), c, (q, k))
    at = [p + i for p, n in zip(past, new) for i in range(n)]
    for y, x in zip(got, (q, k)):
        want, size = rope(x, at, rope_frequencies(c), "halves")
        assert (np.abs(y - want) / (size * STEP)).max() <= 9
        assert np.array_equal(y[..., 128:], x[..., 128:])
