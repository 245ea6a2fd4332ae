"""What bch_verify_drafts makes of the last that is left: of the target where all of it was drafted."""
from __future__ import annotations

import numpy as np
import pytest

from bobcat_amd.backend import NO_TOKEN
from test_gpu_verify import plan_of, verdict

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
