"""Paged attention against float64 inside the bounds of each output's own terms
(tests/_paged_bounds.py): on contexts long enough that keys are split among
waves, steps, workgroups and launches, a key that is left out at a border or a
part of a query or probability that is lost does not pass
(tests/test_paged_bounds.py)."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import Batch, Pool, attention
from _paged_bounds import case, excess, terms
from test_gpu_paged import FORMATS, attend, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (4, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("seqs,page", [([(1029, 1)], 64), ([(700, 1), (31, 1), (32, 1), (1000, 1)], 16),
                                       ([(1000, 3), (40, 4)], 48), ([(0, 17), (500, 5), (33, 2)], 32),
                                       ([(900, 40)], 128), ([(0, 70), (600, 33)], 16)])
def test_outputs_are_close(hip, fmt, heads, kv, hd, seqs, page):
    say("attention_paged close", fmt, heads, kv, hd, seqs, page)
    pool, batch, q = case(np.random.default_rng(hd + page), fmt, heads, kv, hd, page, seqs)
    got, row = attend(hip, pool, batch, heads, q), 0
    for s, (past, new) in enumerate(seqs):
        worst, mean = excess(got[row:row + new], *terms(q[row:row + new], *batch.gather(pool, s), past))
        assert worst <= 1 and mean <= 1, (s, worst, mean)
        row += new


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("past,new", [(1024, 1), (1000, 3), (1000, 40)])
def test_probabilities_of_long_contexts(hip, fmt, hd, past, new):
    """Key i has 64 in element i % hd alone and value i has 1 there: output element d is the summed probability of n/hd
    equal keys, split among waves, steps and workgroups.  A score s is off by s·(2^-22 + 8·2^-24) (the query's two parts
    and eight f32 roundings) and by 64·2^-25 for the end of its low part; a probability by twice the largest of that and
    2^-22 for its parts.  All terms of the sums are positive, so a rounding is one of 2^-24 of the whole: fewer than 48 for
    a step, the waves and the pieces, and three for each of n/32 steps, 48 + n/8 with those of the products."""
    say("attention_paged probabilities", fmt, hd, past, new)
    rng = np.random.default_rng(past + new)
    page, n = 64, past + new
    batch = Batch(rng, [(past, new)], page)
    pool = Pool(fmt, 1, hd, page, batch.n_pages)
    eye = np.eye(hd, dtype=np.float32)
    for i in range(n):
        pool.put(batch.pages[0][i // page], i % page, 64 * eye[None, i % hd], eye[None, i % hd])
    q = rng.standard_normal((new, 4, hd)).astype(np.float32)
    got, (k, v) = attend(hip, pool, batch, 4, q), batch.gather(pool, 0)
    want = attention(q, k, v, past)
    size = 64 / np.sqrt(hd) * np.abs(q).max()
    bound = 2 * (size * (2.0 ** -22 + 8 * 2.0 ** -24) + 64 * 2.0 ** -25) + 2.0 ** -22 + (48 + n / 8) * 2.0 ** -24
    assert (np.abs(got - want) <= bound * want + n / hd * 2.0 ** -33).all()
