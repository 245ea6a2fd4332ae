"""CPU checks of the paged attention's tolerances: the kernels' arithmetic is
inside them, and the mistakes that they are there for are not — a key left
out at either end of a long context, queries or probabilities in one f16 part."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import attention
from _paged_bounds import case, excess, restated, terms

CASES = [("i8", 4, 2, 64, 16, (600, 1)), ("f16", 4, 1, 64, 48, (1029, 2)), ("f8", 2, 1, 128, 32, (700, 2)),
         ("i8", 2, 1, 256, 64, (1029, 1)), ("f16", 2, 1, 256, 32, (300, 3))]


def inputs(fmt, heads, kv, hd, page, seq):
    pool, batch, q = case(np.random.default_rng(hd + seq[0]), fmt, heads, kv, hd, page, [seq])
    return (q, *batch.gather(pool, 0), seq[0])


@pytest.mark.parametrize("args", CASES)
def test_the_arithmetic_is_inside(args):
    q, k, v, past = inputs(*args)
    want, hard, rms = terms(q, k, v, past)
    assert np.abs(want - attention(q, k, v, past)).max() < 1e-12
    worst, mean = excess(restated(q, k, v, past), want, hard, rms)
    assert worst <= 1 and mean <= 1


@pytest.mark.parametrize("args", CASES)
@pytest.mark.parametrize("mistake", [dict(drop=0), dict(drop=-1), dict(query_parts=1), dict(p_parts=1)])
def test_mistakes_are_outside(args, mistake):
    q, k, v, past = inputs(*args)
    worst, mean = excess(restated(q, k, v, past, **mistake), *terms(q, k, v, past))
    assert max(worst, mean) > 1, (worst, mean)
