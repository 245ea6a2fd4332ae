"""Paged attention over value rows of very different size.  Rows of 8 bits have a
scale of their own each, and a row that is 2^16 to 2^34 times its neighbours but
that a query hardly sees takes nothing from the precision of what it does see:
each output is inside the bound of its own terms (tests/_paged_bounds.py),
whether the batch sends the query to a narrow tile or to a wide one."""
from __future__ import annotations

import numpy as np
import pytest

from _paged_bounds import LN2, case, excess, terms
from test_gpu_paged import attend, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,hd", [("i8", 64), ("f8", 64), ("i8", 128), ("f8", 128), ("i8", 256), ("f8", 256)])
@pytest.mark.parametrize("log_ratio", [16, 24, 34])
@pytest.mark.parametrize("seq,at", [((300, 40), 5), ((300, 40), 303), ((300, 1), 5)])
def test_values_of_negligible_weight(hip, fmt, hd, log_ratio, seq, at):
    """The key at `at` scores 60 (of base 2) below zero for every query, its value row is 2^log_ratio times the others."""
    say("attention_paged outliers", fmt, hd, log_ratio, seq, at)
    rng = np.random.default_rng(hd + log_ratio)
    pool, batch, q = case(rng, fmt, 4, 1, hd, 48, [seq])
    for s, position in [(0, i) for i in range(seq[0] + seq[1])]:  # the others' element 0 is 0
        k, v = (a.astype(np.float32) for a in pool.get(batch.pages[s][position // 48], position % 48))
        k[:, 0] = 0.0
        if position == at:
            k[:] = 0.0
            k[:, 0] = -60 * LN2 * np.sqrt(hd) / 8
            v *= np.float32(2.0 ** log_ratio)
        pool.put(batch.pages[s][position // 48], position % 48, k, v)
    q[..., 0] = 8.0
    got = attend(hip, pool, batch, 4, q)
    want, hard, rms = terms(q, *batch.gather(pool, 0), seq[0])
    worst, mean = excess(got, want, hard, rms)
    assert worst <= 1 and mean <= 1, (worst, mean)
