"""Infinities in f16 value rows: an element that a query sees makes that element
of its output NaN wherever it lies among the steps, and changes no other."""
from __future__ import annotations

import numpy as np
import pytest

from _paged_bounds import case
from test_gpu_paged import attend, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("past,new", [(40, 1), (620, 1), (620, 3), (300, 40), (0, 70)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, 70000.0])
def test_an_infinite_value_makes_its_element_nan(hip, hd, past, new, value):
    say("attention_paged infinite", hd, past, new, value)
    pool, batch, q = case(np.random.default_rng(hd), "f16", 4, 1, hd, 48, [(past, new)])
    before = attend(hip, pool, batch, 4, q)
    n = past + new
    spoilt = np.zeros((new, hd), bool)
    # The first position, one in the middle, the last one before the new tokens and one of those: an element each.
    for d, at in ((9, 0), (17, n // 2), (40, max(past - 1, 0)), (63, past + new // 2)):
        k, v = (a.astype(np.float32) for a in pool.get(batch.pages[0][at // 48], at % 48))
        v[:, d] = value
        pool.put(batch.pages[0][at // 48], at % 48, k, v)
        spoilt[max(at - past, 0):, d] = True
    after = attend(hip, pool, batch, 4, q)
    spoilt = np.broadcast_to(spoilt[:, None], after.shape)
    assert np.isnan(after[spoilt]).all()
    assert np.array_equal(after[~spoilt], before[~spoilt])
