"""Infinities in f16 rows: each is its element's alone in the cache, and one that
a query sees among its values makes that element of its output NaN, wherever it
lies among the steps, and changes no other."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import Batch, Pool
from _paged_bounds import case
from test_gpu_paged import attend, plan_of, say

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


def test_f16_rows_read_back_element_by_element(hip):
    """A NaN or an infinity is that element's alone, also one that comes from a finite number past f16's end."""
    rng = np.random.default_rng(6)
    kv, hd, page = 2, 64, 16
    batch = Batch(rng, [(0, 20)], page)
    pool = Pool("f16", kv, hd, page, batch.n_pages)
    x = rng.standard_normal((20, kv, hd)).astype(np.float32)
    x[3, 0, 5], x[4, 1, 6], x[5, 0, 7], x[6, 1, 8], x[7, 0, 9] = np.nan, np.inf, -np.inf, 65520.0, 65519.0
    cache, plan, xb = hip.buffer_from(pool.bytes), plan_of(hip, pool, batch, kv), hip.buffer_from(x)
    out = [hip.new_buffer(x.nbytes) for _ in range(2)]
    hip.begin()
    hip.kv_store(plan, cache.at(0), xb.at(0), kv * hd, xb.at(0), kv * hd)
    hip.kv_load(plan, cache.at(0), 0, 0, 20, out[0].at(0), out[1].at(0))
    hip.end()
    with np.errstate(over="ignore"):
        want = x.astype(np.float16).astype(np.float32)
    assert np.isinf(want).sum() == 3 and np.isnan(want).sum() == 1
    for buffer in out:
        assert np.array_equal(hip.read(buffer.at(0), np.empty_like(x)), want, equal_nan=True)
