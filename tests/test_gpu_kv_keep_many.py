"""bch_kv_keep over more sequences than a launch has workgroups."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import Pool
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS, check, lib
from test_gpu_kv_keep import run

pytestmark = pytest.mark.gpu


def test_more_sequences_than_a_launch_has_workgroups(hip):
    """2^24 sequences, all but the first without new tokens: refused as they are, moved in two calls."""
    n = 1 << 24
    past, new, pages = np.zeros(n, np.uint32), np.zeros(n, np.uint32), np.zeros(1, np.uint32)
    new[0] = 3
    plan = hip.kv_plan("f16", 1, 64, 16, 1, 1)
    check(lib().bch_kv_plan_set(plan.handle, n, past.ctypes.data, new.ctypes.data, pages.ctypes.data, 1))
    bytes_ = np.random.default_rng(5).integers(0, 256, 4096, np.uint8)
    cache, path = hip.buffer_from(bytes_), hip.buffer_from(np.array([0, 2, 2], np.uint32))
    kept = hip.new_buffer(4 * n)
    hip.write(kept.at(0), np.array([2], np.uint32))
    hip.begin()
    with pytest.raises(BobcatError) as e:
        hip.kv_keep(plan, 0, n, cache.at(0), 1, 0, kept.at(0), path.at(0))
    hip.discard()
    assert e.value.status == STATUS["Argument"], str(e.value)
    run(hip, lambda: (hip.kv_keep(plan, 0, n - 1, cache.at(0), 1, 0, kept.at(0), path.at(0)),
                      hip.kv_keep(plan, n - 1, 1, cache.at(0), 1, 0, kept.at(4 * (n - 1)), path.at(12))))
    got, want = hip.read(cache.at(0), np.empty(4096, np.uint8)).view(np.uint16), bytes_.view(np.uint16).copy()
    pool = Pool("f16", 1, 64, 16, 1)
    for part, at in ((0, pool.key_at), (1024, pool.value_at)):
        want[part + at[1]] = want[part + at[2]]
    assert np.array_equal(got, want)
