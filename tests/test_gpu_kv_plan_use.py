"""When a plan's batch may be given: not while recorded or running work reads
it, and at any other time, inside an open recording too."""
from __future__ import annotations

import numpy as np
import pytest

from _paged_bounds import case
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS
from test_gpu_paged import attend, plan_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def setup(hip):
    pool, batch, q = case(np.random.default_rng(1), "i8", 4, 2, 64, 16, [(20, 3)])
    return pool, batch, q, hip.buffer_from(pool.bytes), hip.new_buffer(1 << 16), plan_of(hip, pool, batch, 4)


def give(plan, batch):
    plan.set(batch.past, batch.new, batch.pages)


def busy(plan, batch):
    with pytest.raises(BobcatError) as e:
        give(plan, batch)
    assert e.value.status == STATUS["Busy"]


def test_refused_calls_do_not_use_the_plan(hip, setup):
    pool, batch, q, cache, b, plan = setup
    refused = [lambda: hip.kv_load(plan, cache.at(0), 1, 0, 1, b.at(0), b.at(1 << 15)),
               lambda: hip.kv_load(plan, cache.at(0), 0, 0, 2, b.at(0), b.at(16)),
               lambda: hip.kv_store(plan, cache.at(0), b.at(8), 128, b.at(0), 128),
               lambda: hip.attention_paged(plan, cache.at(0), b.at(0), 252, b.at(1 << 15), 256),
               lambda: hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(0), 256)]
    hip.begin()
    try:
        for call in refused:
            with pytest.raises(BobcatError):
                call()
            give(plan, batch)
    finally:
        hip.discard()
    # With no recording open every call is refused, and the next recording finds the plan unused.
    with pytest.raises(BobcatError) as e:
        hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(1 << 15), 256)
    assert e.value.status == STATUS["NotRecording"]
    hip.begin()
    give(plan, batch)
    hip.discard()


def test_a_discarded_recording_does_not_hold_the_plan(hip, setup):
    pool, batch, q, cache, b, plan = setup

    def use():
        hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(1 << 15), 256)

    hip.begin()
    use()
    hip.discard()
    hip.begin()  # nothing in this one reads the plan
    give(plan, batch)
    use()
    busy(plan, batch)
    first = hip.commit()
    busy(plan, batch)
    hip.begin()
    busy(plan, batch)  # the committed one still runs, as far as the host knows
    hip.wait(first)
    give(plan, batch)
    use()
    hip.discard()
    hip.begin()
    ticket = hip.commit()  # without the plan
    give(plan, batch)
    hip.wait(ticket)
    assert np.array_equal(attend(hip, pool, batch, 4, q, plan=plan), attend(hip, pool, batch, 4, q))


def test_one_plan_for_the_layers_of_a_step(hip):
    """Two layers' caches as views of one buffer, and two plans, in one recording."""
    rng = np.random.default_rng(4)
    pool, batch, q = case(rng, "i8", 4, 2, 64, 16, [(40, 1), (700, 2)])
    other, other_batch, other_q = case(rng, "i8", 4, 2, 64, 16, [(900, 1)])
    second = pool.bytes.copy()
    second[..., :2 * 16 * 64] ^= 1  # other keys and values
    size = pool.bytes.nbytes
    cache, other_cache = hip.buffer_from(np.concatenate([pool.bytes.reshape(-1), second.reshape(-1)])), hip.buffer_from(other.bytes)
    want = attend(hip, pool, batch, 4, q), None, attend(hip, other, other_batch, 4, other_q)
    pool.bytes = second
    want = want[0], attend(hip, pool, batch, 4, q), want[2]
    plan, other_plan = plan_of(hip, pool, batch, 4), plan_of(hip, other, other_batch, 4)
    qb, ob = hip.buffer_from(q), hip.buffer_from(other_q)
    outs = [hip.new_buffer(q.nbytes), hip.new_buffer(q.nbytes), hip.new_buffer(other_q.nbytes)]
    hip.begin()
    hip.attention_paged(plan, cache.at(0), qb.at(0), 256, outs[0].at(0), 256)
    hip.attention_paged(other_plan, other_cache.at(0), ob.at(0), 256, outs[2].at(0), 256)
    hip.attention_paged(plan, cache.at(size), qb.at(0), 256, outs[1].at(0), 256)
    hip.end()
    for out, w in zip(outs, want):
        assert np.array_equal(hip.read(out.at(0), np.empty_like(w)), w)
