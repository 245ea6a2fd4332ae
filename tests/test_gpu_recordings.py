"""Recordings queued behind each other share an event; what bch_wait says of their time stays sound, whatever is waited
for, discarded or left open in between."""
from __future__ import annotations

import numpy as np
import pytest

from bobcat_amd.backend import Hip

pytestmark = pytest.mark.gpu

N = 1 << 22


@pytest.fixture
def own():
    with Hip() as h:
        yield h


def work(h, b, times):
    for _ in range(times):
        h.copy(b.at(0), b.at(4 * N), N)


def test_times_of_queued_recordings(own):
    b = own.new_buffer(8 * N)
    tickets = []
    for i in range(12):
        own.begin()
        work(own, b, 20 if i % 3 else 0)
        tickets.append(own.commit())
    times = [own.wait(t) for t in tickets]
    # Each copy moves 32 MiB: no card does that in 2 us, and none takes 10 ms.
    for i, s in enumerate(times):
        assert 0 <= s < 0.2 and (i % 3 == 0 or s > 20 * 2e-6), times


def test_waits_discards_and_open_recordings_in_any_order(own):
    rng = np.random.default_rng(3)
    b = own.new_buffer(8 * N)
    tickets, open_ = [], False
    for step in range(400):
        what = rng.integers(5)
        if what <= 1 and not open_:
            own.begin()
            open_ = True
        elif what == 2 and open_:
            work(own, b, int(rng.integers(3)))
            tickets.append(own.commit())
            open_ = False
        elif what == 3 and open_:
            work(own, b, int(rng.integers(3)))
            own.discard()
            open_ = False
        elif what == 4 and tickets:
            assert 0 <= own.wait(tickets[int(rng.integers(len(tickets)))]) < 1
    if open_:
        own.discard()
    own.begin()
    work(own, b, 3)
    assert 3 * 2e-6 < own.end() < 1
