"""CPU checks of the page lists that Python hands to a plan: each sequence's own
list has its own number of pages, and numbers are whole and in range."""
from __future__ import annotations

import numpy as np
import pytest

from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS
from bobcat_amd.backend import kv_plan_check, kv_shape

SHAPE = kv_shape("i8", 2, 64, 32, 10)


@pytest.mark.parametrize("pages", [[[4, 7], [1]],         # one too many and one too few
                                   [[4, 7, 1]], [[4], [7], [1]], [[], [4, 7, 1]]])
def test_lists_of_other_sequences(pages):
    """Three pages for sequences of one and two: their sum alone says nothing."""
    kv_plan_check(SHAPE, 8, [20, 40], [3, 1], [[4], [7, 1]])
    with pytest.raises(BobcatError) as e:
        kv_plan_check(SHAPE, 8, [20, 40], [3, 1], pages)
    assert e.value.status == STATUS["Argument"]


def test_long_batches():
    past, new = [40] * 20, [1] * 20
    pages = [[i % 5, 5 + i % 5] for i in range(20)]
    with pytest.raises(BobcatError):
        kv_plan_check(SHAPE, 8, past, new, pages[:-2] + [[1], [2, 3, 4]])


@pytest.mark.parametrize("number", [1.5, -1, 2 ** 32 + 1])
def test_numbers_that_are_refused(number):
    """As Python's numbers and as arrays', whose 2^32 + 1 would else be 1."""
    for bad in (number, np.asarray(number)[()]):
        for past, new, page in ((bad, 1, 4), (1, bad, 4), (1, 1, bad)):
            with pytest.raises(ValueError):
                kv_plan_check(SHAPE, 8, [past], [new], [[page]])
    for past, new, page in ((number, 1, 4), (1, number, 4), (1, 1, number)):
        with pytest.raises(ValueError):
            kv_plan_check(SHAPE, 8, np.asarray([past]), np.asarray([new]), [np.asarray([page])])


def test_arrays():
    kv_plan_check(SHAPE, 8, np.asarray([20, 40]), np.asarray([3, 1], np.uint8), [np.asarray([4]), np.asarray([7, 1], np.int32)])
    kv_plan_check(SHAPE, 8, np.empty(0, np.uint32), [], [])


def test_iterators_and_single_numbers():
    """Lists that can be gone through once, rows of an array, and a single sequence's lengths."""
    kv_plan_check(SHAPE, 8, [20, 40], [3, 1], iter([[4], [7, 1]]))
    kv_plan_check(SHAPE, 8, [20, 40], [3, 1], (iter(p) for p in ([4], [7, 1])))
    kv_plan_check(SHAPE, 8, (33, 34), (1, 1), np.asarray([[1, 2], [3, 4]]))
    kv_plan_check(SHAPE, 8, 20, 3, [[4]])
    kv_plan_check(SHAPE, 8, np.uint32(20), np.int64(3), [[4]])
    with pytest.raises(ValueError):
        kv_plan_check(SHAPE, 8, np.asarray([[20]]), np.asarray([[3]]), [[4]])
