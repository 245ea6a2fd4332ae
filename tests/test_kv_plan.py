"""CPU checks of the paged cache's plans: every batch that would let a kernel
read or write outside its pages, or two sequences write one, is refused on the
host; what is allowed passes.  No device is needed."""
from __future__ import annotations

import ctypes as C

import pytest

from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS, lib
from bobcat_amd.backend import kv_page_bytes, kv_plan_check, kv_shape

SHAPE = kv_shape("i8", 2, 64, 32, 10)


def refused(status, shape=SHAPE, heads=8, past=(40,), new=(3,), pages=((4, 7),)):
    with pytest.raises(BobcatError) as e:
        kv_plan_check(shape, heads, past, new, pages)
    assert e.value.status == STATUS[status], str(e.value)


@pytest.mark.parametrize("fmt,kv,hd,page,want", [
    ("f16", 1, 64, 16, 4096), ("i8", 1, 64, 16, 2176), ("f8", 8, 128, 48, 8 * 3 * 4224), ("f16", 2, 256, 512, 2 * 32 * 16384)])
def test_page_bytes(fmt, kv, hd, page, want):
    assert kv_page_bytes(kv_shape(fmt, kv, hd, page, 1)) == want


@pytest.mark.parametrize("args", [(3, 2, 64, 32, 10), (1, 0, 64, 32, 10), (1, 257, 64, 32, 10), (1, 2, 96, 32, 10),
                                  (1, 2, 64, 0, 10), (1, 2, 64, 24, 10), (1, 2, 64, 528, 10), (1, 2, 64, 32, 0)])
def test_shapes_that_are_refused(args):
    shape = kv_shape(*args)
    assert kv_page_bytes(shape) == 0
    with pytest.raises(BobcatError):
        kv_plan_check(shape, 8, [], [], [])


@pytest.mark.parametrize("heads", [0, 3, 66])
def test_head_groups_that_are_refused(heads):
    refused("AttentionLimits", heads=heads)


def test_batches_that_are_refused():
    refused("OutOfBounds", pages=((4, 10),))
    refused("OutOfBounds", pages=((4, 0xFFFFFFFF),))
    refused("Argument", pages=((4,),))
    refused("Argument", pages=((4, 7, 8),))
    refused("Argument", past=(0,), new=(0,), pages=((1,),))
    refused("Argument", past=(0x3FFFFFFF,), new=(1,), pages=((),))
    refused("Argument", past=(0xFFFFFFFF,), new=(0xFFFFFFFF,), pages=((),))
    # A page that receives tokens, named twice: by two sequences, by one, and as another's prefix.
    refused("Argument", past=(40, 0), new=(3, 5), pages=((4, 7), (7,)))
    refused("Argument", past=(0,), new=(40,), pages=((4, 4),))
    refused("Argument", past=(40, 32), new=(3, 0), pages=((4, 7), (7,)))


def test_batches_that_no_launch_could_take():
    shape = kv_shape("i8", 2, 64, 512, 1 << 20)
    kv_plan_check(shape, 8, [1 << 27], [0], [range(1 << 18)])
    kv_plan_check(shape, 8, [0], [1 << 23], [range(1 << 14)])
    refused("Argument", shape, 8, [1 << 27], [1], [range((1 << 18) + 1)])
    refused("Argument", shape, 8, [0, 0], [1 << 23, 1], [range(1 << 14), [1 << 14]])


def test_batches_that_are_allowed():
    kv_plan_check(SHAPE, 8, [], [], [])
    kv_plan_check(SHAPE, 64, [0], [0], [[]])
    kv_plan_check(SHAPE, 8, [31], [2], [[9, 0]])
    # A shared prefix: only read by both.
    kv_plan_check(SHAPE, 8, [64, 33, 64], [1, 3, 0], [[1, 2, 3], [1, 4], [1, 2]])
    # A page number does not cost the memory of the cache's pages.
    kv_plan_check(kv_shape("i8", 2, 64, 32, 0xFFFFFFFF), 8, [5], [1], [[0xFFFFFFF0]])


def test_null_arguments():
    some = (C.c_uint32 * 1)(1)
    assert lib().bch_kv_page_bytes(None) == 0
    assert lib().bch_kv_plan_check(None, 8, 0, None, None, None, 0) == STATUS["Argument"]
    assert lib().bch_kv_plan_check(C.byref(SHAPE), 8, 1, None, None, None, 0) == STATUS["Argument"]
    assert lib().bch_kv_plan_check(C.byref(SHAPE), 8, 1, some, some, None, 1) == STATUS["Argument"]
    assert lib().bch_kv_plan_new(None, C.byref(SHAPE), 8, None) == STATUS["Argument"]
    out = C.c_void_p(1)
    assert lib().bch_kv_plan_new(None, C.byref(SHAPE), 8, C.byref(out)) == STATUS["Argument"]
    assert out.value is None
    assert lib().bch_kv_plan_set(None, 0, None, None, None, 0) == STATUS["Argument"]
    lib().bch_kv_plan_free(None)
