"""CPU checks of plans with trees and of rotary specs: what a launch could not run on is refused on the host, and the
frequencies are the definition's.  No device is needed."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS, RopeSpec, lib
from bobcat_amd.backend import NO_PARENT, kv_plan_check, kv_shape, rope_frequencies, rope_spec

SHAPE = kv_shape("i8", 2, 64, 32, 100)


def check(new, parents, past=None, pages=None):
    past = [0] * len(new) if past is None else past
    need, at = [-(-(p + n) // 32) for p, n in zip(past, new)], 0
    pages = []
    for n in need:
        pages.append(list(range(at, at + n)))
        at += n
    kv_plan_check(SHAPE, 8, past, new, pages, parents=parents)


def refused(new, parents):
    with pytest.raises(BobcatError) as e:
        check(new, parents)
    assert e.value.status == STATUS["Argument"], str(e.value)


def test_trees_that_are_allowed():
    check([3], [[NO_PARENT, 0, 0]])
    check([3], [[NO_PARENT, NO_PARENT, 0]])
    check([0, 1, 4], [[], [NO_PARENT], [NO_PARENT, 0, 1, 1]])
    check([2, 3], [None, [NO_PARENT, 0, 0]])
    check([3000], [None])                                        # a chain of any length
    check([1024], [[NO_PARENT] * 1024])
    check([3, 2], iter([np.array([NO_PARENT, 0, 0], np.uint32), None]))


def test_trees_that_are_refused():
    refused([3], [[NO_PARENT, 0, 2]])                            # its own parent
    refused([3], [[1, NO_PARENT, 0]])                            # before its parent
    refused([3], [[NO_PARENT, 0, 0xFFFFFFFE]])
    refused([3], [[0, 0, 0]])
    refused([3], [[NO_PARENT, 0]])
    refused([3], [[NO_PARENT, 0, 0, 0]])
    refused([3, 2], [[NO_PARENT, 0, 0]])
    refused([1025], [[NO_PARENT] * 1025])
    refused([3000], [[NO_PARENT, *range(2998), 2997]])           # nearly a chain
    with pytest.raises(ValueError):
        check([2], [[NO_PARENT, -1]])


def test_null_arguments():
    one, some = (C.c_uint32 * 1)(1), (C.c_uint32 * 2)(0, 0)
    args = (C.byref(SHAPE), 8, 1, (C.c_uint32 * 1)(0), one, (C.c_uint32 * 1)(0), 1)
    assert lib().bch_kv_plan_check_trees(*args, None, 1) == STATUS["Argument"]
    assert lib().bch_kv_plan_check_trees(*args, some, 2) == STATUS["Argument"]
    assert lib().bch_kv_plan_check_trees(*args, (C.c_uint32 * 1)(NO_PARENT), 1) == STATUS["OK"]
    assert lib().bch_kv_plan_set_trees(None, *args[2:], some, 1) == STATUS["Argument"]
    assert lib().bch_rope_frequencies(None, None) == STATUS["Argument"]
    assert lib().bch_rope_frequencies(C.byref(rope_spec(4, 1e4)), None) == STATUS["Argument"]
    out = C.c_void_p(1)
    assert lib().bch_rope_new(None, C.byref(rope_spec(4, 1e4)), None, C.byref(out)) == STATUS["Argument"]
    assert out.value is None
    assert lib().bch_rope_new(None, C.byref(rope_spec(4, 1e4)), None, None) == STATUS["Argument"]
    lib().bch_rope_free(None)
    assert lib().bch_rope_paged(None, None, None, None, None) == STATUS["Argument"]
    from bobcat_amd._lib import View
    assert lib().bch_kv_keep(None, None, 0, 0, View(), 1, 0, View(), View()) == STATUS["Argument"]
    assert lib().bch_verify_drafts(None, None, 0, 0, 1, None, None) == STATUS["Argument"]


@pytest.mark.parametrize("change", [
    dict(n_rot=0), dict(n_rot=3), dict(n_rot=258), dict(theta=0.0), dict(theta=-1.0), dict(theta=math.inf), dict(theta=math.nan),
    dict(layout=2), dict(scaling=3), dict(scaling="linear", factor=0.0), dict(scaling="linear", factor=math.nan),
    dict(scaling="parts", factor=4.0), dict(scaling="parts", factor=4.0, n_original=100, slow=32.0, fast=32.0),
    dict(scaling="parts", factor=4.0, n_original=100, slow=math.nan), dict(magnitude=math.inf), dict(magnitude=math.nan)])
def test_specs_that_are_refused(change):
    args = dict(n_rot=64, theta=1e4) | change
    with pytest.raises(BobcatError) as e:
        rope_frequencies(rope_spec(args.pop("n_rot"), args.pop("theta"), **args))
    assert e.value.status == STATUS["Argument"]


def test_frequencies():
    j = np.arange(32)
    plain = 1e6 ** (-2 * j / 64)
    near = lambda a, b: np.testing.assert_allclose(a, b, rtol=1e-14)  # noqa: E731  (pow's rounding)
    near(rope_frequencies(rope_spec(64, 1e6)), plain)
    near(rope_frequencies(rope_spec(64, 1e6, factor=4.0)), plain)
    near(rope_frequencies(rope_spec(64, 1e6, scaling="linear", factor=4.0)), plain / 4)
    got = rope_frequencies(rope_spec(64, 1e6, scaling="parts", factor=4.0, n_original=8192, slow=1.0, fast=32.0))
    turns = 8192 * plain / (2 * np.pi)
    near(got[turns >= 32], plain[turns >= 32])
    near(got[turns <= 1], plain[turns <= 1] / 4)
    between = (turns > 1) & (turns < 32)
    assert between.any()
    w = (turns[between] - 1) / 31
    np.testing.assert_allclose(got[between], plain[between] * (w + (1 - w) / 4), rtol=1e-12)


def test_sizes_of_the_structs():
    from bobcat_amd._lib import Drafts, RopeRowsC, Verdict
    assert C.sizeof(RopeSpec) == 56 and C.sizeof(RopeRowsC) == 72 and C.sizeof(Drafts) == 88 and C.sizeof(Verdict) == 64
