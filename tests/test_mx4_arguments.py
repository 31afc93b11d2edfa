"""Arguments of the 4-bit product at their limits: what the header allows is taken, the rest is a status before anything is enqueued."""

import ctypes
from ctypes import c_void_p

import pytest
import torch

from triturus_amd import _lib

one, null = c_void_p(16), c_void_p(None)  # never dereferenced: every host-only call below is rejected first


def call(a=one, a_scales=one, T=4, E=1, K=64, N=8, sa=(32, 2), sb=(0, 32, 0, 2), a_type=-1, dtype=_lib.TRT_BF16, tile=1):
    i64 = lambda v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731
    return _lib.load().trt_mx4_mm(a, a_scales, one, one, null, one, T, E, K, N, i64(sa), i64(sb), a_type, dtype, 0, tile, null, 0, null)


@pytest.mark.parametrize("a_type", [-2, -7, -(1 << 31)])
def test_types_of_a_other_than_the_documented_ones(a_type):
    assert call(a_type=a_type, a_scales=null) == -1
    assert call(a_type=a_type, T=1 << 31) == -1  # were it taken for codes: a status that enqueues nothing either
