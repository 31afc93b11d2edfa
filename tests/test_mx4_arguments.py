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


def test_rows_of_values_may_be_long_and_far_apart():
    """The 8 MiB between rows are for codes: rows of values are quantised first, or read with 64-bit offsets."""
    far = 1 << 23
    assert call(sa=(far, 2)) == -4
    # a workspace is asked for and not given: past the range check, and nothing enqueued
    assert call(sa=(far, 0), a_type=_lib.TRT_BF16) == -3
    assert call(sa=(1 << 40, 0), a_type=_lib.TRT_F32, K=far + 96, sb=(0, far // 2 + 64, 0, 1 << 18)) == -3
    assert call(sa=(1 << 25, 0), a_type=_lib.TRT_F32, K=(1 << 24) + 1, sb=(0, far - 1, 0, 1 << 19)) == -4  # codes of a row beyond 8 MiB


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4])
def test_long_rows_of_values(dev, tile):
    """Contractions past 2^23 values against the same product in parts, whose codes are the same blocks."""
    from triturus_amd.mx4 import MX4, mm_mx4, mx4_quantize

    T, N, K = 3, 5, (1 << 23) + 96
    a, w = torch.randn(T, K, device=dev).bfloat16(), mx4_quantize(torch.randn(N, K, device=dev))
    c = mm_mx4(a, w, dtype=torch.float32, _tile=tile)
    want, size = torch.zeros(T, N, dtype=torch.float64, device=dev), torch.zeros(T, N, dtype=torch.float64, device=dev)
    from triturus_amd.mx4 import mx4_dequantize

    q = mx4_quantize(a)
    for k in range(0, K, 1 << 20):
        part = [mx4_dequantize(MX4(x.codes[:, k // 2:(k + (1 << 20)) // 2].contiguous(), x.scales[:, k // 32:(k + (1 << 20)) // 32].contiguous(),
                                   min(1 << 20, K - k))).double() for x in (q, w)]
        want += part[0] @ part[1].T
        size += part[0].abs() @ part[1].abs().T
    assert torch.equal(mm_mx4(q, w, dtype=torch.float32, _tile=tile), c)
    # an fp32 sum of n terms taken one after the other is off by at most n 2^-23 of the sum of magnitudes; wavefronts and blocks only shorten it
    assert ((c.double() - want).abs() <= (K + 1) * 2.0 ** -23 * size).all()
    far = torch.empty(T, K + 32, dtype=a.dtype, device=dev)[:, :K].copy_(a)
    assert torch.equal(mm_mx4(far, w, dtype=torch.float32, _tile=tile), c)
