"""mx4: the microscaled 4-bit format (MXFP4) and its matrix products, on MI355X.

The step below ``set_matrix_precision("bf16x3")`` for weights that may be coarse: 32 neighbours along a row share a
power of two, and each is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign -- 17 bytes for 32 values.  The reference has no
counterpart.

    w = mx4_quantize(weights)              # N x K (or E x N x K), blocks along the contracted axis K
    c = mm_mx4(a, w)                       # a: T x K  ->  T x N, a @ w.T over the 4-bit values of BOTH operands
    c = mm_mx4(a, w, sizes)                # w: E x N x K, rows of a in groups as for ``gmm``
    y = mx4_dequantize(w)                  # the values that codes and scales stand for

Quantisation follows the OCP Microscaling Formats specification v1.0: the block's exponent is floor(log2 max |x|) - 2,
values round to nearest with ties to the even code and stop at 6; a block with a NaN or an infinity stands for NaN.  A
row whose length is not a multiple of 32 has a last block filled up with zeros.
Products are exact, their sums fp32, and a result is rounded once.
``a`` may be quantised already, or a tensor of values, which is quantised within the call.
"""

from __future__ import annotations

from typing import NamedTuple

import ctypes

import torch

from triturus_amd import _lib

BLOCK = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_I64x2, _I64x4 = ctypes.c_int64 * 2, ctypes.c_int64 * 4


class MX4(NamedTuple):
    """Rows of 4-bit values: codes (..., 16 ceil(K / 32)) and scales (..., ceil(K / 32)), both uint8, and the rows' length K."""

    codes: torch.Tensor
    scales: torch.Tensor
    length: int


def _type_code(dtype: torch.dtype, op: str) -> int:
    if dtype not in _TYPES:
        raise NotImplementedError(f"{op} supports bf16/fp16/fp32, got {dtype}")
    return _lib.DTYPE_CODES[dtype]


def _check(q: MX4) -> None:
    blocks = -(-q.length // BLOCK)
    assert q.length >= 0
    assert q.codes.dtype == q.scales.dtype == torch.uint8
    assert len(q.codes.shape) >= 1 and q.codes.shape[:-1] == q.scales.shape[:-1]
    assert q.codes.shape[-1] == 16 * blocks and q.scales.shape[-1] == blocks
    assert q.codes.device == q.scales.device
    _lib.require_gpu(q.codes, q.scales)


def _unit(t: torch.Tensor) -> torch.Tensor:
    """Bytes of a row next to each other, in place where they are."""
    st = t.stride()
    if min(st) >= 0 and (st[-1] == 1 or t.shape[-1] == 1):
        return t
    return t.contiguous()


def mx4_quantize(x: torch.Tensor) -> MX4:
    """The 4-bit form of x along its last axis."""
    assert len(x.shape) >= 1
    code = _type_code(x.dtype, "mx4_quantize")
    _lib.require_gpu(x)
    K = x.shape[-1]
    blocks = -(-K // BLOCK)
    codes = torch.empty((*x.shape[:-1], 16 * blocks), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], blocks), dtype=torch.uint8, device=x.device)
    if codes.numel() == 0:
        return MX4(codes, scales, K)
    flat = x.detach().reshape(-1, K)
    if K > 1 and flat.stride(1) != 1 or flat.stride(0) < 0:
        flat = flat.contiguous()
    with _lib.on_device(x.device):
        status = _lib.load().trt_mx4_quantize(flat.data_ptr(), codes.data_ptr(), scales.data_ptr(), flat.shape[0], K,
                                              flat.stride(0), code, _lib.raw_stream(x.device))
    if status:
        _lib.check(status, "trt_mx4_quantize")
    return MX4(codes, scales, K)


def mx4_dequantize(q: MX4, *, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that q stands for (exact in fp32, and in bf16 unless its exponent range ends)."""
    _check(q)
    code = _type_code(dtype, "mx4_dequantize")
    y = torch.empty((*q.codes.shape[:-1], q.length), dtype=dtype, device=q.codes.device)
    if y.numel() == 0:
        return y
    codes, scales = _unit(q.codes.reshape(-1, q.codes.shape[-1])), _unit(q.scales.reshape(-1, q.scales.shape[-1]))
    with _lib.on_device(y.device):
        status = _lib.load().trt_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), codes.shape[0], q.length,
                                                codes.stride(0), scales.stride(0), code, _lib.raw_stream(y.device))
    if status:
        _lib.check(status, "trt_mx4_dequantize")
    return y


def mm_mx4(a: torch.Tensor | MX4, b: MX4, sizes: torch.Tensor | None = None, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """c[r, n] = sum_k a[r, k] b[n, k], or with ``sizes`` b[e(r), n, k]; ``dtype``: of c, by default a's (bf16 for an MX4)."""
    if not isinstance(a, MX4):
        assert len(a.shape) == 2
        dtype = dtype or a.dtype
        _type_code(a.dtype, "mm_mx4")
        if a.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("mm_mx4 has no gradient: detach its operand")
        a = mx4_quantize(a)
    dtype = dtype or torch.bfloat16
    code = _type_code(dtype, "mm_mx4")
    _check(a)
    _check(b)
    assert len(a.codes.shape) == 2 and len(b.codes.shape) == (2 if sizes is None else 3)
    assert a.length == b.length
    assert a.codes.device == b.codes.device
    T, N, K = a.codes.shape[0], b.codes.shape[-2], a.length
    E = 1 if sizes is None else b.codes.shape[0]
    if sizes is not None:
        assert len(sizes.shape) == 1 and sizes.shape[0] == E >= 1
        assert sizes.dtype in (torch.int32, torch.int64)
        assert sizes.device == a.codes.device
        sizes = sizes.contiguous()
    c = torch.empty((T, N), dtype=dtype, device=a.codes.device)
    if c.numel() == 0:
        return c
    if K == 0:
        return c.zero_()
    ac, as_, bc, bs = _unit(a.codes), _unit(a.scales), _unit(b.codes), _unit(b.scales)
    with _lib.on_device(c.device):
        status = _lib.load().trt_mx4_mm(
            ac.data_ptr(), as_.data_ptr(), bc.data_ptr(), bs.data_ptr(), None if sizes is None else sizes.data_ptr(), c.data_ptr(),
            T, E, K, N, _I64x2(ac.stride(0), as_.stride(0)),
            _I64x4(0 if sizes is None else bc.stride(0), bc.stride(-2), 0 if sizes is None else bs.stride(0), bs.stride(-2)),
            code, sizes is not None and sizes.dtype == torch.int64, _lib.raw_stream(c.device),
        )
    if status:
        _lib.check(status, "trt_mx4_mm")
    return c
