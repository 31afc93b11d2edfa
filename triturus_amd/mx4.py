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
from triturus_amd.gmm import ROW_STRIDE_LIMIT, dense, dual, refuse_tangents

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
    codes, scales, length = q
    shape, blocks = codes.shape, -(-length // BLOCK)
    assert length >= 0
    assert codes.dtype is torch.uint8 and scales.dtype is torch.uint8
    assert len(shape) >= 1 and shape[-1] == 16 * blocks
    assert scales.shape == (*shape[:-1], blocks)
    assert codes.device == scales.device
    _lib.require_gpu(codes)


def _unit(t: torch.Tensor) -> torch.Tensor:
    """Bytes of a row next to each other, in place where they are."""
    st = t.stride()
    if (st[-1] == 1 or t.shape[-1] == 1) and min(st) >= 0 and st[-2] < ROW_STRIDE_LIMIT:
        return t
    return dense(t)


def _values(x: torch.Tensor) -> torch.Tensor:
    """Rows of values with a unit trailing stride, in place where the tensor has them."""
    st = x.stride()
    return x if (st[1] == 1 or x.shape[1] == 1) and st[0] >= 0 else x.contiguous()


def mx4_quantize(x: torch.Tensor) -> MX4:
    """The 4-bit form of x along its last axis.  Codes and scales are whole numbers and carry no gradient, as ``torch.argmax``'s."""
    shape = x.shape
    assert len(shape) >= 1
    code = _type_code(x.dtype, "mx4_quantize")
    _lib.require_gpu(x)
    K, dev = shape[-1], x.device
    blocks = -(-K // BLOCK)
    codes = torch.empty((*shape[:-1], 16 * blocks), dtype=torch.uint8, device=dev)
    scales = torch.empty((*shape[:-1], blocks), dtype=torch.uint8, device=dev)
    if codes.numel() == 0:
        return MX4(codes, scales, K)
    x = x.detach() if x.requires_grad else x
    x = _values(x if len(shape) == 2 else x.reshape(-1, K))
    with _lib.on_device(dev):
        status = _lib.load().trt_mx4_quantize(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.shape[0], K, x.stride(0), code,
                                              _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_mx4_quantize")
    return MX4(codes, scales, K)


def mx4_dequantize(q: MX4, *, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that q stands for (exact in fp32, and in bf16 unless its exponent range ends)."""
    _check(q)
    code = _type_code(dtype, "mx4_dequantize")
    codes, scales, K = q
    shape, dev = codes.shape, codes.device
    y = torch.empty((*shape[:-1], K), dtype=dtype, device=dev)
    if y.numel() == 0:
        return y
    if len(shape) != 2:
        codes, scales = codes.reshape(-1, shape[-1]), scales.reshape(-1, scales.shape[-1])
    codes, scales = _unit(codes), _unit(scales)
    with _lib.on_device(dev):
        status = _lib.load().trt_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), codes.shape[0], K,
                                                codes.stride(0), scales.stride(0), code, _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_mx4_dequantize")
    return y


_ws_bytes: dict = {}  # (T, E, K, N, types, tile) -> workspace bytes, as reported by the library


def mm_mx4(a: torch.Tensor | MX4, b: MX4, sizes: torch.Tensor | None = None, *, dtype: torch.dtype | None = None,
           _tile: int = 0) -> torch.Tensor:
    """c[r, n] = sum_k a[r, k] b[n, k], or with ``sizes`` b[e(r), n, k]; ``dtype``: of c, by default a's (bf16 for an MX4).

    ``_tile`` forces a kernel (tests, timing)."""
    if dual._current_level >= 0 and not isinstance(a, MX4):
        refuse_tangents("mm_mx4", a)
    _check(b)
    bc, bs, K = b
    shape = bc.shape
    if isinstance(a, MX4):
        _check(a)
        assert len(a.codes.shape) == 2 and a.length == K
        ac, as_, a_type = _unit(a.codes), _unit(a.scales), -1
        dtype = dtype or torch.bfloat16
        sa = _I64x2(ac.stride(0), as_.stride(0))
    else:
        assert len(a.shape) == 2 and a.shape[1] == K
        a_type = _type_code(a.dtype, "mm_mx4")
        if a.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("mm_mx4 has no gradient: detach its operand")
        ac = as_ = _values(a)
        dtype = dtype or a.dtype
        sa = _I64x2(ac.stride(0), 0)
    code = _type_code(dtype, "mm_mx4")
    dev = ac.device
    assert dev == bc.device
    T, N = ac.shape[0], shape[-2] if len(shape) > 1 else 0
    if sizes is None:
        assert len(shape) == 2
        E, wide, sizes_ptr = 1, False, None
    else:
        assert len(shape) == 3 and len(sizes.shape) == 1
        E, wide = shape[0], sizes.dtype is torch.int64
        assert sizes.shape[0] == E >= 1
        assert wide or sizes.dtype is torch.int32
        assert sizes.device == dev
        sizes = sizes.contiguous()
        sizes_ptr = sizes.data_ptr()
    c = torch.empty((T, N), dtype=dtype, device=dev)
    if T == 0 or N == 0:
        return c
    if K == 0:
        return c.zero_()
    bc, bs = _unit(bc), _unit(bs)
    lib = _lib.load()
    nbytes = 0
    if a_type >= 0:
        key = (T, E, K, N, a_type, code, _tile)
        nbytes = _ws_bytes.get(key)
        if nbytes is None:
            if len(_ws_bytes) > 4096:
                _ws_bytes.clear()
            nbytes = _ws_bytes[key] = lib.trt_mx4_mm_workspace_bytes(*key)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    cst, sst = bc.stride(), bs.stride()
    sb = _I64x4(0, cst[0], 0, sst[0]) if sizes is None else _I64x4(cst[0], cst[1], sst[0], sst[1])
    with _lib.on_device(dev):
        status = lib.trt_mx4_mm(ac.data_ptr(), as_.data_ptr(), bc.data_ptr(), bs.data_ptr(), sizes_ptr, c.data_ptr(), T, E, K, N, sa, sb,
                                a_type, code, wide, _tile, ws.data_ptr() if nbytes else None, nbytes, _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_mx4_mm")
    return c
