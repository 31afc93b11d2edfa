"""gmm: matrix products grouped by expert, with ragged sizes, on MI355X.

``mm`` (triturus/mm.py:181-214) has one matrix for all rows; here T rows lie in E consecutive groups of
``sizes[e]`` rows and every group has its own matrix: the products of a mixture layer.  The reference has no
counterpart.  ``sizes`` stays on the device (nothing here waits for it), so a router's output can be passed on.

    c = gmm(a, b, sizes)                  # a: T x K, b: E x K x N, sizes: E  ->  c: T x N
    da, db = gmm_grad(g, a, b, sizes)     # of sum(g * c)

Types: bfloat16, float16 and float32, one for all operands.  Sums are fp32; a result is rounded once to the
operands' type.  fp32 contracts in IEEE fp32 on the fp32 matrix pipe whatever ``set_tf32_enabled`` says.
Rows behind the last group (a padded batch) give zeros, take no gradient and are never read as terms of a sum.
Groups may be empty.  Sizes that are negative or reach past T in sum are clamped: nothing outside the tensors is touched.

``gmm`` takes part in autograd.  Under HIP graph capture it refuses operands that require a gradient: capture
``gmm`` on detached operands and ``gmm_grad`` instead (a backward pass of autograd captured while another graph
of the same leaves is alive ends the process inside torch).  ``gmm_grad`` itself takes no part in autograd.  Forward-mode
derivatives are refused.
"""

from __future__ import annotations

from types import SimpleNamespace

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from triturus_amd import _lib

_TYPES = (torch.bfloat16, torch.float16, torch.float32)

try:
    _is_capturing = torch._C._cuda_isCurrentStreamCapturing
except AttributeError:  # pragma: no cover
    _is_capturing = torch.cuda.is_current_stream_capturing


def refuse_capture(op: str) -> None:
    if _is_capturing():
        raise RuntimeError(
            f"{op}: operands that require a gradient are refused under graph capture; "
            f"capture {op} on detached operands and {op}_grad"
        )


# Outside of dual levels (-1) no tensor has a tangent: callers look there first, which costs less than a call.
dual = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)


def refuse_tangents(op: str, *tensors: torch.Tensor) -> None:
    """Operands with a forward-mode tangent: they do not require a gradient, and the result would lose it without a word."""
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{op} has no forward-mode derivative: pass the primal of its operands")


# The kernels address 256 rows of a tile with 31-bit byte offsets: rows further apart than this many bytes are copied
# (the last token of long sequences, ``h[:, -1]``).
ROW_STRIDE_LIMIT = 1 << 23


def dense(t: torch.Tensor) -> torch.Tensor:
    """A copy whose strides are those of its shape (``contiguous()`` keeps any stride of an axis of length one)."""
    return t.clone(memory_format=torch.contiguous_format)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows with a unit trailing stride, in place where the tensor has them."""
    st = t.stride()
    return t if (st[1] == 1 or t.shape[1] == 1) and 0 <= st[0] * t.itemsize < ROW_STRIDE_LIMIT else dense(t)


def _matrices(b: torch.Tensor) -> torch.Tensor:
    """Matrices with a unit stride along one of their axes, in place where the tensor has them."""
    st, most = b.stride(), ROW_STRIDE_LIMIT // b.itemsize
    if min(st) >= 0:
        if (st[1] == 1 and st[2] < most) or (st[2] == 1 and st[1] < most):
            return b
        if b.shape[2] == 1 and st[1] < most:
            return b.as_strided(b.shape, (st[0], st[1], 1), b.storage_offset())
        if b.shape[1] == 1 and st[2] < most:
            return b.as_strided(b.shape, (st[0], 1, st[2]), b.storage_offset())
    return dense(b)


def _few_rows(T: int, E: int) -> bool:
    """Whether the library cuts no group into pieces, whatever the matrices: a piece has at least 256 bytes of a column (64 rows of
    fp32, 128 of 16-bit types) and is a multiple of 32 rows, and groups of at most 32 rows on average leave pieces of 32."""
    return T <= 32 * E


_pieces: dict = {}  # (T, E, K, N, type, tile) -> bytes of the pieces' sums of operands on the boundaries, as reported by the library


def _piece_bytes(lib, pa: int, pg: int, T: int, E: int, K: int, N: int, lda: int, ldg: int, code: int, tile: int = 0) -> int:
    key = (T, E, K, N, code, tile)
    n = _pieces.get(key)
    if n is None:
        if len(_pieces) > 4096:
            _pieces.clear()
        n = _pieces[key] = lib.trt_gmm_weights_workspace_bytes(pa, pg, T, E, K, N, lda, ldg, code, tile)
    return n


def _check(a: torch.Tensor, b: torch.Tensor, sizes: torch.Tensor) -> None:
    sa, sb, ss = a.shape, b.shape, sizes.shape
    assert len(sa) == 2 and len(sb) == 3 and len(ss) == 1
    assert sa[1] == sb[1]
    assert sb[0] == ss[0] >= 1
    dtype = a.dtype
    assert dtype is b.dtype
    assert sizes.dtype in (torch.int32, torch.int64)
    dev = a.device
    assert dev == b.device and dev == sizes.device
    if dtype not in _TYPES:
        raise NotImplementedError(f"gmm supports bf16/fp16/fp32, got {dtype}")
    _lib.require_gpu(a)


def _forward(a: torch.Tensor, b: torch.Tensor, sizes: torch.Tensor, tile: int = 0) -> torch.Tensor:
    T, K = a.shape
    E, _, N = b.shape
    dtype, dev = a.dtype, a.device
    c = a.new_empty((T, N))
    if T == 0 or N == 0:
        return c
    if K == 0:
        return c.zero_()
    a, b, sizes = _rows(a), _matrices(b), sizes.contiguous()
    lib, code = _lib.load(), _lib.DTYPE_CODES[dtype]
    pa, pb, lda, sb = a.data_ptr(), b.data_ptr(), a.stride(0), _lib.strides3(b)
    ws_ptr, nbytes, ws = None, 0, None
    if (pa | pb) & 15 or (K | N | lda | sb[0] | (sb[2] if sb[1] == 1 else sb[1])) & 7:  # then a copy may pay
        nbytes = lib.trt_gmm_workspace_bytes(pa, pb, T, E, K, N, lda, sb, code, tile)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ws_ptr = ws.data_ptr()
    with _lib.on_device(dev):
        status = lib.trt_gmm(pa, pb, sizes.data_ptr(), c.data_ptr(), T, E, K, N, lda, sb, code, sizes.dtype is torch.int64, tile,
                             ws_ptr, nbytes, _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_gmm")
    return c


def _weights(a: torch.Tensor, g: torch.Tensor, sizes: torch.Tensor, tile: int = 0) -> torch.Tensor:
    T, K = a.shape
    E, N = sizes.shape[0], g.shape[1]
    dtype, dev = a.dtype, a.device
    d = a.new_empty((E, K, N))
    if d.numel() == 0:
        return d
    if T == 0:
        return d.zero_()
    a, g, sizes = _rows(a), _rows(g), sizes.contiguous()
    lib, code = _lib.load(), _lib.DTYPE_CODES[dtype]
    pa, pg, lda, ldg = a.data_ptr(), g.data_ptr(), a.stride(0), g.stride(0)
    ws_ptr, nbytes, ws = None, 0, None
    if (pa | pg) & 15 or (K | N | lda | ldg) & 7:  # a copy may pay
        nbytes = lib.trt_gmm_weights_workspace_bytes(pa, pg, T, E, K, N, lda, ldg, code, tile)
    elif not _few_rows(T, E):
        nbytes = _piece_bytes(lib, pa, pg, T, E, K, N, lda, ldg, code, tile)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ws_ptr = ws.data_ptr()
    with _lib.on_device(dev):
        status = lib.trt_gmm_weights(pa, pg, sizes.data_ptr(), d.data_ptr(), T, E, K, N, lda, ldg, code, sizes.dtype is torch.int64, tile,
                                     ws_ptr, nbytes, _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_gmm_weights")
    return d


class _Gmm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, sizes):
        need = ctx.needs_input_grad  # a gradient takes the other operand's values alone
        ctx.save_for_backward(a if need[1] else None, b if need[0] else None, sizes)
        return _forward(a, b, sizes)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        refuse_capture("gmm")
        if dual._current_level >= 0:
            refuse_tangents("gmm's backward pass", g)
        a, b, sizes = ctx.saved_tensors
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[1]:
            return *gmm_grad(g, a, b, sizes), None
        da = _forward(g, b.transpose(1, 2), sizes) if ctx.needs_input_grad[0] else None
        db = _weights(a, g, sizes) if ctx.needs_input_grad[1] else None
        return da, db, None


def gmm(a: torch.Tensor, b: torch.Tensor, sizes: torch.Tensor) -> torch.Tensor:
    """c[r] = a[r] @ b[e(r)], e(r) the group that row r lies in; zeros behind the last group."""
    if dual._current_level >= 0:
        refuse_tangents("gmm", a, b)
    _check(a, b, sizes)
    if (a.requires_grad or b.requires_grad) and torch.is_grad_enabled():
        refuse_capture("gmm")
        return _Gmm.apply(a, b, sizes)
    return _forward(a, b, sizes)


def gmm_grad(g: torch.Tensor, a: torch.Tensor, b: torch.Tensor, sizes: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients (of a, of b) of sum(g * gmm(a, b, sizes)), in the operands' type; zero for rows behind the last group
    and for matrices of empty groups."""
    if dual._current_level >= 0:
        refuse_tangents("gmm_grad", g, a, b)
    _check(a, b, sizes)
    assert g.shape == (a.shape[0], b.shape[2])
    assert g.dtype == a.dtype and g.device == a.device
    T, K = a.shape
    E, _, N = b.shape
    if not (T and K and N):
        with torch.no_grad():
            return _forward(g, b.transpose(1, 2), sizes), _weights(a, g, sizes)
    dev = a.device
    da, db = a.new_empty((T, K)), a.new_empty((E, K, N))
    g, a, b, sizes = _rows(g), _rows(a), _matrices(b), sizes.contiguous()
    lib, code = _lib.load(), _lib.DTYPE_CODES[a.dtype]
    pg, pa, pb, ldg, lda, sb = g.data_ptr(), a.data_ptr(), b.data_ptr(), g.stride(0), a.stride(0), _lib.strides3(b)
    ws_ptr, nbytes, ws = None, 0, None
    if (pg | pa | pb) & 15 or (K | N | ldg | lda | sb[0] | (sb[2] if sb[1] == 1 else sb[1])) & 7:  # a copy may pay
        nbytes = lib.trt_gmm_grad_workspace_bytes(pg, pa, pb, T, E, K, N, ldg, lda, sb, code)
    elif not _few_rows(T, E):
        nbytes = _piece_bytes(lib, pa, pg, T, E, K, N, lda, ldg, code)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        ws_ptr = ws.data_ptr()
    with _lib.on_device(dev):
        status = lib.trt_gmm_grad(pg, pa, pb, sizes.data_ptr(), da.data_ptr(), db.data_ptr(), T, E, K, N, ldg, lda, sb, code,
                                  sizes.dtype is torch.int64, ws_ptr, nbytes, _lib.raw_stream(dev))
    if status:
        _lib.check(status, "trt_gmm_grad")
    return da, db
