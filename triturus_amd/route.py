"""route: the router of a mixture layer, on MI355X.

The max reductions' k-fold relative: each row of a T x E matrix of logits chooses its k largest ("experts"), and the
chosen pairs (row, choice) are ordered by expert, ready for the grouped products of ``gmm`` and ``mm_mx4``.  The
reference has no counterpart.

    r = route(logits, k)
    y = gmm(x[r.rows], w, r.sizes)                          # each expert's rows in one group
    out = (y[r.slots] * r.weights[..., None]).sum(1)        # back to rows, weighted

``normalize=True``: weights are the softmax of the chosen logits among themselves; ``False``: among all of the row.  Equal logits go
to the lowest index; a NaN comes first, and it or +inf makes the row's weights NaN, as in ``torch.softmax``.  A logit of -inf is
never chosen: its pair has expert -1, slot -1, weight 0 and no place in the order, so a row of -inf (padding) takes no expert's
time.  Places behind the last pair hold row 0, and ``gmm`` gives zeros there.
Everything stays on the device, in a fixed order: the same logits give the same result bit for bit.

Limits: k <= 16, E <= 1024.  ``weights`` takes part in autograd; under HIP graph capture logits that
require a gradient are refused, as by ``gmm``: capture ``route`` and ``route_grad`` instead.  ``route_grad`` itself takes no part
in autograd.  Forward-mode derivatives are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from triturus_amd import _lib
from triturus_amd.gmm import dual, refuse_capture, refuse_tangents

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_empty = torch.empty_strided


class Routes(NamedTuple):
    weights: torch.Tensor  # T x k, float32
    experts: torch.Tensor  # T x k, int32: the chosen experts, best first; -1: none
    rows: torch.Tensor     # T * k, int32: the row of each pair, ordered by expert and then by row; 0 behind the last pair
    slots: torch.Tensor    # T x k, int32: the place of each pair in that order; -1: none
    sizes: torch.Tensor    # E, int32: pairs of each expert


def _check(logits: torch.Tensor, k: int) -> int:
    assert len(logits.shape) == 2
    assert 1 <= k <= logits.shape[1]
    if logits.dtype not in _TYPES:
        raise NotImplementedError(f"route supports bf16/fp16/fp32, got {logits.dtype}")
    _lib.require_gpu(logits)
    return _lib.DTYPE_CODES[logits.dtype]


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x if (x.stride(1) == 1 or x.shape[1] == 1) and x.stride(0) >= 0 else x.contiguous()


def _route(logits: torch.Tensor, k: int, normalize: bool) -> Routes:
    code = _check(logits, k)
    T, E = logits.shape
    dev = logits.device
    # five allocations: views of one would share its version, and a change of one in place would spoil what autograd saved of another
    out = Routes(
        _empty((T, k), (k, 1), dtype=torch.float32, device=dev), _empty((T, k), (k, 1), dtype=torch.int32, device=dev),
        _empty((T * k,), (1,), dtype=torch.int32, device=dev), _empty((T, k), (k, 1), dtype=torch.int32, device=dev),
        _empty((E,), (1,), dtype=torch.int32, device=dev),
    )
    weights, experts, rows, slots, sizes = out
    if T == 0:
        sizes.zero_()
        return out
    logits = _rows(logits)
    lib = _lib.load()
    nbytes = lib.trt_route_workspace_bytes(T, E)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.on_device(dev):
        status = lib.trt_route(
            logits.data_ptr(), weights.data_ptr(), experts.data_ptr(), rows.data_ptr(), slots.data_ptr(), sizes.data_ptr(), T, E, k, logits.stride(0), code, int(bool(normalize)),
            ws.data_ptr() if nbytes else None, nbytes, _lib.raw_stream(dev),
        )
    if status:
        _lib.check(status, "trt_route")
    return out


def _grad(g: torch.Tensor, logits: torch.Tensor, weights: torch.Tensor, experts: torch.Tensor, normalize: bool) -> torch.Tensor:
    T, E = logits.shape
    d = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    if T == 0:
        return d
    logits, g, weights, experts = _rows(logits), g.contiguous(), weights.contiguous(), experts.contiguous()
    with _lib.on_device(d.device):
        status = _lib.load().trt_route_grad(
            g.data_ptr(), logits.data_ptr(), weights.data_ptr(), experts.data_ptr(), d.data_ptr(), T, E, g.shape[1],
            logits.stride(0), _lib.DTYPE_CODES[logits.dtype], int(bool(normalize)), _lib.raw_stream(d.device),
        )
    if status:
        _lib.check(status, "trt_route_grad")
    return d


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, normalize):
        out = _route(logits, k, normalize)
        ctx.save_for_backward(logits, out.weights, out.experts)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        refuse_capture("route")
        if dual._current_level >= 0:
            refuse_tangents("route's backward pass", g)
        return _grad(g, *ctx.saved_tensors, ctx.normalize), None, None


def route(logits: torch.Tensor, k: int, *, normalize: bool = True) -> Routes:
    """The k largest logits of every row, their weights, and the pairs ordered by expert."""
    if dual._current_level >= 0:
        refuse_tangents("route", logits)
    if logits.requires_grad and torch.is_grad_enabled():
        _check(logits, k)
        refuse_capture("route")
        return Routes(*_Route.apply(logits, k, normalize))
    return _route(logits, k, normalize)


def route_grad(g: torch.Tensor, logits: torch.Tensor, routes: Routes, *, normalize: bool = True) -> torch.Tensor:
    """Gradient of sum(g * routes.weights) with respect to the logits, in their type; ``normalize`` and ``routes`` as of ``route``
    (an expert stands at most once in a row)."""
    if dual._current_level >= 0:
        refuse_tangents("route_grad", g, logits, routes.weights)
    _check(logits, routes.weights.shape[1])
    shape = (logits.shape[0], routes.weights.shape[1])
    assert g.shape == routes.weights.shape == routes.experts.shape == shape
    assert g.dtype == routes.weights.dtype == torch.float32 and routes.experts.dtype == torch.int32
    assert g.device == logits.device == routes.weights.device == routes.experts.device
    with torch.no_grad():
        return _grad(g, logits, routes.weights, routes.experts, normalize)
