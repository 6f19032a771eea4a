"""Softmax cross entropy of embeddings against a large table of vectors.

``linear_cross_entropy`` is the classification loss beside the kernel losses
of this package: every row of ``x`` (node embeddings, hidden states) is
scored against all rows of ``weight`` (class vectors, a vocabulary), and the
loss is the negative log-probability of its target.  The logits are never
held: the forward joins per-tile maxima and sums as a tensor-core product
makes them, the backward makes them again a piece of the vocabulary at a time
(``csrc/ra_ce.cuh``).  Inputs must be CUDA tensors: there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
from typing import Tuple

import torch

from . import _lib

Tensor = torch.Tensor

__all__ = ["linear_cross_entropy"]

_REDUCTIONS = {"none": _lib.RA_REDUCE_NONE, "sum": _lib.RA_REDUCE_SUM,
               "mean": _lib.RA_REDUCE_MEAN}

_SMALL = 1 << 20  # bytes of a workspace that may live as long as its call's state


def _rows16(t: Tensor) -> Tensor:
    """`t` (a matrix) as the kernels read it: unit stride along its rows and,
    for the 16-bit types, 16-byte aligned rows (copied where it is not)."""
    if t.dtype == torch.float32:
        return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and \
            t.data_ptr() % 16 == 0:
        return t
    n, d = t.shape
    padded = torch.empty((n, (d + 7) // 8 * 8), dtype=t.dtype, device=t.device)[:, :d]
    padded.copy_(t)
    return padded


def _operands(d, x: Tensor, weight: Tensor) -> Tuple[Tensor, Tensor]:
    """Both matrices as one pass of the kernels reads them, their strides into `d`."""
    xk, wk = _rows16(x), _rows16(weight)
    # of a single row PyTorch keeps any stride, and calls it contiguous
    d.ld_x = max(xk.stride(0), d.dim) if d.rows else (d.dim + 7) // 8 * 8
    d.ld_w = max(wk.stride(0), d.dim)
    return xk, wk


class _LinearCrossEntropy(torch.autograd.Function):
    """(x, weight) -> (loss, lse), both float32."""

    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, target: Tensor, scale: float, softcap: float,
                ignore_index: int, reduction: int):
        lib = _lib.load()
        dev = x.device
        d = _lib.RaCeDesc()
        d.rows, d.dim = x.shape
        d.vocab = weight.shape[0]
        xk, wk = _operands(d, x, weight)
        d.ignore_index, d.dtype, d.reduction = ignore_index, _lib.DTYPES[x.dtype], reduction
        d.scale, d.softcap, d.status = scale, softcap, _lib.status_word()
        if ctx is None and (x.dtype != torch.float32
                            or wk.data_ptr() % 16 == 0 and d.ld_w % 4 == 0):
            d.forward_only = 1
        with _lib.on_device(dev):
            n_state = lib.ra_ce_state_bytes(ctypes.byref(d))
            n_ws = lib.ra_ce_workspace_bytes(ctypes.byref(d), 0)
            # a small workspace lies behind the state
            held = (n_state + 255) // 256 * 256
            ws = _lib.scratch(n_ws, dev) if n_ws > _SMALL else None
            state = _lib.scratch(held if ws is not None else held + n_ws, dev)
            shape = (d.rows,) if reduction == _lib.RA_REDUCE_NONE else ()
            loss = torch.empty(shape, dtype=torch.float32, device=dev)
            lse = torch.empty(d.rows, dtype=torch.float32, device=dev)
            rc = lib.ra_ce_forward(ctypes.byref(d), xk.data_ptr(), wk.data_ptr(),
                                   target.data_ptr(), loss.data_ptr(), lse.data_ptr(),
                                   state.data_ptr(), n_state,
                                   state.data_ptr() + held if ws is None else ws.data_ptr(), n_ws,
                                   _lib.stream_handle(dev))
        _lib.check(rc, "linear cross entropy")
        if ctx is None:  # no gradient wanted: without autograd's share of a small call
            return loss, lse
        ctx.desc = d
        ctx.save_for_backward(x, weight, target, state)  # freed with the graph
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, g_lse):
        lib = _lib.load()
        # not always the forward's tensors: a checkpoint makes them again, hooks
        # on saved tensors may bring them back elsewhere and with other strides
        x, weight, target, state = ctx.saved_tensors
        d, dev = ctx.desc, x.device
        xk, wk = _operands(d, x, weight)
        target = target.contiguous()
        need_x, need_w = ctx.needs_input_grad[:2]
        gl = None if g_loss is None else g_loss.to(torch.float32).contiguous()
        ge = None if g_lse is None else g_lse.to(torch.float32).contiguous()
        with _lib.on_device(dev):
            state = _lib.aligned(state)
            dx = _lib.empty_as(x) if need_x else None
            dw = _lib.empty_as(weight) if need_w else None
            ws = _lib.scratch(lib.ra_ce_workspace_bytes(ctypes.byref(d), 1), dev)
            rc = lib.ra_ce_backward(ctypes.byref(d), xk.data_ptr(), wk.data_ptr(),
                                    target.data_ptr(), _lib.ptr(gl), _lib.ptr(ge), _lib.ptr(dx),
                                    _lib.ptr(dw), state.data_ptr(), state.numel(),
                                    ws.data_ptr(), ws.numel(), _lib.stream_handle(dev))
        _lib.check(rc, "linear cross entropy backward")
        return dx, dw, None, None, None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, target: Tensor, *, scale: float = 1.0,
                         softcap: float = 0.0, ignore_index: int = -100,
                         reduction: str = "mean") -> Tuple[Tensor, Tensor]:
    """Softmax cross entropy of ``x @ weight.T`` without the logits in memory.

    Args:
        x: (N, D) rows, float32, bfloat16 or float16.
        weight: (V, D) table of the same dtype.
        target: (N,) integer rows of the table; rows with ``ignore_index``
            have loss 0 and no part in the mean.  A target outside the table
            is not read: its loss (and with it the mean or sum, and the
            gradients) is NaN.
        scale: factor of the logits (an inverse temperature).
        softcap: where positive, the logits are ``softcap * tanh(z / softcap)``.
        reduction: "mean" over the rows with a target, "sum" or "none".

    Returns:
        ``(loss, lse)`` in float32: the loss () or (N,), and the logarithm of
        every row's sum of exponentials (N,).  Both are differentiable in
        ``x`` and ``weight`` (``lse`` gives a z-loss: ``(lse ** 2).mean()``).

    float32 inputs are multiplied as pairs of float16 halves (22 bits), 16-bit
    inputs as they are, always with float32 sums; the logits' gradients are
    rounded to the inputs' type before the two gradient products.  Gradients
    are bitwise repeatable.  The call never waits for the device and can be
    captured into a graph.
    """
    if x.ndim != 2 or weight.ndim != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError("x and weight must be (N,d) and (V,d) with same d")
    if target.ndim != 1 or target.shape[0] != x.shape[0]:
        raise ValueError("target length must equal number of rows")
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
        raise ValueError("target must hold integers")
    if x.dtype != weight.dtype or x.dtype not in _lib.DTYPES:
        raise ValueError("x and weight must share dtype float32, bfloat16 or float16")
    if weight.shape[0] == 0 or x.shape[1] == 0:
        raise ValueError("weight must have at least one row and one column")
    if x.shape[1] > 65536 or x.shape[0] > 2 ** 31 - 256 or weight.shape[0] > 2 ** 31 - 512:
        raise ValueError("linear_cross_entropy: at most 65536 columns and 2^31 - 512 rows")
    scale, softcap = float(scale), float(softcap)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not (softcap == 0.0 or (softcap >= 1e-6 and math.isfinite(softcap))):
        raise ValueError("softcap must be 0 (none), or finite and at least 1e-6")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Unsupported reduction: {reduction}")
    device = _lib.require_cuda(x, weight, target)
    if weight.device != device or target.device != device:
        raise ValueError("x, weight and target must be on the same device")
    _lib.check_status("linear cross entropy")
    if target.dtype != torch.long or not target.is_contiguous():
        target = target.to(torch.long).contiguous()
    args = (x, weight, target, scale, softcap, int(ignore_index), _REDUCTIONS[reduction])
    if _lib.past_autograd((x, weight)):
        return _LinearCrossEntropy.forward(None, *args)
    return _LinearCrossEntropy.apply(*args)
