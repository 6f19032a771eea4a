"""Kernel attention over ragged batches of graphs and padded clouds.

Attention of the points (nodes) of each graph over the points of the same
graph, with an optional Gaussian kernel of the points' distances: the score
of query i and key j in head h is

    softcap * tanh(u / softcap) or u,  u = scale * q_i . k_j,
    minus |p_i - p_j|^2 / (2 sigma_h^2)

so with q = k = 0 the weights are the kernel terms that ``kde_mmd_loss`` adds
up, normalised per point.  ``pyg_kernel_attention`` takes ragged batches (ptr
offsets or sorted batch vectors, as ``pyg_kde_mmd_loss``),
``kernel_attention_dense`` padded clouds with masks (as
``kde_mmd_loss_dense``).  Both are differentiable in q, k, v, the positions and
sigma.  Inputs must be CUDA tensors: there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .kde import _ensure_ptr, _read_back

Tensor = torch.Tensor

__all__ = ["AttentionSegments", "attention_segments", "kernel_attention_dense",
           "pyg_kernel_attention"]

_TILE = 128  # rows of a work item
_MAX_DIM = 256


@dataclass(frozen=True)
class AttentionSegments:
    """The graphs of a ragged batch as the attention kernels take them: made
    (and checked) once per batch by ``attention_segments``, used by any number
    of calls.  Holds its own copy of the offsets."""
    q_ptr: Tensor
    k_ptr: Tensor
    q_tiles: Tensor
    k_tiles: Tensor
    graphs: int
    num_q: int
    num_k: int
    max_q: int
    max_k: int


def _tiles(first: Tensor, lengths: Tensor, other_first: Tensor, other_lengths: Tensor,
           total: int) -> Tensor:
    """Every 128 rows of every graph: their first row and count, then the other
    side's first row and count; the tiles with the most work first."""
    dev = lengths.device
    if total == 0:
        return torch.zeros((0, 4), dtype=torch.int32, device=dev)
    order = torch.argsort(other_lengths, descending=True, stable=True)
    lengths = lengths[order]
    each = (lengths + _TILE - 1) // _TILE
    graph = torch.repeat_interleave(each, output_size=total)  # places in `order`
    row = (torch.arange(total, device=dev) - (each.cumsum(0) - each)[graph]) * _TILE
    count = (lengths[graph] - row).clamp(max=_TILE)
    graph = order[graph]
    return torch.stack([first[graph] + row, count, other_first[graph], other_lengths[graph]],
                       1).to(torch.int32).contiguous()


def attention_segments(q_ptr: Optional[Tensor] = None, k_ptr: Optional[Tensor] = None, *,
                       q_batch: Optional[Tensor] = None,
                       k_batch: Optional[Tensor] = None) -> AttentionSegments:
    """Checks the graphs' offsets (one host synchronisation) and lays out the
    work.  Queries and keys come as ptr offsets (graphs + 1) or sorted batch
    vectors; without keys' the keys are the queries' rows (self-attention)."""
    if q_ptr is None and q_batch is None:
        raise ValueError("either ptr or batch must be provided")
    device = _lib.require_cuda(q_ptr if q_ptr is not None else q_batch)
    qp = _ensure_ptr(q_ptr, q_batch, 0 if q_batch is None else q_batch.numel(), device)[0].clone()
    if k_ptr is None and k_batch is None:
        kp = qp
    else:
        kp = _ensure_ptr(k_ptr, k_batch, 0 if k_batch is None else k_batch.numel(),
                         device)[0].clone()
    if qp.numel() != kp.numel():
        raise ValueError("query and key batches must have the same length")
    graphs = qp.numel() - 1
    nq, nk = qp[1:] - qp[:-1], kp[1:] - kp[:-1]
    zero = torch.zeros((), dtype=torch.long, device=device)

    def facts(p, n):
        if graphs == 0:
            return [p[0], p[0], zero, zero, zero]
        return [p[0], p[-1], n.min(), n.max(), ((n + _TILE - 1) // _TILE).sum()]

    info = _read_back(torch.stack(facts(qp, nq) + facts(kp, nk)))
    for first, _, least, _, _ in (info[:5], info[5:]):
        if first != 0:
            raise ValueError("ptr must start at 0")
        if least < 0:
            raise ValueError("ptr offsets must match node stacks")
    if max(info[1], info[6]) > 2 ** 31 - 256:
        raise ValueError("attention_segments: at most 2^31 - 256 rows")
    return AttentionSegments(qp, kp, _tiles(qp[:-1], nq, kp[:-1], nk, info[4]),
                             _tiles(kp[:-1], nk, qp[:-1], nq, info[9]), graphs, info[1], info[6],
                             info[3], info[8])


def _rows(t: Tensor) -> Tensor:
    """`t` as rows of heads (rows, heads, dim), the leading dimensions of a padded
    batch as one: unit stride along the head dimension, and for the 16-bit
    tensor-core kernels (widths that are multiples of 8) 16-byte aligned rows
    and no broadcast; copied where it is not so.  (Called without autograd: a
    view for it costs more than a small kernel.)"""
    if t.dim() == 4:
        b, n = t.shape[:2]
        if b != 1 and n != 1 and t.stride(0) != n * t.stride(1):
            t = t.contiguous()
        t = t.flatten(0, 1)
    strides, shape = t.stride(), t.shape
    ok = strides[2] == 1 or shape[2] == 1
    if ok and t.dtype != torch.float32 and shape[2] % 8 == 0:
        ok = t.data_ptr() % 16 == 0 and all(
            strides[i] % 8 == 0 and (strides[i] > 0 or shape[i] == 1) for i in (0, 1))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _floats(t: Tensor) -> Tensor:
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _dense16(t: Tensor) -> Tensor:
    """`t` contiguous, on a 16-byte boundary."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _operands(d, q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, plan):
    """What the kernels read of one pass's tensors: the strides into `d`, the
    addresses, and the tensors these belong to (copies among them), which have to
    live until the pass is launched."""
    qr, kr, vr = _rows(q), _rows(k), _rows(v)
    d.q_row, d.q_head, _ = qr.stride()
    d.k_row, d.k_head, _ = kr.stride()
    d.v_row, d.v_head, _ = vr.stride()
    q_mask, k_mask = _dense(q_mask), _dense(k_mask)
    if q_pos is not None:
        d.pos_dim = q_pos.shape[-1]
        q_pos, k_pos = _floats(q_pos), _floats(k_pos)
        if sigma.dtype != torch.float32 or sigma.device != q.device:
            sigma = sigma.to(device=q.device, dtype=torch.float32)
        if sigma.shape != (d.heads,) or not sigma.is_contiguous():
            sigma = sigma.reshape(-1).expand(d.heads).contiguous()
    kept = (qr, kr, vr, *plan, q_pos, k_pos, sigma, q_mask, k_mask)
    return _lib.RaAttnInputs(*[None if t is None else t.data_ptr() for t in kept]), kept


class _KernelAttention(torch.autograd.Function):
    """(q, k, v, q_pos, k_pos, sigma) -> out, for rows of heads or padded
    batches of them."""

    @staticmethod
    def forward(ctx, q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, shape, scale, softcap):
        lib = _lib.load()
        need_grad = ctx is not None
        dev = q.device
        d = _lib.RaAttnDesc()
        (d.graphs, d.num_q, d.num_k, d.max_q, d.max_k) = shape[:5]
        q_ptr, k_ptr, q_tiles, k_tiles = plan = shape[5:]
        if q_ptr is None:
            d.q_tiles = d.graphs * -(-d.max_q // _TILE)
            d.k_tiles = d.graphs * -(-d.max_k // _TILE)
        else:
            d.q_tiles, d.k_tiles = q_tiles.shape[0], k_tiles.shape[0]
        d.heads, d.kv_heads, d.dim = q.shape[-2], k.shape[-2], q.shape[-1]
        d.dtype, d.scale, d.softcap = _lib.DTYPES[q.dtype], scale, softcap
        d.status = _lib.status_word()
        inp, kept = _operands(d, q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, plan)
        if not need_grad and (q.dtype != torch.float32 or all(
                t.data_ptr() % 16 == 0 and t.stride(0) % 4 == 0 and t.stride(1) % 4 == 0
                for t in kept[:3])):
            d.forward_only = 1
        ref = ctypes.byref(d)
        with _lib.on_device(dev):
            out = _lib.empty_as(q)
            out32 = None
            n_stats = 0
            if need_grad:
                # unrounded outputs: the backward's do.o would carry the
                # rounding of 16 bits into every score's gradient
                if q.dtype != torch.float32:
                    out32 = _lib.empty_as(q, torch.float32)
                n_stats = 8 * d.heads * d.num_q
            n_state, n_ws = lib.ra_attn_state_bytes(ref), lib.ra_attn_workspace_bytes(ref, 0)
            # the state, a small workspace and the statistics share a buffer
            held = (n_state + 255) // 256 * 256
            at_stats = held + (n_ws if n_ws <= 256 else 0)
            state = _lib.scratch(at_stats + n_stats, dev)
            ws = None if n_ws <= 256 else _lib.scratch(n_ws, dev)
            base = state.data_ptr()
            stats = base + at_stats if n_stats else None
            rc = lib.ra_attn_forward(ref, ctypes.byref(inp), out.data_ptr(), _lib.ptr(out32),
                                     stats, base, n_state,
                                     base + held if ws is None else ws.data_ptr(), n_ws,
                                     _lib.stream_handle(dev))
        _lib.check(rc, "kernel attention")
        if need_grad:
            ctx.desc, ctx.at_stats = d, at_stats
            # all of it saved, so that it is freed with the graph
            ctx.save_for_backward(q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, *plan,
                                  out if out32 is None else out32, state)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        lib = _lib.load()
        # not always the forward's tensors: a checkpoint makes them again, hooks
        # on saved tensors may bring them back elsewhere and with other strides
        *saved, out32, state = ctx.saved_tensors
        q, k, v, q_pos, k_pos, sigma = saved[:6]
        d, dev = ctx.desc, q.device
        inp, kept = _operands(d, *saved[:8], saved[8:])
        g, out32 = _dense16(g), _dense16(out32)
        need = ctx.needs_input_grad
        with _lib.on_device(dev):
            state = _lib.aligned(state)
            stats = state.data_ptr() + ctx.at_stats if d.num_q else None
            grads = [_lib.empty_as(t) if need[i] else None for i, t in enumerate((q, k, v))]
            grads += [_lib.empty_as(t, torch.float32) if t is not None and need[3 + i] else None
                      for i, t in enumerate((q_pos, k_pos))]
            grads.append(torch.empty(d.heads, dtype=torch.float32, device=dev) if need[5] else None)
            gr = _lib.RaAttnGrads(*[_lib.ptr(t) for t in grads])
            n_ws = lib.ra_attn_workspace_bytes(ctypes.byref(d), 1)
            ws = _lib.scratch(n_ws, dev)
            f32 = q.dtype == torch.float32
            rc = lib.ra_attn_backward(ctypes.byref(d), ctypes.byref(inp), g.data_ptr(),
                                      out32.data_ptr() if f32 else None,
                                      None if f32 else out32.data_ptr(), stats,
                                      ctypes.byref(gr), state.data_ptr(), state.numel(),
                                      ws.data_ptr(), ws.numel(), _lib.stream_handle(dev))
        _lib.check(rc, "kernel attention backward")
        for i, t in ((3, q_pos), (4, k_pos)):
            if grads[i] is not None and t.dtype != torch.float32:
                grads[i] = grads[i].to(t.dtype)
        if grads[5] is not None and not (sigma.shape == grads[5].shape and sigma.device == dev
                                         and sigma.dtype == torch.float32):
            s = grads[5] if sigma.numel() == d.heads else grads[5].sum()
            grads[5] = s.reshape(sigma.shape).to(device=sigma.device, dtype=sigma.dtype)
        return (*grads, None, None, None, None, None)


def _checked(q, k, v, ndim, shape_text):
    if q.ndim != ndim or k.ndim != ndim or v.ndim != ndim:
        raise ValueError(f"q, k and v must have shape {shape_text}")
    if k.shape != v.shape or q.shape[-1] != k.shape[-1]:
        raise ValueError("k and v must have the same shape, and q the same head dimension")
    if q.dtype not in _lib.DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share dtype float32, bfloat16 or float16")
    heads, kv_heads, dim = q.shape[-2], k.shape[-2], q.shape[-1]
    if heads < 1 or kv_heads < 1 or heads > 4096 or heads % kv_heads:
        raise ValueError("the heads of q must be a multiple of those of k and v")
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"head dimension must be between 1 and {_MAX_DIM}")
    if not (k.device == q.device and v.device == q.device):
        raise ValueError("q, k and v must be on the same device")


def _positions(q_pos, k_pos, sigma, num_q, num_k, heads, device):
    """Positions (rows, c) and sigma (heads,) or one, or three Nones.  `num`:
    the shape of the rows."""
    if q_pos is None:
        if k_pos is not None or sigma is not None:
            raise ValueError("positions of queries and sigma go together")
        return None, None, None
    if sigma is None:
        raise ValueError("positions need a sigma")
    if k_pos is None:
        k_pos = q_pos
    lead = len(num_q)
    if q_pos.ndim != lead + 1 or k_pos.ndim != lead + 1 or \
            q_pos.shape[-1] != k_pos.shape[-1] or not 1 <= q_pos.shape[-1] <= 3:
        raise ValueError("positions must have 1 to 3 coordinates, the same for queries and keys")
    if tuple(q_pos.shape[:-1]) != tuple(num_q) or tuple(k_pos.shape[:-1]) != tuple(num_k):
        raise ValueError("positions length must equal number of rows")
    if not (q_pos.is_floating_point() and k_pos.is_floating_point()):
        raise ValueError("positions must be floating point")
    if not isinstance(sigma, Tensor):
        if not sigma > 0:
            raise ValueError("sigma must be positive")
        sigma = torch.full((heads,), float(sigma), dtype=torch.float32, device=device)
    elif sigma.numel() != 1 and sigma.shape != (heads,):
        raise ValueError("sigma must be a scalar or one value per head")
    if q_pos.device != device or k_pos.device != device:
        raise ValueError("positions must be on the device of q")
    return q_pos, k_pos, sigma


def _factors(scale, softcap, dim):
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    softcap = float(softcap)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not (softcap == 0.0 or (softcap >= 1e-6 and math.isfinite(softcap))):
        raise ValueError("softcap must be 0 (none), or finite and at least 1e-6")
    return scale, softcap


def _mask(mask, shape, device):
    if mask is None:
        return None
    if tuple(mask.shape) != tuple(shape):
        raise ValueError(f"masks must have shape {tuple(shape)}")
    mask = mask.to(device=device, dtype=torch.bool)
    return (mask if mask.is_contiguous() else mask.contiguous()).view(torch.uint8)


def _run(q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, shape, scale, softcap):
    _lib.check_status("kernel attention")
    args = (q, k, v, q_pos, k_pos, sigma, q_mask, k_mask, shape, scale, softcap)
    if _lib.past_autograd(args[:6]):  # without autograd's share of a small call
        return _KernelAttention.forward(None, *args)
    return _KernelAttention.apply(*args)


def pyg_kernel_attention(q: Tensor, k: Tensor, v: Tensor, *, q_ptr: Optional[Tensor] = None,
                         k_ptr: Optional[Tensor] = None, q_batch: Optional[Tensor] = None,
                         k_batch: Optional[Tensor] = None,
                         segments: Optional[AttentionSegments] = None,
                         q_pos: Optional[Tensor] = None, k_pos: Optional[Tensor] = None,
                         sigma=None, q_mask: Optional[Tensor] = None,
                         k_mask: Optional[Tensor] = None, scale: Optional[float] = None,
                         softcap: float = 0.0) -> Tensor:
    """Attention inside each graph of a ragged batch.

    Args:
        q: (Nq, H, D), float32, bfloat16 or float16, D up to 256.
        k, v: (Nk, H', D) of the same dtype; H is a multiple of H', and heads
            h of q use head h // (H / H') of k and v.
        q_ptr, k_ptr / q_batch, k_batch: the graphs, as ptr offsets or sorted
            batch vectors; without the keys', keys are the queries' rows.
            Checked with one host synchronisation.
        segments: instead of those, ``attention_segments(...)`` of the batch:
            no call with it waits for the device (and it can be captured).
        q_pos, k_pos: (Nq, c), (Nk, c) positions, c = 1 to 3, with ``sigma``, a
            number or a tensor () or (H,): the Gaussian kernel's bandwidth.
            k_pos defaults to q_pos.  A number is checked; a tensor's zeros
            give NaN.
        q_mask, k_mask: (Nq,), (Nk,) booleans: masked keys take no part
            (whatever their rows hold), masked queries give 0.
        scale: factor of the products, 1 / sqrt(D) by default.
        softcap: where positive, products are capped by softcap * tanh.

    Returns:
        (Nq, H, D) in q's dtype; 0 for a query without keys.  Differentiable
        in q, k, v, the positions and sigma (bitwise repeatable).
    """
    _checked(q, k, v, 3, "(N, heads, dim)")
    scale, softcap = _factors(scale, softcap, q.shape[2])
    device = _lib.require_cuda(q, k, v)
    if segments is None:
        segments = attention_segments(q_ptr, k_ptr, q_batch=q_batch, k_batch=k_batch)
    elif any(t is not None for t in (q_ptr, k_ptr, q_batch, k_batch)):
        raise ValueError("give either segments or ptr and batch")
    if segments.num_q != q.shape[0] or segments.num_k != k.shape[0]:
        raise ValueError("ptr[-1] must equal number of nodes")
    if segments.q_ptr.device != device:
        raise ValueError("segments must be on the device of q")
    pos = _positions(q_pos, k_pos, sigma, q.shape[:1], k.shape[:1], q.shape[1], device)
    shape = (segments.graphs, segments.num_q, segments.num_k, segments.max_q, segments.max_k,
             segments.q_ptr, segments.k_ptr, segments.q_tiles, segments.k_tiles)
    return _run(q, k, v, *pos, _mask(q_mask, q.shape[:1], device),
                _mask(k_mask, k.shape[:1], device), shape, scale, softcap)


def kernel_attention_dense(q: Tensor, k: Tensor, v: Tensor, mask_q: Optional[Tensor] = None,
                           mask_k: Optional[Tensor] = None, *, q_pos: Optional[Tensor] = None,
                           k_pos: Optional[Tensor] = None, sigma=None,
                           scale: Optional[float] = None, softcap: float = 0.0) -> Tensor:
    """``pyg_kernel_attention`` on padded clouds: q (B, N, H, D), k and v
    (B, M, H', D), masks (B, N) and (B, M) of any pattern (None: all valid),
    positions (B, N, c) and (B, M, c).  Returns (B, N, H, D); masked queries
    and clouds without valid keys give 0, and what masked rows hold (NaN too)
    reaches no result and no gradient."""
    _checked(q, k, v, 4, "(B, N, heads, dim)")
    B, N, H, D = q.shape
    M = k.shape[1]
    if k.shape[0] != B:
        raise ValueError("q, k and v must have the same number of clouds")
    scale, softcap = _factors(scale, softcap, D)
    device = _lib.require_cuda(q, k, v)
    pos = _positions(q_pos, k_pos, sigma, (B, N), (B, M), H, device)
    shape = (B, B * N, B * M, N if B else 0, M if B else 0, None, None, None, None)
    return _run(q, k, v, *pos, _mask(mask_q, (B, N), device), _mask(mask_k, (B, M), device), shape,
                scale, softcap)
