"""The norms around a block, fused with its gate and residual scale, on the HIP kernels.

``residual_norm`` takes the residual stream and a block's output to the new stream and the next
block's input in one pass over memory, and its gradients in another
(``dmuon_residual_norm`` / ``dmuon_residual_norm_grad``). There is no CPU path: tensors must live
on the GPU.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _C
from .vocab_loss import _dense_rows, _pitch

_CODES = {torch.float32: _C.DTYPE_F32, torch.bfloat16: _C.DTYPE_BF16, torch.float16: _C.DTYPE_F16}
_MAX_DIM = 16384


def _describe(x, y, pre, post, gate, scale, eps):
    a = _C.ResidualNormArgs(rows=x.shape[0], dim=x.shape[1], scale=scale, eps=eps, ld_x=_pitch(x),
                            dtype=_CODES[x.dtype], x=x.data_ptr())
    if y is not None:
        a.y, a.ld_y = y.data_ptr(), _pitch(y)
    for name, t in (("pre", pre), ("post", post), ("gate", gate)):
        if t is not None:
            setattr(a, name if name == "gate" else "w_" + name, t.data_ptr())
            setattr(a, name + "_dtype", _CODES[t.dtype])
    if gate is not None:
        a.gates = gate.shape[0]
    return a


def _gate_rows(who: str, gate: Tensor, x: Tensor) -> Tensor:
    """The gate as [g, dim], row i for the i-th of g equal runs of x's rows."""
    dim, lead, over = x.shape[-1], gate.shape[:-1], x.shape[:-1]
    fits = gate.dim() >= 1 and gate.shape[-1] == dim
    if fits and x.dim() == 2 and gate.dim() == 2:
        fits = lead[0] >= 1 and over[0] % lead[0] == 0
    elif fits and gate.dim() > 1:
        # leading dimensions of x, then ones: what broadcasting spreads over consecutive rows
        same = 0
        while same < len(lead) and len(lead) == len(over) and lead[same] == over[same]:
            same += 1
        fits = len(lead) == len(over) and all(n == 1 for n in lead[same:])
    if not fits:
        raise ValueError(f"{who}: a gate of {tuple(gate.shape)} has no row for each of equal runs "
                         f"of the rows of x {tuple(x.shape)}")
    if not gate.numel():
        return gate.new_zeros(1, dim)
    return gate if gate.dim() == 2 else gate.reshape(-1, dim)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, pre, post, gate, scale, eps, grads):
        ctx.scalars = scale, eps
        a = _describe(x, y, pre, post, gate, scale, eps)
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        x_new = torch.empty_like(h) if y is not None or scale != 1.0 else None
        stats = None
        if grads:
            stats = torch.empty(x.shape[0], 2, dtype=torch.float32, device=x.device)
            a.stats = stats.data_ptr()
        a.h = h.data_ptr()
        if x_new is not None:
            a.x_new = x_new.data_ptr()
        _C.call_on(x.device, "dmuon_residual_norm", ctypes.byref(a))
        ctx.save_for_backward(x, y, pre, post, gate, stats)
        ctx.set_materialize_grads(False)
        return x_new, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_new, dh):
        x, y, pre, post, gate, stats = ctx.saved_tensors
        a = _describe(x, y, pre, post, gate, *ctx.scalars)
        a.stats = stats.data_ptr()
        held = []
        for name, g in (("dx_new", dx_new), ("dh", dh)):
            if g is not None:
                g = _dense_rows(g)
                held.append(g)
                setattr(a, name, g.data_ptr())
                setattr(a, "ld_" + name, _pitch(g))
        out = []
        for name, t, need in zip(("dx", "dy", "d_pre", "d_post", "d_gate"),
                                 (x, y, pre, post, gate), ctx.needs_input_grad):
            g = None
            if t is not None and need:
                g = torch.empty_like(t, memory_format=torch.contiguous_format)
                setattr(a, name, g.data_ptr())
            out.append(g)
        need = _C.c_i64()
        _C.call("dmuon_residual_norm_grad_workspace_size", ctypes.byref(a), ctypes.byref(need))
        ws = torch.empty(need.value, dtype=torch.uint8, device=x.device)
        _C.call_on(x.device, "dmuon_residual_norm_grad", ctypes.byref(a), ws.data_ptr(), need.value)
        return (*out, None, None, None)


def residual_norm(x: Tensor, y: Optional[Tensor], pre_weight: Tensor, *,
                  post_weight: Optional[Tensor] = None, gate: Optional[Tensor] = None,
                  residual_scale: float = 1.0, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    """From the residual stream ``x`` and a block's output ``y`` (both ``[..., dim]``) to the new
    stream and the next block's input::

        u     = y * rsqrt(mean(y**2) + eps) * post_weight        (post_weight None: u = y)
        x_new = residual_scale * x + gate * u                    (gate None: 1)
        h     = x_new * rsqrt(mean(x_new**2) + eps) * pre_weight

    Returns ``(x_new, h)``. ``y=None`` is the first block's norm: ``x_new`` is the scaled ``x``.
    ``x`` and ``y`` share a dtype (fp32, bf16 or fp16) that the results have too; the weights
    (``[dim]``) and the gate may have it or fp32, each on its own. ``gate`` is ``[dim]``, or
    has ``x``'s leading dimensions followed by ones (``[b, 1, dim]``: a gate per sequence;
    ``x.shape``: per token); for a two-dimensional ``x`` it may be ``[g, dim]``, one row for every
    ``rows / g`` consecutive rows. Arithmetic is fp32 and every result is rounded once; the
    gradients of the weights and of a shared gate sum in a fixed order. Can be captured into a
    graph.
    """
    who = "residual_norm"
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_DIM:
        raise ValueError(f"{who}: x must be [..., dim] with 1 <= dim <= {_MAX_DIM}, got "
                         f"{tuple(x.shape)}")
    if x.dtype not in _CODES:
        raise ValueError(f"{who}: unsupported dtype {x.dtype}")
    dim = x.shape[-1]
    if y is not None and (y.shape != x.shape or y.dtype != x.dtype):
        raise ValueError(f"{who}: y must match x ({tuple(x.shape)}, {x.dtype}), got "
                         f"{tuple(y.shape)}, {y.dtype}")
    if y is None and (post_weight is not None or gate is not None):
        raise ValueError(f"{who}: post_weight and gate need the block's output y")
    for name, t in (("pre_weight", pre_weight), ("post_weight", post_weight)):
        if t is not None and tuple(t.shape) != (dim,):
            raise ValueError(f"{who}: {name} must be [{dim}], got {tuple(t.shape)}")
    # a two-dimensional x takes no views: each would be a node of the gradient's graph
    flat = x.dim() == 2
    rows = x if flat else x.reshape(-1, dim)
    if gate is not None:
        gate = _gate_rows(who, gate, x)
    for name, t in (("pre_weight", pre_weight), ("post_weight", post_weight), ("gate", gate)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{who}: {name} must be {x.dtype} or float32, got {t.dtype}")
    for t in (x, y, pre_weight, post_weight, gate):
        if t is not None and (t.device.type != "cuda" or t.device != x.device):
            raise RuntimeError(f"{who}: tensors must live on one GPU (HIP kernel only)")
    contiguous = (None if t is None else t.contiguous() for t in (pre_weight, post_weight, gate))
    x_new, h = _ResidualNorm.apply(_dense_rows(rows),
                                   None if y is None else _dense_rows(y if flat else y.reshape(-1, dim)),
                                   *contiguous, float(residual_scale), float(eps),
                                   torch.is_grad_enabled())
    if x_new is None:
        x_new = x
    return (x_new, h) if flat else (x_new.view(x.shape), h.view(x.shape))
