"""The norms around a block and those of its attention's heads, on the HIP kernels.

``rotary_heads`` norms queries and keys head by head and turns them by their positions in one pass
(``dmuon_rotary_heads`` / ``dmuon_rotary_heads_grad``). ``residual_norm`` takes the residual stream and a block's output to the new stream and the next
block's input in one pass over memory, and its gradients in another
(``dmuon_residual_norm`` / ``dmuon_residual_norm_grad``). The autograd operators are native
(``csrc/torch_binding.cpp``). There is no CPU path: tensors must live on the GPU.
"""
from __future__ import annotations

from typing import Optional, Tuple

from torch import Tensor

from . import _C

_MAX_DIM = 16384


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
    gradients of the weights and of a shared gate sum in a fixed order, and have no gradients of their
    own. Dual tensors (forward-mode gradients), tracers and wrapper subclasses raise. Can be captured
    into a graph.
    """
    return _C.torch_ops().residual_norm(x, y, pre_weight, post_weight, gate, float(residual_scale),
                                        float(eps), _MAX_DIM)


def rotary_heads(q: Tensor, k: Tensor, positions: Tensor, inv_freq: Tensor, *,
                 q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """Queries ``q`` (``[..., heads, dim]``) and keys ``k`` (``[..., kv_heads, dim]``), normed head by
    head and rotated by their positions::

        z = x * rsqrt(mean(x**2) + eps) * weight           (weight None: z = x)
        y[i], y[j] = z[i] cos t - z[j] sin t, z[j] cos t + z[i] sin t,   t = position * inv_freq[i]

    with the pairs ``j = i + r / 2`` of the first ``r = 2 * len(inv_freq)`` values, or, ``interleaved``, the
    neighbours ``2 i`` and ``2 i + 1``; values behind them are not turned. ``positions`` are integers
    of the leading shape or of its trailing part (``[tokens]`` for a batch), ``inv_freq`` fp32 or fp64: the
    angle is formed and reduced in twice 64 bits, so that far positions (all of 64 bits, with frequencies up
    to 1) are as exact as near ones. ``q`` and ``k``
    share a dtype (fp32, bf16 or fp16) that the results, which are dense, have too; the weights (``[dim]``)
    may have it or fp32. ``dim`` is even and at most 512. Views into one product for q, k and v are read in
    place. Arithmetic is fp32, every result is rounded once; gradients go to q, k and the weights (their
    sums in a fixed order) and have none of their own. Dual tensors, tracers and wrapper subclasses raise.
    Can be captured into a graph.
    """
    return _C.torch_ops().rotary_heads(q, k, positions, inv_freq, q_weight, k_weight, float(eps),
                                       bool(interleaved))
