"""The norms around a block, fused with its gate and residual scale, on the HIP kernels.

``residual_norm`` takes the residual stream and a block's output to the new stream and the next
block's input in one pass over memory, and its gradients in another
(``dmuon_residual_norm`` / ``dmuon_residual_norm_grad``). The autograd operator is native
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
