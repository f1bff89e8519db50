"""The token lookup with its gradient, on the HIP kernels.

``embedding`` runs ``dmuon_embedding`` / ``dmuon_embedding_grad``; the gradient sorts the tokens and sums
each class's rows in their order. The autograd operator is native (``csrc/torch_binding.cpp``). There is
no CPU path: tensors must live on the GPU. Dual tensors, tracers and wrapper subclasses raise.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _C


def embedding(tokens: Tensor, weight: Tensor, *, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> Tensor:
    """``scale * weight[tokens]``: a row of ``weight`` ``[vocab, dim]`` (fp32, bf16 or fp16, rows of any
    pitch) for every token (integers of any shape), in ``weight``'s dtype. ``scale`` is 0 or a normal fp32
    number.

    The gradient of ``weight`` is dense and of its dtype; sums are fp32 in a fixed order, rounded once.
    Tokens equal to ``padding_idx`` (which may count from the vocabulary's end) have no share in it. A token
    outside the vocabulary gives a row of NaN and has no gradient. The gradient has no gradient of its own.
    Can be captured into a graph.
    """
    return _C.torch_ops().embedding(tokens, weight, float(scale),
                                    None if padding_idx is None else int(padding_idx))
