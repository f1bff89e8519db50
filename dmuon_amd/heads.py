"""Attention over heads with its gradients, on the HIP kernels.

``attention`` runs ``dmuon_attention`` / ``dmuon_attention_grad``: one pass over the keys with the running
maximum and sum of each row, and gradients that form the probabilities anew, so that no matrix of scores
is held. The autograd operator is native (``csrc/torch_binding.cpp``). There is no CPU path: tensors must
live on the GPU. Dual tensors (forward-mode gradients), tracers and wrapper subclasses raise.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _C


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = True, window: Optional[int] = None,
              scale: Optional[float] = None, kv_lengths: Optional[Tensor] = None,
              q_starts: Optional[Tensor] = None, kv_starts: Optional[Tensor] = None) -> Tensor:
    """``softmax(scale * q k^T) v`` for every head, over the keys that a query sees.

    ``q`` is ``[batch, tokens, heads, dim]``, ``k`` and ``v`` ``[batch, kv_tokens, kv_heads, dim]`` (all
    bf16 or all fp16; ``heads`` a multiple of ``kv_heads``: each key head serves ``heads / kv_heads``
    consecutive query heads; ``dim`` a multiple of 8 up to 128); the result has ``q``'s shape. ``causal``
    lines the last query up with the last key: query ``i`` sees the keys up to ``i + kv_tokens - tokens``, and
    with a ``window`` the last ``window`` of those. A query that sees nothing gives 0 and has no gradient.
    ``scale`` defaults to ``dim ** -0.5``.

    ``kv_lengths`` (integers ``[batch]``) says how many keys of each sequence are there, as in a cache
    that is not full; what lies behind them is not read, and has the gradient 0. ``q_starts`` and
    ``kv_starts`` (integers ``[n + 1]``, not falling) say that ``q`` ``[tokens, heads, dim]`` and ``k``, ``v``
    ``[kv_tokens, kv_heads, dim]`` hold n sequences one behind the other, sequence ``i`` the tokens
    ``starts[i]`` to ``starts[i + 1]``; tokens in no sequence give 0 and have no gradient. None of these need
    be known on the host.

    Scores, sums and statistics are fp32; the probabilities, and in the gradient theirs, are rounded to
    the operands' type between the products. A value or key of no number (infinity or NaN) reaches every row
    that sees it, and may reach rows near those, whose mask hides it. (A key whose score is minus infinity has
    no share in a row; a row that sees only such keys is NaN, as the formula has it.) In the gradient a query
    or a gradient of no number likewise reaches the keys that its row sees, and may reach keys near those; of
    rows that see nothing they are not read. The same call gives the same bits. The gradient has no gradient
    of its own. Can be captured into a graph.
    """
    return _C.torch_ops().attention(
        q, k, v, bool(causal), None if window is None else int(window),
        None if scale is None else float(scale), kv_lengths, q_starts, kv_starts)
