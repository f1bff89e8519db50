"""Losses over a large vocabulary without the logits, with their gradients, on the HIP kernels.

``linear_cross_entropy`` is the cross entropy of ``hidden @ weight.T`` against the next token,
``linear_distillation`` the divergence from a teacher of which the top logits are known. Both run
``dmuon_head_loss``: the rows go through in chunks whose logits live in a workspace, so that a token
more costs a few bytes and not a row of logits, and in training the gradients are formed in the
forward pass, where the logits are (``backward`` only multiplies them by the incoming gradient; a
bf16 gradient rounds again there unless the factor is a power of two). The autograd operators are
native (``csrc/torch_binding.cpp``). There is no CPU path: tensors must live on the GPU. Nor are
there forward-mode gradients or traces: dual tensors, ``torch.jit.trace`` and ``make_fx`` raise, and
so do wrapper subclasses, which have no memory of their own.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from . import _C

_REDUCTIONS = {"none": _C.LOSS_ROWS, "mean": _C.LOSS_MEAN, "sum": _C.LOSS_SUM}


def _options(who: str, reduction: str, chunk_tokens: Optional[int]) -> tuple:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{who}: reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if chunk_tokens is not None and int(chunk_tokens) < 1:
        raise ValueError(f"{who}: chunk_tokens must be positive, got {chunk_tokens}")
    return _REDUCTIONS[reduction], int(chunk_tokens or 0)


def linear_cross_entropy(hidden: Tensor, weight: Tensor, target: Tensor, *,
                         ignore_index: int = -100, z_loss: float = 0.0, reduction: str = "mean",
                         chunk_tokens: Optional[int] = None) -> Tensor:
    """Cross entropy of the logits ``hidden @ weight.T`` against ``target``, in fp32.

    ``hidden`` is ``[..., dim]``, ``weight`` ``[vocab, dim]`` (both bf16 or both fp16, rows of any
    pitch), ``target`` integers of ``hidden``'s leading shape. The loss of a token is
    ``lse - logit[target] + z_loss * lse**2`` with the log-sum-exp ``lse`` of its logits; tokens
    whose target is ``ignore_index`` have loss 0 and no gradient, and ``"mean"`` divides by the
    number of the others (0 where there are none). Any other target outside the vocabulary gives a
    NaN loss and NaN gradients. ``reduction="none"`` returns the tokens' losses; its backward pass
    forms the logits a second time, since the incoming gradients weigh the tokens.

    ``chunk_tokens`` bounds the rows of logits held at a time, in whole 256 past 256 (default: at most
    4 GiB of logits, their gradient and statistics); losses keep their bits. Several chunks sum the
    weight's gradient in fp32, 4 bytes a value of the weight, and small ones are slow (8192 tokens of
    128256 classes x 4096 in bf16: 19.3 ms and 2.1 GiB of workspace at once, 37.9 ms and 2.2 GiB in
    chunks of 1024): a bound for frozen weights, fp16 and long calls. The gradient has no gradient of
    its own. Can be captured into a graph.
    """
    return _C.torch_ops().linear_cross_entropy(
        hidden, weight, target, int(ignore_index), float(z_loss),
        *_options("linear_cross_entropy", reduction, chunk_tokens))


def linear_distillation(hidden: Tensor, weight: Tensor, teacher_ids: Tensor,
                        teacher_logits: Tensor, *, teacher_lse: Optional[Tensor] = None,
                        temperature: float = 1.0, reduction: str = "mean",
                        chunk_tokens: Optional[int] = None) -> Tensor:
    """Divergence of the student's distribution from a teacher's top logits, in fp32.

    With ``p = softmax(hidden @ weight.T / temperature)`` over the whole vocabulary and the
    teacher's probabilities ``q`` of the classes ``teacher_ids`` (``[..., k]``), a token's loss is
    ``temperature**2 * sum(q * (log q - log p[ids]))``. ``q`` is the softmax of
    ``teacher_logits / temperature`` over the list, or, where ``teacher_lse`` (``[...]``) gives the
    log-sum-exp of all of the teacher's logits over the temperature, ``exp(teacher_logits /
    temperature - teacher_lse)``: the teacher's own probabilities, whose missing tail then has no
    term. Negative ids are padding and logits of ``-inf`` have no weight; a token with padding only
    has loss 0, no gradient, and is not counted by ``"mean"``. Ids past the vocabulary give a NaN
    loss. ``temperature`` is a positive normal fp32 number. Gradients go to ``hidden`` and ``weight``, not to the teacher. Types, ``reduction`` and
    ``chunk_tokens`` as in ``linear_cross_entropy``.
    """
    # normal fp32 numbers: the kernels take its inverse too
    if not 2.0 ** -126 <= float(temperature) < 2.0 ** 128:
        raise ValueError("linear_distillation: temperature must be positive and within fp32, got "
                         f"{temperature}")
    return _C.torch_ops().linear_distillation(
        hidden, weight, teacher_ids, teacher_logits, teacher_lse, float(temperature),
        *_options("linear_distillation", reduction, chunk_tokens))
