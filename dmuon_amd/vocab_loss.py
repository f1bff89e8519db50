"""Losses over a large vocabulary without the logits, with their gradients, on the HIP kernels.

``linear_cross_entropy`` is the cross entropy of ``hidden @ weight.T`` against the next token,
``linear_distillation`` the divergence from a teacher of which the top logits are known. Both run
``dmuon_head_loss``: the rows go through in chunks whose logits live in a workspace, so the memory
does not grow with the number of tokens, and in training the gradients are formed in the forward
pass, where the logits are (``backward`` only multiplies them by the incoming gradient). There is
no CPU path: tensors must live on the GPU.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _C

_CODES = {torch.bfloat16: _C.DTYPE_BF16, torch.float16: _C.DTYPE_F16}
_REDUCTIONS = {"none": _C.LOSS_ROWS, "mean": _C.LOSS_MEAN, "sum": _C.LOSS_SUM}


def _dense_rows(t: Tensor) -> Tensor:
    """``t`` with its last dimension contiguous and rows that do not overlap."""
    if t.dim() != 2 or (t.stride(1) == 1 or t.shape[1] == 1) and \
            (t.stride(0) >= t.shape[1] or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _pitch(t: Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


class _Targets:
    """What a call is measured against, and the launches on it."""

    def __init__(self, who: str, **tensors: Optional[Tensor]) -> None:
        self.who, self.tensors = who, tensors
        self.ignore_index, self.z_loss, self.temperature, self.k_list = -100, 0.0, 1.0, 1
        self.chunk = 0

    def launch(self, hidden: Tensor, weight: Tensor, reduction: int, want, *,
               row_grad: Optional[Tensor] = None, grad_dtype: Optional[torch.dtype] = None):
        """(loss of each token, reduced loss, d_hidden, d_weight); ``want`` says which gradients."""
        dev, dt = hidden.device, hidden.dtype
        n, dim = hidden.shape
        vocab = weight.shape[0]
        grad_dtype = grad_dtype or dt
        loss = torch.empty(n, dtype=torch.float32, device=dev)
        reduced = torch.empty((), dtype=torch.float32, device=dev) if reduction else None
        dh = torch.empty(n, dim, dtype=grad_dtype, device=dev) if want[0] else None
        dw = torch.empty(vocab, dim, dtype=grad_dtype, device=dev) if want[1] else None
        a = _C.HeadLossArgs(
            dtype=_CODES[dt], grad_dtype=_CODES.get(grad_dtype, _C.DTYPE_F32), reduction=reduction,
            tokens=n, vocab=vocab, dim=dim, k_list=self.k_list, chunk_tokens=self.chunk,
            ld_hidden=_pitch(hidden), ld_weight=_pitch(weight), ignore_index=self.ignore_index,
            z_loss=self.z_loss, temperature=self.temperature)
        for name, t in (("hidden", hidden), ("weight", weight), ("row_grad", row_grad),
                        ("loss", loss), ("reduced", reduced), ("d_hidden", dh), ("d_weight", dw),
                        *self.tensors.items()):
            if t is not None:
                setattr(a, name, t.data_ptr())
        need = _C.c_i64()
        _C.call("dmuon_head_loss_workspace_size", ctypes.byref(a), ctypes.byref(need))
        # from the caching allocator: reused in this stream's order, nothing is kept
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        _C.call_on(dev, "dmuon_head_loss", ctypes.byref(a), ws.data_ptr(), need.value)
        return loss, reduced, dh, dw


def _scaled(g: Optional[Tensor], dtype: torch.dtype, factor: Tensor) -> Optional[Tensor]:
    """``g * factor`` in ``dtype``, in place where ``g`` has it."""
    if g is None:
        return None
    out = g if g.dtype == dtype else torch.empty_like(g, dtype=dtype)
    _C.call_on(g.device, "dmuon_scale_by", g.data_ptr(), _CODES.get(g.dtype, _C.DTYPE_F32),
               out.data_ptr(), _CODES.get(dtype, _C.DTYPE_F32), g.numel(), factor.data_ptr())
    return out


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, reduction, grads):
        want = ctx.needs_input_grad[:2]
        ctx.targets, ctx.reduction = targets, reduction
        # fp16: the mean's gradients may only fit the type once a loss scale has multiplied them
        ctx.held_dtype = torch.float32 if hidden.dtype == torch.float16 else hidden.dtype
        now = grads and reduction and any(want)
        loss, reduced, dh, dw = targets.launch(hidden, weight, reduction, want if now else (0, 0),
                                               grad_dtype=ctx.held_dtype)
        ctx.grads = (dh, dw) if now else None
        ctx.save_for_backward(hidden, weight)
        return reduced if reduction else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        if not ctx.reduction:
            _, _, dh, dw = ctx.targets.launch(hidden, weight, ctx.reduction, want,
                                              row_grad=grad.float().contiguous())
            return dh, dw, None, None, None
        grads, ctx.grads = ctx.grads, None
        if grads is None:                  # a second pass over a retained graph
            grads = ctx.targets.launch(hidden, weight, ctx.reduction, want,
                                       grad_dtype=ctx.held_dtype)[2:]
        factor = grad.float().contiguous()
        return (*(_scaled(g, hidden.dtype, factor) for g in grads), None, None, None)


def _check(who: str, hidden: Tensor, weight: Tensor, reduction: str, chunk_tokens) -> None:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{who}: reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{who}: hidden [..., dim] and weight [vocab, dim] do not fit: "
                         f"{tuple(hidden.shape)}, {tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{who}: weight has no values: {tuple(weight.shape)}")
    if hidden.dtype not in _CODES or weight.dtype != hidden.dtype:
        raise ValueError(f"{who}: hidden and weight must both be bfloat16 or float16, got "
                         f"{hidden.dtype} and {weight.dtype}")
    if hidden.device.type != "cuda" or weight.device != hidden.device:
        raise RuntimeError(f"{who}: tensors must live on one GPU (HIP kernel only)")
    if chunk_tokens is not None and int(chunk_tokens) < 1:
        raise ValueError(f"{who}: chunk_tokens must be positive, got {chunk_tokens}")


def _index(who: str, name: str, t: Tensor, shape, device) -> Tensor:
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise ValueError(f"{who}: {name} must be integers, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{who}: {name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{who}: {name} must live on {device}")
    return t.to(torch.int64).contiguous()


def _run(targets: _Targets, hidden: Tensor, weight: Tensor, reduction: str) -> Tensor:
    shape = hidden.shape[:-1]
    # a two-dimensional hidden takes no view: it would be a node of the gradient's graph
    rows = _dense_rows(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1]))
    out = _HeadLoss.apply(rows, _dense_rows(weight), targets, _REDUCTIONS[reduction],
                          torch.is_grad_enabled())
    return out.view(shape) if reduction == "none" and len(shape) != 1 else out


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

    ``chunk_tokens`` bounds the rows of logits held at a time (default: about 4 GiB of workspace).
    Can be captured into a graph.
    """
    who = "linear_cross_entropy"
    _check(who, hidden, weight, reduction, chunk_tokens)
    t = _Targets(who, targets=_index(who, "target", target, hidden.shape[:-1], hidden.device))
    t.ignore_index, t.z_loss, t.chunk = int(ignore_index), float(z_loss), int(chunk_tokens or 0)
    return _run(t, hidden, weight, reduction)


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
    loss. Gradients go to ``hidden`` and ``weight``, not to the teacher. Types, ``reduction`` and
    ``chunk_tokens`` as in ``linear_cross_entropy``.
    """
    who = "linear_distillation"
    _check(who, hidden, weight, reduction, chunk_tokens)
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError(f"{who}: temperature must be positive, got {temperature}")
    if teacher_ids.dim() != hidden.dim() or not 1 <= teacher_ids.shape[-1] <= 4096:
        raise ValueError(f"{who}: teacher_ids must be [..., k] with 1 <= k <= 4096, got "
                         f"{tuple(teacher_ids.shape)}")
    k = teacher_ids.shape[-1]
    ids = _index(who, "teacher_ids", teacher_ids, (*hidden.shape[:-1], k), hidden.device)
    given = {"teacher_logits": (teacher_logits, ids.shape)}
    if teacher_lse is not None:
        given["teacher_lse"] = (teacher_lse, hidden.shape[:-1])
    floats = {}
    for name, (x, shape) in given.items():
        if not x.dtype.is_floating_point or x.shape != shape:
            raise ValueError(f"{who}: {name} must be floating-point of the shape {tuple(shape)}, "
                             f"got {x.dtype} {tuple(x.shape)}")
        if x.device != hidden.device:
            raise RuntimeError(f"{who}: {name} must live on {hidden.device}")
        floats[name] = x.detach().float().contiguous()
    t = _Targets(who, teacher_ids=ids, **floats)
    t.temperature, t.k_list, t.chunk = float(temperature), k, int(chunk_tokens or 0)
    return _run(t, hidden, weight, reduction)
