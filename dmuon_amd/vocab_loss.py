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


def _dense_float(t: Tensor) -> Tensor:
    if t.dtype is torch.float32 and t.is_contiguous() and not t.requires_grad:
        return t                           # each no-op of torch costs a microsecond of the host
    return t.detach().to(torch.float32).contiguous()


class _Targets:
    """What a call is measured against, and the launches on it."""

    def __init__(self, targets: Optional[Tensor] = None, ids: Optional[Tensor] = None,
                 logits: Optional[Tensor] = None, lse: Optional[Tensor] = None, *,
                 ignore_index: int = -100, z_loss: float = 0.0, temperature: float = 1.0,
                 k_list: int = 1, chunk: int = 0) -> None:
        self.tensors = targets, ids, logits, lse
        self.pointers = tuple(None if t is None else t.data_ptr() for t in self.tensors)
        self.k_list, self.chunk, self.ignore_index = k_list, chunk, ignore_index
        self.z_loss, self.temperature = z_loss, temperature

    def launch(self, hidden: Tensor, weight: Tensor, reduction: int, want, grad_dtype: torch.dtype,
               row_grad: Optional[Tensor] = None):
        """(the loss, of each token or reduced, d_hidden, d_weight); ``want`` says which gradients."""
        dev = hidden.device
        n, dim = hidden.shape
        vocab = weight.shape[0]
        loss = torch.empty(() if reduction else n, dtype=torch.float32, device=dev)
        dh = torch.empty((n, dim), dtype=grad_dtype, device=dev) if want[0] else None
        dw = torch.empty((vocab, dim), dtype=grad_dtype, device=dev) if want[1] else None
        a = _C.HeadLossArgs(
            hidden.data_ptr(), weight.data_ptr(), *self.pointers,
            None if row_grad is None else row_grad.data_ptr(),
            None if reduction else loss.data_ptr(), loss.data_ptr() if reduction else None,
            None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(),
            _pitch(hidden), _pitch(weight), n, vocab, dim, self.k_list, self.chunk,
            self.ignore_index, self.z_loss, self.temperature, _CODES[hidden.dtype],
            _CODES.get(grad_dtype, _C.DTYPE_F32), reduction)
        need = _C.c_i64()
        _C.call("dmuon_head_loss_workspace_size", ctypes.byref(a), ctypes.byref(need))
        # from the caching allocator: reused in this stream's order, nothing is kept
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        _C.call_on(dev, "dmuon_head_loss", ctypes.byref(a), ws.data_ptr(), need.value)
        return loss, dh, dw


def _scaled(grads, dtype: torch.dtype, factor: Tensor):
    """The gradients (two, each may be None) times ``factor`` in ``dtype``, in place where they have
    it."""
    factor = _dense_float(factor)
    out = [g if g is None or g.dtype == dtype else torch.empty_like(g, dtype=dtype) for g in grads]
    args = []
    for g, o in zip(grads, out):
        args += (None, None, 0) if g is None else (g.data_ptr(), o.data_ptr(), g.numel())
    held = next(g.dtype for g in grads if g is not None)
    _C.call_on(factor.device, "dmuon_scale_by", *args, _CODES.get(held, _C.DTYPE_F32),
               _CODES[dtype], factor.data_ptr())
    return out


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, reduction, grads):
        want = ctx.needs_input_grad[:2]
        # fp16: the mean's gradients may only fit the type once a loss scale has multiplied them
        held = torch.float32 if hidden.dtype == torch.float16 and reduction else hidden.dtype
        now = grads and reduction and (want[0] or want[1])
        loss, dh, dw = targets.launch(hidden, weight, reduction, want if now else (False, False),
                                      held)
        if grads:
            ctx.call, ctx.dtype = (targets, reduction, want, held), hidden.dtype
            ctx.grads = (dh, dw) if now else None
            ctx.save_for_backward(hidden, weight)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        grads, ctx.grads = ctx.grads, None
        if grads is None:                  # unreduced losses, or a second pass over a kept graph
            targets, reduction, want, held = ctx.call
            row_grad = None if reduction else _dense_float(grad)
            _, *grads = targets.launch(*ctx.saved_tensors, reduction, want, held, row_grad)
            if not reduction:
                return (*grads, None, None, None)
        return (*_scaled(grads, ctx.dtype, grad), None, None, None)


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
    if t.shape != shape:
        raise ValueError(f"{who}: {name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{who}: {name} must live on {device}")
    return t if t.dtype is torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def _floats(who: str, name: str, t: Tensor, shape, device) -> Tensor:
    if not t.dtype.is_floating_point or t.shape != shape:
        raise ValueError(f"{who}: {name} must be floating-point of the shape {tuple(shape)}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{who}: {name} must live on {device}")
    return _dense_float(t)


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
    t = _index(who, "target", target, hidden.shape[:-1], hidden.device)
    return _run(_Targets(t, ignore_index=int(ignore_index), z_loss=float(z_loss),
                         chunk=int(chunk_tokens or 0)), hidden, weight, reduction)


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
    logits = _floats(who, "teacher_logits", teacher_logits, ids.shape, hidden.device)
    lse = None if teacher_lse is None else \
        _floats(who, "teacher_lse", teacher_lse, hidden.shape[:-1], hidden.device)
    return _run(_Targets(None, ids, logits, lse, temperature=float(temperature), k_list=k,
                         chunk=int(chunk_tokens or 0)), hidden, weight, reduction)
