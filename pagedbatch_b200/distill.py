"""Distillation of a draft model from a teacher's top entries: the loss of each row of student logits
and its gradient, in one pass over the logits each way. The reference does not train
(pagedbatch has no optimiser) and has no counterpart.

The teacher's record of a row is what ``top_logprobs`` returns for it: K log-probabilities and token
ids. Formulas and edge cases are stated at ``pb_distill_forward`` in ``include/pagedbatch_b200.h``.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .logprobs import check_temperature

__all__ = ["distill_loss"]

STATS = 32  # bytes of a row's statistics (pb_distill_stats_bytes)


def _prepare(z, lp, idx, row_weight, temperature):
    """Refuses what the kernels do not take; the teacher's entries, the weights and the temperature as they take them."""
    if not z.is_cuda:
        raise ValueError("pagedbatch_b200.distill_loss needs CUDA logits; move the tensor with .cuda() first")
    if z.dim() != 2 or (z.stride(1) != 1 and z.shape[1] > 1):
        raise ValueError("student_logits must be a [rows, vocab] tensor with a contiguous last dimension")
    if z.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"unsupported student_logits dtype {z.dtype}")
    n, V = z.shape
    if not 1 <= V <= _lib.DISTILL_MAX_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {_lib.DISTILL_MAX_VOCAB} tokens, got {V}")
    if lp.dim() != 2 or lp.shape[0] != n or not 1 <= lp.shape[1] <= _lib.DISTILL_MAX_ENTRIES:
        raise ValueError(f"teacher_logprobs must be [{n}, K] with K in [1, {_lib.DISTILL_MAX_ENTRIES}]")
    if lp.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"unsupported teacher_logprobs dtype {lp.dtype}")
    if idx.shape != lp.shape or idx.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_indices must be int32 or int64, of teacher_logprobs' shape")
    if lp.requires_grad or (row_weight is not None and row_weight.requires_grad):
        raise ValueError("the teacher's entries and the row weights take no gradient: detach them")
    if row_weight is not None and (row_weight.dtype != torch.float32 or row_weight.shape != (n,)):
        raise ValueError(f"row_weight must be a float32 tensor of {n} values")
    dev = z.device
    if lp.device != dev or idx.device != dev or (row_weight is not None and row_weight.device != dev):
        raise ValueError(f"the teacher's entries and the row weights must be on the logits' device {dev}")
    t = check_temperature(temperature)
    if lp.dtype != torch.float32:
        lp = lp.float()
    if lp.stride(1) != 1:
        lp = lp.contiguous()
    if idx.stride(1) != 1:
        idx = idx.contiguous()
    if row_weight is not None:
        row_weight = row_weight.contiguous()
    return lp, idx, row_weight, t


def _arguments(z, lp, idx, temperature):
    """What the forward and the backward call have in common."""
    n, V = z.shape
    return (z.data_ptr(), ops._DTYPE_CODE[z.dtype], n, V, z.stride(0), lp.data_ptr(), lp.stride(0), idx.data_ptr(),
            idx.stride(0), 8 if idx.dtype == torch.int64 else 4, idx.shape[1], temperature)


def _forward(z, lp, idx, weight, temperature, tail, total):
    """The rows' losses (or their sum), and a buffer that starts with their statistics."""
    L = _lib.load()
    dev = z.device
    args = _arguments(z, lp, idx, temperature)
    n = args[2]
    n_ws = L.pb_distill_ws_bytes(n, args[3], args[1])
    buf = torch.empty(n * STATS + n_ws, dtype=torch.uint8, device=dev)  # statistics, then the launch's own workspace
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    base, stream = buf.data_ptr(), ops.raw_stream(dev)
    with ops.on_device(dev):
        _lib.check(L.pb_distill_forward(*args, tail, None if weight is None else weight.data_ptr(), loss.data_ptr(), base,
                                        base + n * STATS, n_ws, stream), "pb_distill_forward")
        if total:
            rows, loss = loss, torch.empty((), dtype=torch.float32, device=dev)
            _lib.check(L.pb_distill_sum(rows.data_ptr(), n, loss.data_ptr(), stream), "pb_distill_sum")
    return loss, buf


def _backward(z, lp, idx, weight, stats, temperature, grad_loss):
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    # a gradient of one value for all rows (from a sum or mean) is read through its stride of 0
    with ops.on_device(z.device):
        _lib.check(_lib.load().pb_distill_backward(
            *_arguments(z, lp, idx, temperature), None if weight is None else weight.data_ptr(), stats.data_ptr(),
            grad_loss.data_ptr(), grad_loss.stride(0) if grad_loss.dim() else 0, dz.data_ptr(), ops.raw_stream(z.device)),
            "pb_distill_backward")
    return dz


@torch.library.custom_op("pagedbatch_b200::distill_loss", mutates_args=())
def distill_op(student_logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_indices: torch.Tensor,
               row_weight: torch.Tensor | None, temperature: float, tail: bool,
               total: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows' losses (or their sum) and their statistics."""
    prepared = _prepare(student_logits, teacher_logprobs, teacher_indices, row_weight, temperature)
    loss, buf = _forward(student_logits, *prepared, tail, total)
    return loss, buf[: student_logits.shape[0] * STATS].clone()


@distill_op.register_fake
def _(student_logits, teacher_logprobs, teacher_indices, row_weight, temperature, tail, total):
    _prepare(student_logits, teacher_logprobs, teacher_indices, row_weight, temperature)
    n = student_logits.shape[0]
    return (student_logits.new_empty(() if total else (n,), dtype=torch.float32),
            student_logits.new_empty((n * STATS,), dtype=torch.uint8))


def _check_backward(z, stats, grad_loss):
    n = z.shape[0]
    if stats.dtype != torch.uint8 or stats.shape != (n * STATS,) or not stats.is_contiguous() or stats.device != z.device:
        raise ValueError("stats must be those of the forward call on the same rows")
    if grad_loss.dtype != torch.float32 or grad_loss.shape not in ((), (n,)) or grad_loss.device != z.device:
        raise ValueError(f"grad_loss must be one float32 value or {n} of them")


@torch.library.custom_op("pagedbatch_b200::distill_loss_backward", mutates_args=())
def distill_backward_op(student_logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_indices: torch.Tensor,
                        row_weight: torch.Tensor | None, stats: torch.Tensor, temperature: float,
                        grad_loss: torch.Tensor) -> torch.Tensor:
    """The gradient in the student's logits."""
    lp, idx, weight, t = _prepare(student_logits, teacher_logprobs, teacher_indices, row_weight, temperature)
    _check_backward(student_logits, stats, grad_loss)
    return _backward(student_logits, lp, idx, weight, stats, t, grad_loss)


@distill_backward_op.register_fake
def _(student_logits, teacher_logprobs, teacher_indices, row_weight, stats, temperature, grad_loss):
    _prepare(student_logits, teacher_logprobs, teacher_indices, row_weight, temperature)
    _check_backward(student_logits, stats, grad_loss)
    return student_logits.new_empty(student_logits.shape)


def _save(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:4], output[1])
    ctx.temperature = inputs[4]


def _backward_traced(ctx, grad_loss, _):
    dz = distill_backward_op(*ctx.saved_tensors, ctx.temperature, grad_loss)
    return dz, None, None, None, None, None, None


distill_op.register_autograd(_backward_traced, setup_context=_save)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, lp, idx, weight, temperature, tail, total):
        loss, stats = _forward(z, lp, idx, weight, temperature, tail, total)
        ctx.save_for_backward(z, lp, idx, weight, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        dz = _backward(*ctx.saved_tensors, ctx.temperature, grad_loss)
        return dz, None, None, None, None, None, None


def distill_loss(student_logits: torch.Tensor, teacher_logprobs: torch.Tensor, teacher_indices: torch.Tensor, *,
                 temperature: float = 1.0, tail: bool = False, row_weight: torch.Tensor | None = None,
                 reduction: str = "none") -> torch.Tensor:
    """KL divergence of the student's distribution from the teacher's, per row of ``student_logits
    [n, V]`` (CUDA, float32 / bfloat16 / float16, last dim contiguous, V at most 2^20): float32 ``[n]``,
    or their sum with ``reduction="sum"``. Differentiable in ``student_logits`` (once).

    * ``teacher_logprobs [n, K]`` (K at most 1024) and ``teacher_indices [n, K]`` (int32 or int64): the
      teacher's entries, index -1 for padding. The teacher's distribution is the softmax of the entries'
      values (any constant per row may be added to them), or with ``tail=True`` their exponentials, the
      rest of the mass being compared with the student's mass outside the entries.
    * ``temperature`` divides the student's logits (the teacher's entries are at it already; multiply
      the loss by its square for the usual scaling).
    * ``row_weight float32[n]``: a factor of each row's loss. Rows of weight 0, and rows whose entries
      are all padding, have loss and gradient 0 whatever their logits hold.

    An index outside [-1, V) makes its row's loss NaN."""
    if reduction not in ("none", "sum"):
        raise ValueError(f"reduction must be 'none' or 'sum', got {reduction!r}")
    z = student_logits
    lp, idx, row_weight, t = _prepare(z, teacher_logprobs, teacher_indices, row_weight, temperature)
    total = reduction == "sum"
    if ops.traced(z):
        return distill_op(z, lp, idx, row_weight, t, bool(tail), total)[0]
    if forward_ad._current_level >= 0 and any(  # (inside a level of dual tensors)
            a is not None and forward_ad.unpack_dual(a).tangent is not None for a in (z, lp, row_weight)):
        raise NotImplementedError("distill_loss has no forward-mode derivative")
    if not (z.requires_grad and torch.is_grad_enabled()):
        return _forward(z, lp, idx, row_weight, t, bool(tail), total)[0]
    return _Distill.apply(z, lp, idx, row_weight, t, bool(tail), total)
