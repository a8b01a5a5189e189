"""Distillation of a draft model from a teacher's top entries: the loss of each row of student logits
and its gradient, in one pass over the logits each way. The reference does not train
(pagedbatch has no optimiser) and has no counterpart.

The teacher's record of a row is what ``top_logprobs`` returns for it: K log-probabilities and token
ids. Formulas and edge cases are stated at ``pb_distill_forward`` in ``include/pagedbatch_b200.h``.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .logprobs import check_temperature

__all__ = ["distill_loss"]

STATS = 32  # bytes of a row's statistics (pb_distill_stats_bytes)


class _Rows:
    """The arguments of one call: student rows, teacher entries, row weights."""

    __slots__ = ("z", "lp", "idx", "weight", "temperature", "args")

    def __init__(self, z, lp, idx, weight, temperature):
        self.z, self.lp, self.idx, self.weight, self.temperature = z, lp, idx, weight, temperature
        self.args = (z.data_ptr(), ops._DTYPE_CODE[z.dtype], z.shape[0], z.shape[1], z.stride(0), lp.data_ptr(),
                     lp.stride(0), idx.data_ptr(), idx.stride(0), idx.element_size(), idx.shape[1], temperature)

    def weight_ptr(self):
        return None if self.weight is None else self.weight.data_ptr()

    def forward(self, tail, total=False):
        """The rows' losses (or their sum) and statistics."""
        z = self.z
        n, V = z.shape
        L = _lib.load()
        n_ws = L.pb_distill_ws_bytes(n, V, self.args[1])
        # one buffer: statistics, losses, and the launch's own workspace
        keep = n * (STATS + 4)
        buf = torch.empty(-(-keep // 16) * 16 + n_ws, dtype=torch.uint8, device=z.device)
        loss = buf[n * STATS : keep].view(torch.float32)
        with ops.on_device(z.device):
            stream = torch.cuda.current_stream(z.device).cuda_stream
            base = buf.data_ptr()
            rc = L.pb_distill_forward(*self.args, int(tail), self.weight_ptr(), base + n * STATS, base,
                                      base + buf.numel() - n_ws, n_ws, stream)
            _lib.check(rc, "pb_distill_forward")
            if total:
                loss = torch.empty((), dtype=torch.float32, device=z.device)
                _lib.check(L.pb_distill_sum(base + n * STATS, n, loss.data_ptr(), stream), "pb_distill_sum")
        return loss, buf

    def backward(self, stats, grad_loss):
        z = self.z
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        with ops.on_device(z.device):
            rc = _lib.load().pb_distill_backward(
                *self.args, self.weight_ptr(), stats.data_ptr(), grad_loss.data_ptr(),
                grad_loss.stride(0) if grad_loss.dim() else 0, dz.data_ptr(),
                torch.cuda.current_stream(z.device).cuda_stream)
        _lib.check(rc, "pb_distill_backward")
        return dz


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, lp, idx, weight, temperature, tail, total):
        loss, stats = _Rows(z, lp, idx, weight, temperature).forward(tail, total)
        ctx.save_for_backward(z, lp, idx, weight, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        z, lp, idx, weight, stats = ctx.saved_tensors
        # a gradient of one value for all rows (from a sum or mean) is read through its stride of 0
        dz = _Rows(z, lp, idx, weight, ctx.temperature).backward(stats, grad_loss)
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
    z, lp, idx = student_logits, teacher_logprobs, teacher_indices
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
    for name, t in (("teacher_logprobs", lp), ("teacher_indices", idx), ("row_weight", row_weight)):
        if t is not None and t.device != z.device:
            raise ValueError(f"{name} must be on the logits' device {z.device}")
    if reduction not in ("none", "sum"):
        raise ValueError(f"reduction must be 'none' or 'sum', got {reduction!r}")
    t = check_temperature(temperature)
    lp = lp.float()
    if lp.stride(1) != 1:
        lp = lp.contiguous()
    if idx.stride(1) != 1:
        idx = idx.contiguous()
    if row_weight is not None:
        row_weight = row_weight.contiguous()
    total = reduction == "sum"
    if not (z.requires_grad and torch.is_grad_enabled()):
        return _Rows(z, lp, idx, row_weight, t).forward(tail, total)[0]
    return _Distill.apply(z, lp, idx, row_weight, t, bool(tail), total)
