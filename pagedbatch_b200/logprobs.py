"""The largest log-probabilities of logits rows: what a server returns beside a token, and what a
teacher records for ``distill_loss``. The reference returns tokens only (pagedbatch/sampling.py:10-27)
and has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, ops

__all__ = ["top_logprobs", "TopLogprobs"]


class TopLogprobs(NamedTuple):
    """Per row: the k largest log-probabilities (float32), their token ids (int32), largest first
    (lowest id first on ties), and the row's log-sum-exp (float32): any other token's log-probability
    is its logit / temperature less that."""

    logprobs: torch.Tensor
    indices: torch.Tensor
    logsumexp: torch.Tensor


def check_temperature(temperature: float) -> float:
    t = float(temperature)
    if not 2.0**-20 <= t <= 2.0**20:
        raise ValueError(f"temperature must be in [2^-20, 2^20], got {temperature}")
    return t


def _check(logits: torch.Tensor, k: int, temperature: float) -> float:
    if not logits.is_cuda:
        raise ValueError("pagedbatch_b200.top_logprobs needs CUDA logits; move the tensor with .cuda() first")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be a [rows, vocab] tensor with a contiguous last dimension")
    if logits.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"unsupported logits dtype {logits.dtype}")
    n, V = logits.shape
    if not 1 <= k <= min(_lib.TOP_MAX, V):
        raise ValueError(f"k must be in [1, {min(_lib.TOP_MAX, V)}], got {k}")
    return check_temperature(temperature)


def _launch(logits: torch.Tensor, k: int, temperature: float):
    t = _check(logits, k, temperature)
    n, V = logits.shape
    dev = logits.device
    lp = torch.empty((n, k), dtype=torch.float32, device=dev)
    idx = torch.empty((n, k), dtype=torch.int32, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    L = _lib.load()
    with ops.on_device(dev):
        code = ops._DTYPE_CODE[logits.dtype]
        n_ws = L.pb_top_ws_bytes(n, V, code)
        ws = torch.empty(n_ws, dtype=torch.uint8, device=dev)
        rc = L.pb_top_logprobs(logits.data_ptr(), code, n, V, logits.stride(0), k, t, lp.data_ptr(), idx.data_ptr(),
                               lse.data_ptr(), ws.data_ptr(), n_ws, ops.raw_stream(dev))
    _lib.check(rc, "pb_top_logprobs")
    return lp, idx, lse


@torch.library.custom_op("pagedbatch_b200::top_logprobs", mutates_args=())
def top_logprobs_op(logits: torch.Tensor, k: int, temperature: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Log-probabilities, token ids and log-sum-exp."""
    return _launch(logits, k, temperature)


@top_logprobs_op.register_fake
def _(logits, k, temperature):
    _check(logits, k, temperature)
    n = logits.shape[0]
    return (logits.new_empty((n, k), dtype=torch.float32), logits.new_empty((n, k), dtype=torch.int32),
            logits.new_empty((n,), dtype=torch.float32))


def top_logprobs(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogprobs:
    """The ``k`` (at most 256) largest log-probabilities of ``softmax(logits / temperature)`` of every
    row of ``logits [n, V]`` (CUDA, float32 / bfloat16 / float16), on the current stream.
    Rows with NaN or +inf logits, or only -inf, have NaN log-probabilities. No gradient flows back."""
    launch = top_logprobs_op if ops.traced(logits) else _launch
    return TopLogprobs(*launch(logits.detach(), int(k), float(temperature)))
