"""Verification of drafted tokens: several tokens a step from one pass of the target model.

A draft model (or a lookup in the prompt) proposes a few tokens for each sequence, the target model
computes its logits at every drafted position in one forward pass, and ``verify`` accepts a prefix of
the drafts and draws one more token, so that the tokens are distributed exactly as the target's own
samples (``sample_tokens`` with the same ``SamplingParams``) are. The reference decodes one token a
step (pagedbatch/engine.py:130-171) and has no counterpart.

Layout: the sequences' rows follow one another; a sequence with ``d`` drafts owns ``d + 1`` rows, row
``j`` being the target's distribution at its ``j``-th draft and the last one that after all of them.
The rule, its arithmetic and the order of the draws are stated at ``pb_verify`` in
``include/pagedbatch_b200.h``.
"""

from __future__ import annotations

import functools
from collections.abc import Sequence

import numpy as np
import torch

from . import _lib, ops
from .sampling import _INVALID_DISTRIBUTION, pack_rows

__all__ = ["verify", "verify_tokens"]


def _kinds(params: torch.Tensor, noted: tuple[int, int] | None, vocab: int) -> int:
    """The kinds of sequences to launch for: those of the records (`noted`, or as the params tensor was uploaded,
    and then any other as well where it was written to since or may be before a replay of this call)."""
    known = noted is not None
    bits, kmax = noted if known else ops.noted_kinds(params)
    if not bits or kmax >= vocab:
        return 0  # (a top_k of the vocabulary or more is no filter: any kind)
    if known or (ops.unchanged(params) and not torch._C._cuda_isCurrentStreamCapturing()):
        return bits
    return bits | _lib.VERIFY_REST


def _check_dtype(name: str, t: torch.Tensor) -> None:
    if t.dtype not in ops._DTYPE_CODE:
        raise ValueError(f"unsupported {name} dtype {t.dtype}")


def _check_probs(draft_probs: torch.Tensor | None, n: int, vocab: int) -> None:
    if draft_probs is None:
        return
    if draft_probs.dim() != 2 or draft_probs.shape != (n, vocab) or (draft_probs.stride(1) != 1 and vocab > 1):
        raise ValueError(f"draft_probs must be [{n}, {vocab}] with a contiguous last dimension: a row per draft")
    _check_dtype("draft_probs", draft_probs)


def _check(logits, params, drafts, row_offsets, uniforms, draft_probs):
    """Refuses what the kernels do not take; rows, vocabulary, sequences and the device."""
    if not logits.is_cuda:
        raise ValueError("pagedbatch_b200.verify needs CUDA logits; move the tensor with .cuda() first")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be a [rows, vocab] tensor with a contiguous last dimension")
    _check_dtype("logits", logits)
    if params.dtype != torch.uint8 or params.numel() % _lib.ROW_PARAMS.itemsize or not params.is_contiguous():
        raise ValueError("params must be packed pb_row_params records (uint8), one per sequence")
    dev = logits.device
    R, V = logits.shape
    S = params.numel() // _lib.ROW_PARAMS.itemsize
    for name, t, dtype, n in (("drafts", drafts, torch.int64, R), ("row_offsets", row_offsets, torch.int32, S + 1),
                              ("uniforms", uniforms, torch.float64, R)):
        if t.dtype != dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on the logits' device {dev}")
    if params.device != dev or (draft_probs is not None and draft_probs.device != dev):
        raise ValueError(f"params and draft_probs must be on the logits' device {dev}")
    if S > R:
        raise ValueError(f"{S} sequences for {R} rows: every sequence has at least one row")
    _check_probs(draft_probs, R - S, V)
    if S == 0 and R:
        raise ValueError(f"{R} rows for no sequence")
    return R, V, S, dev


@functools.lru_cache(maxsize=256)
def _ws_bytes(rows: int, seqs: int, vocab: int, dtype: int, kinds: int) -> int:
    return _lib.load().pb_verify_ws_bytes(rows, seqs, vocab, dtype, kinds)


def _launch(logits, params, drafts, row_offsets, uniforms, draft_probs, noted=None):
    R, V, S, dev = _check(logits, params, drafts, row_offsets, uniforms, draft_probs)
    tokens = torch.empty(R, dtype=torch.int64, device=dev)
    accepted = torch.empty(S, dtype=torch.int32, device=dev)
    status = torch.empty(S, dtype=torch.int32, device=dev)
    if S == 0:
        return tokens, accepted, status
    L = _lib.load()
    code = ops._DTYPE_CODE[logits.dtype]
    with ops.on_device(dev):
        # a buffer of this call's own: the allocator hands it on in stream order, and a captured
        # graph keeps its copy
        kinds = _kinds(params, noted, V)
        n_ws = _ws_bytes(R, S, V, code, kinds)
        ws = torch.empty(n_ws, dtype=torch.uint8, device=dev)
        rc = L.pb_verify(
            logits.data_ptr(), code, R, V, logits.stride(0) if R > 1 else V, params.data_ptr(), S,
            row_offsets.data_ptr(), drafts.data_ptr(), uniforms.data_ptr(),
            draft_probs.data_ptr() if draft_probs is not None and R > S else None,
            ops._DTYPE_CODE[draft_probs.dtype] if draft_probs is not None else 0, R - S,
            draft_probs.stride(0) if draft_probs is not None and R - S > 1 else V, kinds,
            tokens.data_ptr(), accepted.data_ptr(), status.data_ptr(), ws.data_ptr(), n_ws, ops.raw_stream(dev))
    _lib.check(rc, "pb_verify")
    return tokens, accepted, status


@torch.library.custom_op("pagedbatch_b200::verify", mutates_args=())
def verify_op(logits: torch.Tensor, params: torch.Tensor, drafts: torch.Tensor, row_offsets: torch.Tensor,
              uniforms: torch.Tensor, draft_probs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Tokens and accepted counts."""
    tokens, accepted, _ = _launch(logits, params, drafts, row_offsets, uniforms, draft_probs)
    return tokens, accepted


@torch.library.custom_op("pagedbatch_b200::verify_with_status", mutates_args=())
def verify_with_status_op(
        logits: torch.Tensor, params: torch.Tensor, drafts: torch.Tensor, row_offsets: torch.Tensor, uniforms: torch.Tensor,
        draft_probs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Tokens, accepted counts and status codes."""
    return _launch(logits, params, drafts, row_offsets, uniforms, draft_probs)


@verify_op.register_fake
def _(logits, params, drafts, row_offsets, uniforms, draft_probs=None):
    _, _, s, _ = _check(logits, params, drafts, row_offsets, uniforms, draft_probs)
    return logits.new_empty((logits.shape[0],), dtype=torch.int64), logits.new_empty((s,), dtype=torch.int32)


@verify_with_status_op.register_fake
def _(logits, params, drafts, row_offsets, uniforms, draft_probs=None):
    _, _, s, _ = _check(logits, params, drafts, row_offsets, uniforms, draft_probs)
    return (logits.new_empty((logits.shape[0],), dtype=torch.int64), logits.new_empty((s,), dtype=torch.int32),
            logits.new_empty((s,), dtype=torch.int32))


def verify(logits: torch.Tensor, params: torch.Tensor, drafts: torch.Tensor, row_offsets: torch.Tensor,
           uniforms: torch.Tensor, draft_probs: torch.Tensor | None = None, with_status: bool = False):
    """Verify the drafts of ``S`` sequences against their ``R`` target rows, on the device and without
    a host read: ``(tokens int64[R], accepted int32[S])``.

    * ``logits [R, V]``: CUDA, float32 / bfloat16 / float16, last dim contiguous;
    * ``params``: one packed ``pb_row_params`` record per sequence (``ops.params_tensor``), which may be
      kept from step to step and written to in place, before the replay of a captured call as well (their
      ``uniform`` is not used). The launches are those for the kinds of sequences it was uploaded with;
      sequences of other kinds take the sampler's general kernel and are slower. Writes that torch does not
      count (through ``.data``, or a kernel of one's own) need a clone, which has no note of kinds;
    * ``drafts int64[R]``: the draft each row judges (ignored at a sequence's last row);
    * ``row_offsets int32[S + 1]``: sequence ``s`` owns rows ``row_offsets[s]`` to ``row_offsets[s + 1] - 1``;
      it starts at 0, ends at R and gives every sequence at least one row (not checked on the host);
    * ``uniforms float64[R]``: one random number in [0, 1) per row. It decides the row's draft; that of a
      sequence's last row draws the token after the accepted drafts;
    * ``draft_probs [R - S, V]``: the draft model's distribution at each draft, in row order (float32 /
      bfloat16 / float16), as ``ops.sample(..., with_probs=True)`` returns it. ``None``: the drafts are
      certain (looked up, or a greedy draft model).

    ``tokens`` holds, from each sequence's first row on, its accepted drafts and the token drawn after
    them, then -1. ``with_status`` adds ``int32[S]`` status codes (``PB_ROW_*``; where it is not 0 the
    drawn token is -1). Runs on the current stream of the logits' device and can be captured."""
    if ops.traced(logits):
        op = verify_with_status_op if with_status else verify_op
        return tuple(op(logits, params, drafts, row_offsets, uniforms, draft_probs))
    out = _launch(logits, params, drafts, row_offsets, uniforms, draft_probs)
    return out if with_status else out[:2]


def verify_tokens(logits: torch.Tensor, drafts: Sequence[Sequence[int]], params: Sequence,
                  generators: Sequence[torch.Generator], draft_probs: torch.Tensor | None = None) -> list[list[int]]:
    """The tokens of one verified step, per sequence: its accepted drafts and the one drawn after them.

    ``drafts[s]`` are sequence ``s``'s drafted token ids, ``params[s]`` its ``SamplingParams``;
    ``logits [R, V]`` holds ``len(drafts[s]) + 1`` rows for each sequence, one after another. A sequence that is
    not greedy takes ``len(drafts[s]) + 1`` float64 draws from its generator; a call that is refused takes none.
    CPU logits are copied to the current CUDA device first, as in ``sample_tokens``, and CPU ``draft_probs`` with
    them."""
    S = len(drafts)
    if len(params) != S or len(generators) != S:
        raise ValueError(f"{len(params)} params and {len(generators)} generators for {S} sequences")
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, vocab]")
    V = logits.shape[1]
    lens = np.array([len(d) for d in drafts], dtype=np.int64)
    offsets = np.zeros(S + 1, dtype=np.int32)
    np.cumsum(lens + 1, out=offsets[1:])
    R = int(offsets[-1])
    if logits.shape[0] != R:
        raise ValueError(f"{logits.shape[0]} logits rows for {R} (one per draft and one more per sequence)")
    flat = np.zeros(R, dtype=np.int64)
    for s, d in enumerate(drafts):
        flat[offsets[s] : offsets[s] + len(d)] = d
    if R and (flat.min() < 0 or flat.max() >= V):
        raise ValueError(f"drafts must be token ids in [0, {V})")
    rec = pack_rows(params, np.zeros(S))
    if S == 0:
        return []
    _check_dtype("logits", logits)
    _check_probs(draft_probs, R - S, V)
    if logits.is_cuda:
        dev = logits.device
    elif torch.cuda.is_available():
        dev = torch.device("cuda", torch.cuda.current_device())
    else:
        raise RuntimeError("pagedbatch_b200 verifies on a CUDA device and none is available")
    if draft_probs is not None and draft_probs.device != dev:
        if logits.is_cuda or draft_probs.is_cuda:
            raise ValueError(f"draft_probs must be on the logits' device {dev}")
        draft_probs = draft_probs.to(dev, non_blocking=draft_probs.is_pinned())
    logits = logits.to(dev, non_blocking=not logits.is_cuda and logits.is_pinned())
    uniforms = np.zeros(R)
    for s, (p, g) in enumerate(zip(params, generators, strict=True)):
        if p.temperature != 0:
            n = int(lens[s]) + 1
            uniforms[offsets[s] : offsets[s] + n] = torch.rand(n, dtype=torch.float64, generator=g).numpy()
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    # parameters, random numbers, drafts and offsets in one pinned buffer and one copy
    parts = [rec.view(np.uint8).reshape(-1), uniforms.view(np.uint8), flat.view(np.uint8), offsets.view(np.uint8)]
    ends = np.cumsum([p.size for p in parts])
    host = torch.empty(int(ends[-1]), dtype=torch.uint8, pin_memory=True)
    np.concatenate(parts, out=host.numpy())
    buf = host.to(dev, non_blocking=True)
    tokens, accepted, status = _launch(
        logits, buf[: ends[0]], buf[ends[1] : ends[2]].view(torch.int64), buf[ends[2] : ends[3]].view(torch.int32),
        buf[ends[0] : ends[1]].view(torch.float64), draft_probs, ops.row_kinds(rec))
    got, n_ok, st = tokens.tolist(), accepted.tolist(), status.tolist()
    for s, code in enumerate(st):
        if code == _lib.ROW_NONFINITE:
            raise RuntimeError(_INVALID_DISTRIBUTION)
        if code != _lib.ROW_OK:
            raise RuntimeError(f"verification failed on sequence {s} (status {code})")
    return [got[offsets[s] : offsets[s] + n_ok[s] + 1] for s in range(S)]
