"""The verification rule of ``pb_verify`` restated in whole numbers and single fp64 products, one
sequence at a time (see the rule in ``include/pagedbatch_b200.h``). Rows' kept sets come from the
sampling oracle."""

from __future__ import annotations

import ctypes
import math

import numpy as np

from . import kept_mask, lib, logits_as_numpy, make_params, sample, scaled_keys, to_f32


def weights(keys: np.ndarray, m: float) -> list[int]:
    keys = np.ascontiguousarray(keys, dtype=np.float32)
    q = np.zeros(keys.size, dtype=np.uint64)
    lib().pbo_weights(ctypes.c_void_p(keys.ctypes.data), keys.size, float(m), ctypes.c_void_p(q.ctypes.data))
    return q


def draw(w: np.ndarray, u53: int) -> int:
    """First index whose inclusive prefix exceeds floor(u53 * sum / 2^53)."""
    total = int(w.sum(dtype=object)) if w.size else 0
    t = (u53 * total) >> 53
    run = 0
    for i in np.flatnonzero(w).tolist():
        run += int(w[i])
        if run > t:
            return i
    return -1


def taken(d: np.ndarray, z: int) -> np.ndarray:
    """floor(fp64(d) * fp64(z)), 0 for d <= 0 or NaN, at most 2^64 - 1."""
    d = np.asarray(d, dtype=np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        t = np.where(d > 0, d * np.float64(z), 0.0)
    big = t >= 2.0**63
    return np.where(big, np.uint64(0xFFFFFFFFFFFFFFFF), np.where(big, 0, t).astype(np.uint64))


def verify(logits, params, lens, drafts, uniforms, draft_probs=None):
    """(tokens int64[R], accepted int32[S], status int32[S]). ``params``: (temperature, top_p, top_k)
    per sequence; ``drafts`` and ``uniforms`` per row; ``draft_probs`` [R - S, V] float32 or None."""
    raw, code = logits_as_numpy(logits)
    R, V = raw.shape
    x = to_f32(raw, code)
    S = len(lens)
    tokens = np.full(R, -1, dtype=np.int64)
    accepted, status = np.zeros(S, np.int32), np.zeros(S, np.int32)
    lo = 0
    for s, n in enumerate(lens):
        T, top_p, top_k = params[s]
        for j in range(n + 1):
            r = lo + j
            rec = make_params([T], [top_p], [top_k], [0.0])
            tok, info, _ = sample(raw.view(np.float16)[r : r + 1] if code == 2 else logits[r : r + 1], rec)
            last = j == n
            bad = int(info["status"][0])
            u = float(uniforms[r])
            if bad == 0 and T != 0 and not 0.0 <= u < 1.0:
                bad = 2
            if bad:
                status[s] = bad
                break
            d, u_draw = int(drafts[r]), float(uniforms[lo + n])
            if T == 0:
                if not last and d == int(tok[0]):
                    tokens[r] = d
                    accepted[s] += 1
                    continue
                tokens[r] = tok[0]
                break
            keys = scaled_keys(x[r], T)
            q = weights(keys, float(info["max_key"][0]))
            P = np.where(kept_mask(x[r], T, info[0]), q, np.uint64(0))
            Z = int(info["kept_q"][0])
            assert int(P.sum(dtype=object)) == Z
            if not last:
                px = int(P[d]) if 0 <= d < V else 0
                want = np.float64(u)
                row_d = None
                if draft_probs is not None:
                    row_d = np.asarray(draft_probs[r - s], dtype=np.float32)
                    want = want * np.float64(row_d[d] if 0 <= d < V else np.nan)
                if 0 <= d < V and want * np.float64(Z) < np.float64(px):
                    tokens[r] = d
                    accepted[s] += 1
                    continue
                if row_d is not None:
                    t = taken(row_d, Z)
                    w = np.where(P > t, P - t, np.uint64(0))
                else:
                    w = P.copy()
                    if 0 <= d < V:
                        w[d] = 0
            else:
                w = P
            if not w.any():
                w = P
            if 0.0 <= u_draw < 1.0:
                tokens[r] = draw(w, math.floor(u_draw * 2.0**53))
            else:
                status[s] = 2
            break
        lo += n + 1
    return tokens, accepted, status
