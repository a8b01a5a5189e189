"""Corners of the verification's rule on a B200, against its restatement (oracle/verify.py), token for token."""

import numpy as np
import pytest
import torch

from pagedbatch_b200 import workloads
from test_verify_gpu import _check, _probs

pytestmark = pytest.mark.gpu


def _view(x, shift):
    """The rows on the device, `shift` elements past a 16-byte boundary."""
    buf = torch.zeros(len(x), (x.shape[1] + 31) // 16 * 16, dtype=x.dtype, device="cuda")
    view = buf[:, shift : shift + x.shape[1]]
    view.copy_(x)
    return view


def _rejected(x):
    """A draft per row that no parameters with a filter keep: the row's smallest value."""
    return x.float().argmin(1).numpy().astype(np.int64)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,spread", [(256, 3.0), (4096, 3.0), (4096, 0.0)])
def test_odd_values_at_some_of_the_kept_tokens(cuda, dtype, V, spread, shift):
    """NaN and negative draft probabilities take nothing of a token's weight, infinite ones all of it,
    whichever launch draws: few values near the kept ones, many equal ones (spread 0), rows of any alignment."""
    S, n = 48, 1
    g = torch.Generator().manual_seed(V)
    x = workloads.head_boosted(2 * S, V, seed=V, dtype=dtype)
    if not spread:
        x = torch.randint(-1, 2, (2 * S, V), generator=g).to(dtype)
        x[:, 0] = -3.0
    params = [((1.0, 0.7)[s % 2], (1.0, 0.95)[s // 2 % 2], (5, 20, 50, 128)[s // 4 % 4]) for s in range(S)]
    probs = _probs(x, [n] * S, params, 1)
    top = torch.topk(x[0::2].float(), 40, dim=1).indices
    for j, odd in enumerate((torch.nan, -torch.inf, -0.5, torch.inf, torch.nan)):
        at = top[:, torch.randperm(40, generator=g)[:8]]
        probs.scatter_(1, at, odd)
    probs[:, 0] = 0.1  # (the draft's own is an ordinary one where it is token 0)
    drafts = _rejected(x)
    for seed in range(4):
        u = np.random.default_rng(seed).random(2 * S)
        u[0::2] = 1.0 - 2.0**-53
        _check(x, params, [n] * S, drafts, u, probs, view=_view(x, shift))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low,high", [(-149, -126), (-128, -120), (-126, -100), (-60, -20)])
def test_cuts_next_to_zero(cuda, dtype, low, high, shift):
    """One ordinary value and the rest next to zero, where top-k or top-p cuts: x / T in one rounding decides
    which of them are kept, quotients below the normal numbers included."""
    S, V = 120, 4096
    g = torch.Generator().manual_seed(-low)
    e = torch.randint(low, high + 1, (S, V), generator=g).double()
    x = torch.ldexp(1.0 + torch.rand(S, V, generator=g, dtype=torch.float64), e)
    x *= torch.where(torch.rand(S, V, generator=g) < 0.5, -1.0, 1.0)
    x[1::3] = x[1::3, torch.randint(0, 40, (V,), generator=g)]  # rows of few values, many equal
    x[torch.arange(S), torch.randint(0, V, (S,), generator=g)] = 1.0
    x = x.to(dtype)
    for k, p in ((50, 1.0), (128, 0.7), (300, 1.0), (1500, 0.8), (0, 0.4), (0, 0.9)):
        params = [((0.7, 1.3, 3.0, 1.9999999)[s % 4], p, k) for s in range(S)]
        u = np.random.default_rng(k).random(S)
        _check(x, params, [0] * S, np.zeros(S, np.int64), u, view=_view(x, shift))


@pytest.mark.parametrize("temperature", [1.0, 2.0**-19, 2.0**-22, 1e-12])
def test_negative_shares_of_drafts_without_weight(cuda, temperature):
    """u D Z < P holds for a negative D whatever P is, however little is known of the mass before it is summed."""
    S, V = 8, 4099
    x = workloads.head_boosted(2 * S, V, seed=3)
    probs = torch.full((S, V), 1.0 / V)
    drafts = _rejected(x)
    probs[torch.arange(S), torch.from_numpy(drafts[0::2])] = torch.tensor([-0.5, -1e-30, 0.0, 0.5, -torch.inf, torch.nan, -1.0, 1e-30])
    for u in (0.0, 2.0**-53, 0.5, 1.0 - 2.0**-53):
        _check(x, [(temperature, 1.0, 0)] * S, [1] * S, drafts, np.full(2 * S, u), probs)


@pytest.mark.parametrize("V", [24, 704, 5003])
def test_negative_shares_of_drafts_cut_among_equals(cuda, V):
    """... a draft among the equals of the last kept value, where top-p cuts them, being one without weight."""
    S = 12
    x = torch.zeros(2 * S, V)
    x[:, ::3] = 1.0
    params = [(1.0, (0.3, 0.6)[s % 2], (0, 50, V - 1)[s % 3]) for s in range(S)]
    drafts = np.repeat(np.arange(S) * 3 % V, 2).astype(np.int64)
    drafts[0::4] = (V - 1) // 3 * 3  # the last of the equals
    probs = torch.full((S, V), 1.0 / V)
    probs[:, :] = torch.tensor([-1.0, -1e-30, 1e-30])[torch.arange(S) // 4, None]
    for u in (0.0, 0.25, 1.0 - 2.0**-53):
        _check(x, params, [1] * S, drafts, np.full(2 * S, u), probs)
