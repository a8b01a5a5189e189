"""Rows around the sizes at which they are cut into one segment more: 2048 vectors of 16 bytes, a vector and an
element on either side, from any alignment. Every operator of drafted decoding against its reference."""

import numpy as np
import pytest
import torch

from pagedbatch_b200 import workloads
from test_distill_gpu import check as check_distill
from test_distill_gpu import entries
from test_top_logprobs_gpu import check as check_top
from test_verify_gpu import KINDS, _check, _drafts, _probs

pytestmark = pytest.mark.gpu

SIZES = [(segments, by) for segments in (1, 2, 3) for by in (-1, 0, 1)]


def _view(x, shift):
    buf = torch.full((len(x), (x.shape[1] + 31) // 16 * 16), float("nan"), dtype=x.dtype, device="cuda")
    view = buf[:, shift : shift + x.shape[1]]
    view.copy_(x)
    return view


@pytest.mark.parametrize("segments,by", SIZES)
@pytest.mark.parametrize("dtype,shift", [(torch.float32, 0), (torch.float32, 3), (torch.bfloat16, 0), (torch.float16, 1)])
@pytest.mark.parametrize("part", ["vector", "element"])
def test_around_a_segment(cuda, segments, by, dtype, shift, part):
    epv = 16 // dtype.itemsize
    V = segments * 2048 * epv + by * (epv if part == "vector" else 1)
    x = workloads.head_boosted(6, V, seed=V, dtype=dtype)
    x[0::2, -1] = x.max()  # the ends of a row count
    x[1::2, 0] = x.max()
    view = _view(x, shift)
    check_top(x, 50, view=view)
    for tail in (False, True):
        lp, idx = entries(x, 12, V, 1.0)
        idx[:, 0] = torch.where(torch.arange(6) % 2 == 0, V - 1, 0).to(idx.dtype)
        check_distill(x, lp, idx, tail=tail, view=view)
    lens = [1, 1, 1]
    for kind in ("whole", "topk", "topp", "bigk"):
        params = [KINDS[kind](i) for i in range(3)]
        u = np.random.default_rng(V).random(6)
        _check(x, params, lens, _drafts(x, lens, V), u, _probs(x, lens, params, V), view=view)
