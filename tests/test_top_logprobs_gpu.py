"""The largest log-probabilities of a row on a B200: indices equal to the order of the values (ties by
index), log-probabilities and log-sum-exp within the rounding of their steps of the 64-bit ones."""

import numpy as np
import pytest
import torch

import pagedbatch_b200 as pb
from pagedbatch_b200 import workloads

pytestmark = pytest.mark.gpu

U = 2.0**-24  # half a step of fp32 relative to the value


def _order(x, k):
    """Indices of the k largest, value descending (NaN first), index ascending."""
    y = x.float().numpy().astype(np.float64)
    y = np.where(np.isnan(y), np.inf, y) + 0.0
    nan = x.float().isnan().numpy()
    idx = np.arange(y.shape[1])
    return np.stack([np.lexsort((idx, -y[r], ~nan[r]))[:k] for r in range(len(y))])


def check(x, k, temperature=1.0, view=None):
    lp, idx, lse = pb.top_logprobs(x.cuda() if view is None else view, k, temperature)
    want = _order(x, k)
    assert lp.dtype == lse.dtype == torch.float32 and idx.dtype == torch.int32
    assert np.array_equal(idx.cpu().numpy(), want)
    y = x.double().numpy() / float(np.float32(temperature))
    with np.errstate(all="ignore"):
        m = y.max(1, keepdims=True)
        s = np.exp(y - m)
        log_s = np.log(s.sum(1, keepdims=True))
        e_lse = m + log_s
        # the sum: at most 2^20 terms in at most ~600 sequential additions a thread, each term within two
        # units and the rounding of its exponent (3 U of |y - m|, weighted by the term itself); the
        # rest is a handful of products
        spread = (np.where(s > 0, s * np.nan_to_num(m - y, posinf=0.0), 0)).sum(1, keepdims=True) / s.sum(1, keepdims=True)
        lim = U * (640 + 3 * spread)
        # (the difference from the maximum first: at the lowest value even 64 bits lose log_s beside it)
        e_lp = (np.take_along_axis(y, want, 1) - m) - log_s
        ok = np.isfinite(e_lp)
        got = lp.cpu().numpy().astype(np.float64)
        finite = np.isfinite(e_lse[:, 0])
        assert np.array_equal(np.isnan(got), np.broadcast_to(~finite[:, None], got.shape))
        assert np.array_equal(got == -np.inf, e_lp == -np.inf)
        assert (np.abs(got - e_lp)[ok] <= (lim + 6 * U * np.abs(e_lp))[ok]).all(), np.abs(got - e_lp)[ok].max()
        g_lse = lse.cpu().numpy().astype(np.float64)
        d = np.abs(g_lse - e_lse[:, 0])[finite]
        assert (d <= (lim[:, 0] + 4 * U * (np.abs(e_lse) + np.abs(m))[:, 0])[finite]).all(), d.max()
        assert np.isnan(g_lse[~finite]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,k", [(1, 1), (2, 2), (7, 3), (8, 8), (33, 20), (255, 255), (300, 256), (1000, 1), (4099, 128),
                                 (50021, 7), (128256, 256)])
def test_sizes(cuda, dtype, V, k):
    for n in (1, 5, 40):
        check(workloads.head_boosted(n, V, seed=V + n, dtype=dtype), k, 1.0 if n != 5 else 0.7)


@pytest.mark.parametrize("n", [150, 700])
def test_many_rows(cuda, n):
    check(workloads.head_boosted(n, 4099, seed=n, dtype=torch.bfloat16), 50)


def test_large_vocabulary(cuda):
    x = torch.randn(2, 1_500_007, generator=torch.Generator().manual_seed(0))
    for k in (1, 256):
        check(x, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties(cuda, dtype):
    """Rows of few distinct values: long runs of equals at the k-th place, more than any list holds."""
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.integers(0, 3, (6, 20011)).astype(np.float32)).to(dtype)
    x[1] = 0.25                       # one value
    x[2, :] = -0.0
    x[2, ::3] = 0.0                   # the two zeros are equal
    x[3] = torch.arange(20011).float().to(dtype)
    x[4] = -torch.arange(20011).float().to(dtype)
    for k in (1, 5, 200, 256):
        check(x, k)


def test_masked_rows(cuda):
    V = 5003
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = workloads.head_boosted(10, V, seed=1, dtype=dtype)
        low = torch.finfo(dtype).min
        x[0, 10:] = -torch.inf        # fewer values than k
        x[1, :] = -torch.inf          # nothing left
        x[2, :] = low                 # masked with the lowest value: still a uniform row
        x[3, 1:] = low
        x[4, 100] = torch.nan
        x[5, 100], x[5, 50] = torch.inf, torch.nan
        x[6, 7] = torch.inf
        x[7, ::2] = -torch.inf
        x[8, 5:] = low
        x[9, :-1] = -torch.inf
        check(x, 64)
        check(x, 64, 2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,shift", [(50021, 0), (50021, 3), (600, 1)])
def test_few_allowed_tokens(cuda, dtype, V, shift):
    """Rows of which a mask (-inf, the type's lowest value, any value) leaves a few tokens, fewer or more
    than k: the lowest ids of the masked ones follow them."""
    g = torch.Generator().manual_seed(V)
    low = (-torch.inf, torch.finfo(dtype).min, -30.0)
    left = (0, 1, 5, 30, 255, 300)
    x = torch.empty(len(low) * len(left), V, dtype=dtype)
    for r in range(len(x)):
        n = left[r % len(left)]
        x[r] = low[r // len(left)]
        x[r, torch.randperm(V, generator=g)[:n]] = torch.randn(n, generator=g).to(dtype)
    x[4, -1] = 1.0  # the row's last token
    buf = torch.zeros(len(x), V + 8, dtype=dtype, device="cuda")
    view = buf[:, shift : shift + V]
    view.copy_(x)
    for k in (1, 20, 50, 256):
        check(x, k, view=view)


def test_strides(cuda):
    V = 1003
    for dtype in (torch.float32, torch.float16):
        x = workloads.head_boosted(9, V, seed=3, dtype=dtype)
        for shift, stride in ((1, 1009), (3, 1011), (0, 1024), (5, V)):
            buf = torch.full((9 * stride + 16,), float("nan"), dtype=dtype, device="cuda")
            view = buf[shift:].as_strided((9, V), (stride, 1))
            view.copy_(x)
            check(x, 33, view=view)
        check(x[:1].expand(4, V), 33, view=x[:1].cuda().expand(4, V))
    big = torch.empty((1 << 31) + 16 + V, dtype=torch.bfloat16, device="cuda")
    x = workloads.head_boosted(3, V, seed=4, dtype=torch.bfloat16)
    view = big.as_strided((3, V), ((1 << 30) + 3, 1))
    view.copy_(x)
    check(x, 50, view=view)


def test_temperatures(cuda):
    x = workloads.head_boosted(4, 4099, seed=5)
    for t in (2.0**-20, 0.01, 0.5, 3.0, 2.0**20):
        check(x, 16, t)


def test_streams_graph_and_op(cuda):
    x = [workloads.head_boosted(30, 4099, seed=s).cuda() for s in (1, 2)]
    want = [pb.top_logprobs(v, 20) for v in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.ops.pagedbatch_b200.top_logprobs(x[0], 20, 1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pb.top_logprobs(v, 20)
        graphs.append((g, out))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    assert pb.top_logprobs(x[0][:0], 5).logprobs.shape == (0, 5)


def test_agrees_with_the_sampler(cuda):
    """The greedy token is the first index, and a token's log-probability its sampled probability's."""
    from pagedbatch_b200 import ops

    x = workloads.head_boosted(16, 4099, seed=6).cuda()
    rec = ops.pack_params([0.7] * 16, [1.0] * 16, [0] * 16, np.zeros(16))
    _, _, probs = ops.sample(x, ops.params_tensor(rec, x.device), None, with_probs=True)
    top = pb.top_logprobs(x, 10, 0.7)
    assert torch.equal(top.indices[:, 0].long(), x.argmax(1))
    assert torch.allclose(top.logprobs.exp(), probs.gather(1, top.indices.long()), rtol=1e-4, atol=0)
