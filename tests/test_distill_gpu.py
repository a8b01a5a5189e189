"""The distillation loss and its gradient on a B200 against the formulas in 64 bits, and the gradient
against differences of the 64-bit loss."""

import numpy as np
import pytest
import torch

import pagedbatch_b200 as pb
from pagedbatch_b200 import workloads

pytestmark = pytest.mark.gpu

U = 2.0**-24  # half a step of fp32 relative to the value


def formula(z, lp, idx, temperature=1.0, tail=False, weight=None):
    """Loss [n], gradient [n, V] of the summed loss, and the parts of the error bounds, in 64 bits."""
    tau = float(np.float32(temperature))
    y = z.double() / tau
    n, V = y.shape
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    loss, grad = torch.zeros(n, dtype=torch.float64), torch.zeros_like(y)
    l_err, g_err = torch.zeros(n, dtype=torch.float64), torch.zeros_like(y)
    for r in range(n):
        used = idx[r] >= 0
        ent, val = idx[r][used].long(), lp[r][used].double()
        if not len(ent) or (not tail and bool((val == -torch.inf).all())) or w[r] == 0:
            continue
        t = val.exp() if tail else torch.softmax(val, 0)
        logs = torch.log_softmax(y[r], 0)
        s = logs.exp()
        target = torch.zeros(V, dtype=torch.float64).index_add_(0, ent, t)
        out = torch.ones(V, dtype=torch.bool)
        out[ent] = False
        T, S = 0.0, float(s[out].sum())
        if tail and S > 0:
            T = max(0.0, 1.0 - float(t.sum()))
        pos = t > 0
        logt = torch.log(t[pos]) if tail else torch.log_softmax(val, 0)[pos]
        loss[r] = (t[pos] * (logt - logs[ent][pos])).sum()
        A = float(t.sum()) + T
        K = len(ent)
        grad[r] = A * s - target
        arg = torch.nan_to_num((y[r].max() - y[r]), posinf=0.0)
        lse_err = U * (640 + 3 * float((s * arg).sum()))  # see the top log-probabilities' bound
        l_err[r] = (t[pos] * (lse_err + U * 12 * (logt.abs() + logs[ent][pos].abs() + K))).sum()
        g_err[r] = A * s * (lse_err + 8 * U * (1 + arg) + 4 * U * K) + U * (2 * K + 24) * target
        g_err[r].index_add_(0, ent, t * U * 4 * torch.nan_to_num(val.abs(), posinf=0.0))
        if T > 0:
            logS = float(torch.logsumexp(logs[out], 0))
            loss[r] += T * (np.log(T) - logS)
            T_err = U * (K + 8) * (1 + float((t * val.abs()).nan_to_num().sum()))
            l_err[r] += T * (2 * lse_err + U * 8 * (abs(np.log(T)) + abs(logS))) + T_err * (abs(np.log(T)) + abs(logS) + 1)
            st = torch.where(out, (logs - logS).exp(), 0.0)
            grad[r] -= T * st
            g_err[r] += st * (T * (2 * lse_err + 8 * U * (1 + arg)) + T_err + A * S * (2 * lse_err + 8 * U * (1 + abs(logS)))) + T_err * s
        loss[r] *= w[r]
        l_err[r] = l_err[r] * w[r].abs() + 4 * U * loss[r].abs()
        grad[r] *= w[r] / tau
        g_err[r] = g_err[r] * (w[r] / tau).abs() + 4 * U * grad[r].abs()
    return loss, grad, l_err, g_err


def check(z, lp, idx, temperature=1.0, tail=False, weight=None, reduction="none", view=None, grad_out=None):
    loss64, grad64, l_err, g_err = formula(z, lp, idx, temperature, tail, weight)
    dev = (z.cuda() if view is None else view).detach().requires_grad_()
    loss = pb.distill_loss(dev, lp.cuda(), idx.cuda(), temperature=temperature, tail=tail, reduction=reduction,
                           row_weight=None if weight is None else weight.cuda())
    if reduction == "sum":
        assert loss.shape == ()
        assert abs(loss.item() - float(loss64.sum())) <= float(l_err.sum()) + U * len(z) * float(loss64.abs().sum())
        go = torch.ones(len(z), dtype=torch.float64)
        loss.backward()
    else:
        assert loss.shape == (len(z),) and loss.dtype == torch.float32
        got = loss.detach().cpu().double()
        assert ((got - loss64).abs() <= l_err).all(), ((got - loss64).abs() - l_err).max()
        go = torch.linspace(0.5, 1.5, len(z)).double() if grad_out is None else grad_out.double()
        loss.backward(go.float().cuda())
        go = go.float().double()
    g = dev.grad
    assert g.dtype == z.dtype and g.shape == z.shape
    want, lim = grad64 * go[:, None], g_err * go.abs()[:, None]
    eps = torch.finfo(z.dtype)
    lim = lim + (eps.eps / 2) * want.abs() * 1.01 + eps.smallest_normal * eps.eps  # one rounding to the type
    d = (g.cpu().double() - want).abs()
    assert (d <= lim).all(), (d - lim).max()
    return loss, g


def entries(z, K, seed, temperature=1.0, short=True):
    """A teacher's record: its top K of noisy logits, some rows shorter, one row without entries."""
    g = torch.Generator().manual_seed(seed)
    y = z.float().clamp(min=-1e4) / temperature + torch.randn(z.shape, generator=g)
    top = torch.topk(y, K, dim=1)
    lp, idx = top.values - torch.logsumexp(y, 1, keepdim=True), top.indices.to(torch.int32)
    if short and len(z) > 2:
        idx[0, K // 2 :] = -1
        idx[2] = -1
    return lp, idx


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (1, 2, 1), (3, 7, 7), (4, 33, 5), (5, 1000, 20), (3, 4099, 1024),
                                   (7, 50021, 33), (2, 128256, 64)])
def test_formula(cuda, tail, dtype, n, V, K):
    z = workloads.head_boosted(n, V, seed=V, dtype=dtype)
    lp, idx = entries(z, K, V)
    check(z, lp, idx, tail=tail)
    check(z, lp, idx.long(), tail=tail, temperature=2.0, weight=torch.linspace(0.0, 2.0, n), reduction="sum")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,V", [(torch.float32, 131003), (torch.float32, 131063), (torch.float32, 300007),
                                     (torch.bfloat16, 600011), (torch.float16, 1 << 20)])
def test_long_rows(cuda, tail, dtype, V):
    """Rows at and beyond what a cluster holds in shared memory."""
    z = torch.randn(2, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    lp, idx = entries(z, 40, 1)
    check(z, lp, idx, tail=tail)
    check(z, lp, idx, tail=tail, reduction="sum")


@pytest.mark.parametrize("tail", [False, True])
def test_many_rows(cuda, tail):
    z = workloads.head_boosted(700, 1000, seed=1, dtype=torch.bfloat16)
    lp, idx = entries(z, 16, 2)
    check(z, lp, idx, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,V,K", [(torch.float32, 1, 1), (torch.float32, 7, 3), (torch.float16, 1003, 40),
                                       (torch.bfloat16, 4096, 1000), (torch.float32, 50021, 33), (torch.float32, 65533, 20),
                                       (torch.bfloat16, 128256, 64), (torch.float16, 131057, 64)])
def test_sums_of_many_rows(cuda, tail, dtype, V, K):
    """A sum over more rows than the device has SMs, with rows that do not count and entries that repeat;
    then scaled, and once more."""
    n = 150 if V > 20000 else 333
    z = torch.randn(n, V, generator=torch.Generator().manual_seed(V)).to(dtype) * 2
    lp, idx = entries(z, K, 1)
    if K > 4:
        idx[5:9, 2:4] = idx[5:9, :1]
        idx[10, ::3] = idx[10, 1]
    w = torch.rand(n, generator=torch.Generator().manual_seed(1)) + 0.25
    w[3], w[149] = 0.0, 0.0
    z[3, 0] = torch.nan
    z[n - 1, V // 2] = -torch.inf if V > 1 else 0.0
    loss64, grad64, l_err, g_err = formula(z, lp, idx, 1.25, tail, w)
    dev = z.cuda().requires_grad_()
    loss = pb.distill_loss(dev, lp.cuda(), idx.cuda(), temperature=1.25, tail=tail, row_weight=w.cuda(), reduction="sum")
    if torch.isinf(loss64).any():  # (the masked logit was an entry's)
        assert loss.item() == float("inf")
    else:
        assert abs(loss.item() - float(loss64.sum())) <= float(l_err.sum()) + U * n * float(loss64.abs().sum())
    f = torch.finfo(dtype)
    for scale in (1.0, 1.0, 0.375, 0.0):
        (g,) = torch.autograd.grad(loss * scale, dev, retain_graph=True)
        want = grad64 * scale
        lim = g_err * scale + (f.eps / 2) * want.abs() * 1.01 + f.smallest_normal * f.eps
        d = (g.cpu().double() - want).abs()
        assert (d <= lim).all(), (scale, (d - lim).max(), (d > lim).nonzero()[:4])


@pytest.mark.parametrize("tail", [False, True])
def test_gradient_against_differences(cuda, tail):
    z = workloads.head_boosted(3, 500, seed=3).double().float()
    lp, idx = entries(z, 12, 4, short=False)
    dev = z.cuda().requires_grad_()
    pb.distill_loss(dev, lp.cuda(), idx.cuda(), tail=tail, temperature=1.5, reduction="sum").backward()
    g = torch.Generator().manual_seed(0)
    _, _, _, g_err = formula(z, lp, idx, 1.5, tail)
    for _ in range(10):
        v = torch.randn(z.shape, generator=g, dtype=torch.float64)
        h = 1e-5  # central differences: h^2 times the third derivative (below 1 here), and 1e-16 / h
        a = formula(z.double() + h * v, lp, idx, 1.5, tail)[0].sum()
        b = formula(z.double() - h * v, lp, idx, 1.5, tail)[0].sum()
        slope = (a - b) / (2 * h)
        mine = (dev.grad.cpu().double() * v).sum()
        assert abs(slope - mine) <= (g_err * v.abs()).sum() + 1e-8 * v.abs().pow(3).sum() + 1e-9


@pytest.mark.parametrize("tail", [False, True])
def test_repeated_entries_add_up(cuda, tail):
    z = workloads.head_boosted(4, 1000, seed=5)
    lp, idx = entries(z, 30, 6, short=False)
    idx[:, 5:9] = idx[:, 3:4]
    idx[1] = idx[1, 0]
    lp = lp - 2.0
    check(z, lp, idx, tail=tail)


@pytest.mark.parametrize("tail", [False, True])
def test_masks(cuda, tail):
    """Logits masked with -inf and the lowest value, entries of no weight, entries that are the row."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        low = torch.finfo(dtype).min
        z = workloads.head_boosted(8, 300, seed=7, dtype=dtype)
        lp, idx = entries(z, 6, 8, short=False)
        keep = torch.zeros(8, 300, dtype=torch.bool).scatter_(1, idx.long(), True)
        z[0, ~keep[0]] = -torch.inf          # nothing outside the entries
        z[1, ~keep[1]] = low
        z[2] = low                           # a uniform row
        z[3, ::2] = torch.where(keep[3, ::2], z[3, ::2], -torch.inf)
        lp[4] = -torch.inf                   # no weight at all
        lp[5, 2:] = -torch.inf
        lp[6] += 3.0 if not tail else 0.0    # any constant may be added to the renormalised values
        z[7, idx[7, 0]] = z[7].max() + 20    # a student that is sure
        check(z, lp, idx, tail=tail)
    z = workloads.head_boosted(2, 40, seed=9)
    idx = torch.stack([torch.randperm(40, generator=torch.Generator().manual_seed(i)) for i in (0, 1)]).int()
    lp = torch.log_softmax(torch.randn(2, 40, generator=torch.Generator().manual_seed(2)), 1)
    check(z, lp, idx, tail=tail)             # the entries are the whole vocabulary


def test_an_entry_the_student_excludes(cuda):
    """-inf at an entry of weight: the loss is infinite, the gradient finite and by the formula."""
    z = workloads.head_boosted(2, 100, seed=1)
    lp, idx = entries(z, 4, 2, short=False)
    z[0, idx[0, 1]] = -torch.inf
    dev = z.cuda().requires_grad_()
    loss = pb.distill_loss(dev, lp.cuda(), idx.cuda())
    assert loss[0] == torch.inf and torch.isfinite(loss[1])
    loss[0].backward()
    t = torch.softmax(lp[0].double(), 0)
    want = torch.softmax(z[0].double(), 0).index_add(0, idx[0].long(), -t)
    assert (dev.grad[0].cpu().double() - want).abs().max() < 1e-6 and (dev.grad[1] == 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_rows_that_do_not_count(cuda, tail):
    """Padded rows and rows of weight 0 hold anything; a row of gradient 0 has gradient 0."""
    z = workloads.head_boosted(5, 1000, seed=1)
    lp, idx = entries(z, 8, 2, short=False)
    idx[0] = -1
    z[0] = torch.nan
    z[1] = -torch.inf
    w = torch.tensor([1.0, 0.0, 1.0, 1.0, 1.0])
    z[2, 5] = torch.nan
    idx[3, 2] = 1000          # out of range
    dev = z.cuda().requires_grad_()
    loss = pb.distill_loss(dev, lp.cuda(), idx.cuda(), tail=tail, row_weight=w.cuda())
    got = loss.detach().cpu()
    assert got[0] == 0 and got[1] == 0 and got[2].isnan() and got[3].isnan() and got[4].isfinite()
    loss.backward(torch.tensor([1.0, 1.0, 0.0, 1.0, 1.0]).cuda())
    assert (dev.grad[:3] == 0).all() and dev.grad[3].isnan().all() and dev.grad[4].isfinite().all()
    bad = idx.clone()
    bad[4, 0] = -2
    assert pb.distill_loss(dev, lp.cuda(), bad.cuda(), tail=tail)[4].isnan()
    big = idx.long()
    big[4, 0] = 1 << 40
    assert pb.distill_loss(dev, lp.cuda(), big.cuda(), tail=tail)[4].isnan()
    for i in (0, 300):  # a NaN of the teacher's, alone in its warp or not
        wide_lp, wide = torch.full((1, 400), torch.nan), torch.full((1, 400), -1)
        wide_lp[0, :2], wide[0, :2], wide[0, i] = -1.0, torch.tensor([3, 4]), 7
        wide_lp[0, i] = torch.nan
        assert pb.distill_loss(z[4:].cuda(), wide_lp.cuda(), wide.cuda(), tail=tail).isnan().all()
    z[:] = 1.0
    z[0], z[1] = torch.nan, -torch.inf
    nothing = pb.distill_loss(z[1:2].cuda(), lp[1:2].cuda(), idx[1:2].cuda(), tail=tail)
    assert nothing.isnan().all()  # a row that counts but holds nothing above -inf


def test_strides_and_shared_rows(cuda):
    V, n, K = 1003, 6, 9
    for dtype in (torch.float32, torch.float16):
        z = workloads.head_boosted(n, V, seed=3, dtype=dtype)
        lp, idx = entries(z, K, 4)
        for shift, stride in ((1, 1009), (3, 1011), (0, 1024), (5, V)):
            buf = torch.full((n * stride + 16,), float("nan"), dtype=dtype, device="cuda")
            view = buf[shift:].as_strided((n, V), (stride, 1))
            view.copy_(z)
            check(z, lp, idx, tail=True, view=view)
        # one student row for all teachers: the gradients of its uses add up
        one = z[:1].cuda().requires_grad_()
        pb.distill_loss(one.expand(n, V), lp.cuda(), idx.cuda(), reduction="sum").backward()
        _, g64, _, g_err = formula(z[:1].expand(n, V), lp, idx)
        # n gradients and their sum, each rounded once to the type: by at most eps / 2 of the value, or
        # (a subnormal) half the smallest step, smallest_normal * eps / 2 (fp16: 2^-25, 7 of them 2.1e-7)
        f = torch.finfo(dtype)
        lim = g_err.sum(0) + f.eps * g64.abs().sum(0) + (n + 1) * f.smallest_normal * f.eps / 2
        assert ((one.grad[0].cpu().double() - g64.sum(0)).abs() <= lim).all()
        # the entries strided, and one record for all rows
        wide_lp, wide_idx = torch.zeros(n, 2 * K).cuda(), torch.zeros(n, 2 * K, dtype=torch.int32).cuda()
        wide_lp[:, ::2], wide_idx[:, ::2] = lp.cuda(), idx.cuda()
        a = pb.distill_loss(z.cuda(), wide_lp[:, ::2], wide_idx[:, ::2], tail=True)
        assert torch.equal(a, pb.distill_loss(z.cuda(), lp.cuda(), idx.cuda(), tail=True))
        a = pb.distill_loss(z.cuda(), lp[1:2].cuda().expand(n, K), idx[1:2].cuda().expand(n, K))
        assert torch.equal(a, pb.distill_loss(z.cuda(), lp[1:2].cuda().repeat(n, 1), idx[1:2].cuda().repeat(n, 1)))
    big = torch.empty((1 << 31) + 16 + V, dtype=torch.bfloat16, device="cuda")
    z = workloads.head_boosted(3, V, seed=4, dtype=torch.bfloat16)
    view = big.as_strided((3, V), ((1 << 30) + 3, 1))
    view.copy_(z)
    lp, idx = entries(z, K, 5)
    loss = pb.distill_loss(view, lp.cuda(), idx.cuda(), tail=True)
    assert torch.equal(loss, pb.distill_loss(z.cuda(), lp.cuda(), idx.cuda(), tail=True))


def test_types_of_the_record(cuda):
    z = workloads.head_boosted(4, 500, seed=1)
    lp, idx = entries(z, 8, 2)
    for dtype in (torch.bfloat16, torch.float16):
        check(z, lp.to(dtype).float(), idx)
        a = pb.distill_loss(z.cuda(), lp.to(dtype).cuda(), idx.long().cuda())
        assert torch.equal(a, pb.distill_loss(z.cuda(), lp.to(dtype).float().cuda(), idx.cuda()))


def test_differentiates_once(cuda):
    z = torch.randn(4, 100, device="cuda", requires_grad=True)
    lp, idx = entries(z.detach().cpu(), 5, 1)
    loss = pb.distill_loss(z, lp.cuda(), idx.cuda(), reduction="sum")
    (g,) = torch.autograd.grad(loss, z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeated_entries_give_the_same_bits(cuda, dtype):
    """However the threads meet at an element that several entries name."""
    n, V, K = 64, 1000, 1024
    g = torch.Generator().manual_seed(9)
    z = (3 * torch.randn(n, V, generator=g)).to(dtype).cuda()
    idx = torch.randint(0, 300, (n, K), generator=g).cuda()
    lp = (torch.randn(n, K, generator=g) - 9).cuda()
    want = None
    for _ in range(10):
        x = z.detach().requires_grad_()
        loss = pb.distill_loss(x, lp, idx, tail=True)
        loss.sum().backward()
        got = (loss.detach(), x.grad)
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradient_scale_and_repeats(cuda):
    """Scaled, zero and repeated backward passes, and the same bits each time."""
    z = workloads.head_boosted(40, 4099, seed=1, dtype=torch.bfloat16).cuda().requires_grad_()
    lp, idx = (t.cuda() for t in entries(z.detach().cpu(), 10, 2))
    for reduction in ("none", "sum"):
        loss = pb.distill_loss(z, lp, idx, tail=True, reduction=reduction)
        total = loss.sum()
        (a,) = torch.autograd.grad(total, z, retain_graph=True)
        (b,) = torch.autograd.grad(total, z, retain_graph=True)
        assert torch.equal(a, b)
        (c,) = torch.autograd.grad(total * 4.0, z, retain_graph=True)
        assert torch.equal(c.float(), a.float() * 4.0)
        (d,) = torch.autograd.grad(total * 0.0, z)
        assert (d == 0).all()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(total, z)
    with torch.no_grad():
        assert not pb.distill_loss(z, lp, idx).requires_grad
    assert pb.distill_loss(z[:0], lp[:0], idx[:0]).shape == (0,)


def test_streams_and_graph(cuda):
    """Another stream, and a training step captured and replayed on new logits in place."""
    zs = [workloads.head_boosted(20, 4099, seed=s, dtype=torch.bfloat16).cuda() for s in (1, 2)]
    lp, idx = (t.cuda() for t in entries(zs[0].cpu(), 10, 2))

    def step(z):
        x = z.detach().requires_grad_()
        loss = pb.distill_loss(x, lp, idx, tail=True, reduction="sum")
        (g,) = torch.autograd.grad(loss, x)
        return loss.detach(), g

    want = [step(z) for z in zs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(zs[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    buf = zs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(buf)
    for z, w in zip(zs * 2, want * 2):
        buf.copy_(z)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))
