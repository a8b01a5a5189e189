"""The operators of drafted decoding in recorded calls (make_fx, torch.compile), on fake tensors and under forward
mode: a recorded call computes what the call does, on other inputs as well, and what has no derivative says so."""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import pagedbatch_b200 as pb
from pagedbatch_b200 import workloads
from test_verify_gpu import KINDS, _drafts, _lens, _offsets, _params, _probs

pytestmark = pytest.mark.gpu

S, V = 7, 1003
LENS = _lens(S, 3, 1)
R = sum(LENS) + S


def _verify_inputs(seed):
    x = workloads.head_boosted(R, V, seed=seed)
    params = [KINDS["mixed"](i) for i in range(S)]
    return (x.cuda(), _params(params), torch.from_numpy(_drafts(x, LENS, seed)).cuda(), _offsets(LENS),
            torch.from_numpy(np.random.default_rng(seed).random(R)).cuda(), _probs(x, LENS, params, seed).cuda())


def _distill_inputs(seed):
    z = workloads.head_boosted(9, V, seed=seed).cuda()
    y = workloads.head_boosted(9, V, seed=seed + 10).cuda()
    lp, idx, _ = pb.top_logprobs(y, 12)
    return z, lp, idx, torch.rand(9, generator=torch.Generator().manual_seed(seed)).cuda()


def _step(tail, reduction):
    def step(z, lp, idx, w):
        z = z.detach().requires_grad_()
        loss = pb.distill_loss(z, lp, idx, tail=tail, row_weight=w, reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss.sum(), z)[0]

    return step


def _loss(z, lp, idx, w):
    return pb.distill_loss(z, lp, idx, row_weight=w)


CALLS = {
    "verify": (lambda *a: pb.verify(*a), _verify_inputs),
    "verify, status": (lambda *a: pb.verify(*a, with_status=True), _verify_inputs),
    "top": (lambda x: tuple(pb.top_logprobs(x, 20, temperature=0.7)), lambda seed: _verify_inputs(seed)[:1]),
    "loss": (lambda *a: (_loss(*a),), _distill_inputs),
    "step": (_step(False, "none"), _distill_inputs),
    "step, tail, sum": (_step(True, "sum"), _distill_inputs),
}


@pytest.mark.parametrize("name,mode", [(name, mode) for name in CALLS for mode in ("real", "fake", "compile")
                                       if mode != "compile" or "step" not in name])
def test_recorded_calls(cuda, name, mode):
    call, inputs = CALLS[name]
    if mode == "compile":
        recorded = torch.compile(call, fullgraph=True, backend="aot_eager")
    else:
        recorded = make_fx(call, tracing_mode=mode)(*inputs(1))
    for seed in (1, 2, 3):
        args = inputs(seed)
        got, want = recorded(*args), call(*args)
        assert len(got) == len(want)
        for a, b in zip(got, want, strict=True):
            assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("tail", [False, True])
def test_compiled_training_step(cuda, tail):
    """The gradient through a compiled loss is the one of the loss itself."""
    def loss(table, rows, lp, idx, w):
        return pb.distill_loss(table[rows], lp, idx, tail=tail, row_weight=w, reduction="sum") * 0.5

    compiled = torch.compile(loss, fullgraph=True, backend="aot_eager")
    for seed in (1, 2):
        z, lp, idx, w = _distill_inputs(seed)
        rows = torch.tensor([3, 1, 4, 1, 5, 0, 2, 6, 5], device="cuda")
        a, b = (z.clone().requires_grad_() for _ in range(2))
        la, lb = loss(a, rows, lp, idx, w), compiled(b, rows, lp, idx, w)
        la.backward()
        lb.backward()
        assert torch.equal(la, lb) and torch.equal(a.grad, b.grad) and a.grad.abs().sum() > 0


def test_fake_gradient(cuda):
    with FakeTensorMode():
        z = torch.empty(5, 100, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        lp, idx, _ = pb.top_logprobs(z, 7)
        (grad,) = torch.autograd.grad(pb.distill_loss(z, lp, idx, reduction="sum"), z)
        assert grad.shape == z.shape and grad.dtype == z.dtype


def test_forward_mode_is_refused(cuda):
    """No tangent is lost without a word, in the logits or in the teacher's record."""
    args = _distill_inputs(1)
    with fwAD.dual_level():
        for at in (0, 1, 3):
            a = list(args)
            a[at] = fwAD.make_dual(a[at], torch.ones_like(a[at]))
            with pytest.raises(NotImplementedError):
                _loss(*a)
        assert fwAD.unpack_dual(_loss(*args)).tangent is None


def test_the_op_differentiates_once(cuda):
    z, lp, idx, w = _distill_inputs(1)
    z.requires_grad_()
    loss, _ = torch.ops.pagedbatch_b200.distill_loss(z, lp, idx, w, 1.0, False, True)
    (grad,) = torch.autograd.grad(loss, z, create_graph=True)
    assert torch.equal(grad, torch.autograd.grad(pb.distill_loss(z, lp, idx, row_weight=w, reduction="sum"), z)[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), z)
