"""Parameters that change in place on the device, between calls and between replays of a captured call: whatever
kinds of sequences they were uploaded with, every sequence is verified by what they hold."""

import numpy as np
import pytest
import torch

import oracle.verify
import pagedbatch_b200 as pb
from pagedbatch_b200 import ops, workloads
from test_verify_gpu import KINDS, _drafts, _lens, _offsets, _params, _probs

pytestmark = pytest.mark.gpu

S = 12


def _case(V, dtype, kind, seed):
    lens = _lens(S, 4, seed)
    x = workloads.head_boosted(sum(lens) + S, V, seed=seed, dtype=dtype)
    params = [KINDS[kind](i) for i in range(S)]
    d, u = _drafts(x, lens, seed), np.random.default_rng(seed).random(len(x))
    return x, lens, params, d, u, _probs(x, lens, params, seed)


def _same(out, want):
    tok, acc, st = (t.cpu().numpy() for t in out)
    assert np.array_equal(st, want[2]) and np.array_equal(acc, want[1]) and np.array_equal(tok, want[0])


@pytest.mark.parametrize("noted", ["greedy", "whole", "topk", "topp", "bigk"])
@pytest.mark.parametrize("V,dtype", [(4096, torch.float32), (4099, torch.bfloat16)])
@pytest.mark.parametrize("inference", [False, True])
def test_overwritten_between_calls(cuda, noted, V, dtype, inference):
    with torch.inference_mode(inference):
        pt = _params([KINDS[noted](i) for i in range(S)])
        for kind in ("mixed", "whole", "greedy"):
            x, lens, params, d, u, probs = _case(V, dtype, kind, 1)
            pt.copy_(_params(params))
            for dp in (probs, None):
                out = pb.verify(x.cuda(), pt, torch.from_numpy(d).cuda(), _offsets(lens), torch.from_numpy(u).cuda(),
                                draft_probs=None if dp is None else dp.cuda(), with_status=True)
                _same(out, oracle.verify.verify(x, params, lens, d, u, None if dp is None else dp.numpy()))


@pytest.mark.parametrize("noted", ["greedy", "whole", "topk", "topp", "bigk", "mixed"])
@pytest.mark.parametrize("V,dtype", [(4096, torch.float32), (4096, torch.float16), (4099, torch.bfloat16)])
def test_overwritten_between_replays(cuda, noted, V, dtype):
    """One capture, replayed over other logits, drafts, random numbers and parameters of other kinds."""
    x, lens, params, d, u, probs = _case(V, dtype, noted, 2)
    pt = _params(params)
    bufs = [t.cuda() for t in (x, torch.from_numpy(d), torch.from_numpy(u), probs)]
    off = _offsets(lens)

    def call():
        return pb.verify(bufs[0], pt, bufs[1], off, bufs[2], draft_probs=bufs[3], with_status=True)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for kind in (noted, *KINDS):
        new, _, params, nd, nu, nprobs = _case(V, dtype, kind, 2)
        pt.copy_(_params(params))
        for b, t in zip(bufs, (new, torch.from_numpy(nd), torch.from_numpy(nu), nprobs), strict=True):
            b.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        _same(out, oracle.verify.verify(new, params, lens, nd, nu, nprobs.numpy()))


@pytest.mark.parametrize("noted", ["topk", "whole"])
def test_overwritten_where_equal_values_are_cut(cuda, noted):
    """Draws among many equal values, cut by top-p, by the launches that the note left."""
    n = 2
    rng = np.random.default_rng(0)
    for V in (704, 700):
        x = torch.from_numpy(rng.integers(-3, 4, (S * (n + 1), V)).astype(np.float32))
        params = [(1.0, (0.3, 0.5, 0.8, 0.97)[i % 4], (0, 0, 300, 60)[i % 4]) for i in range(S)]
        d = np.array([rng.choice(np.flatnonzero(r == r.max())) for r in x.numpy()], dtype=np.int64)
        u = rng.random(len(x)) * 0.05
        pt = _params([KINDS[noted](i) for i in range(S)])
        args = (x.cuda(), pt, torch.from_numpy(d).cuda(), _offsets([n] * S), torch.from_numpy(u).cuda())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pb.verify(*args, with_status=True)
        pt.copy_(_params(params))
        g.replay()
        torch.cuda.synchronize()
        _same(out, oracle.verify.verify(x, params, [n] * S, d, u))


def test_draft_distributions_on_the_host(cuda):
    """verify_tokens copies CPU draft_probs with CPU logits; those that are not with the logits are refused, and the
    generators keep their state."""
    lens = [2, 0, 3]
    x = workloads.head_boosted(sum(lens) + 3, 4099, seed=1)
    params = [KINDS["topk"](1), KINDS["whole"](1), KINDS["topp"](1)]
    probs = _probs(x, lens, params, 2)
    at = np.concatenate([[0], np.cumsum(np.array(lens) + 1)])
    drafts = [x[at[s] : at[s] + n].argmax(1).tolist() for s, n in enumerate(lens)]
    sp = [pb.SamplingParams(temperature=t, top_p=p, top_k=k) for t, p, k in params]

    def call(z, p, gens=None):
        return pb.verify_tokens(z, drafts, sp, gens or [torch.Generator().manual_seed(s) for s in range(3)], draft_probs=p)

    want = call(x.cuda(), probs.cuda())
    assert want == call(x, probs) == call(x.pin_memory(), probs.pin_memory()) == call(x, probs.cuda())
    gens = [torch.Generator().manual_seed(s) for s in range(3)]
    for bad in (probs, probs.cuda()[:, :-1], probs.cuda()[1:], probs.cuda().double()):
        with pytest.raises(ValueError):
            call(x.cuda(), bad, gens)
    assert call(x.cuda(), probs.cuda(), gens) == want
