"""Drafted decoding from end to end on a B200: a target model's records of its rows, a draft model trained
on them, drafts sampled from that model and verified against the target, and all of it in one captured graph. The
models are tables of logits per token, so that a row's values do not depend on how many rows are computed."""

import numpy as np
import pytest
import torch

import oracle.verify
import pagedbatch_b200 as pb
from pagedbatch_b200 import SamplingParams, ops, sample_tokens
from test_distill_gpu import U, formula

pytestmark = pytest.mark.gpu

V = 509


def _models(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    target = (3 * torch.randn(V, V, generator=g)).to(dtype)
    draft = target.float() + torch.randn(V, V, generator=g)
    return target, draft


def test_training_step(cuda):
    """A batch of contexts, some padded: the gradient of the draft's table is that of the formula."""
    target, draft = _models()
    ctx = torch.randint(0, V, (96,), generator=torch.Generator().manual_seed(1))
    counts = torch.ones(96)
    counts[-7:] = 0.0
    table = draft.cuda().requires_grad_()
    rec = pb.top_logprobs(target.cuda()[ctx.cuda()], 20)
    for tail in (False, True):
        table.grad = None
        loss = pb.distill_loss(table[ctx.cuda()], rec.logprobs, rec.indices, tail=tail, row_weight=counts.cuda(),
                               reduction="sum")
        loss.backward()
        loss64, grad64, l_err, g_err = formula(draft[ctx], rec.logprobs.cpu(), rec.indices.cpu(), tail=tail, weight=counts)
        assert abs(loss.item() - float(loss64.sum())) <= float(l_err.sum()) + 96 * U * float(loss64.abs().sum())
        want, lim = (torch.zeros(V, V, dtype=torch.float64).index_add_(0, ctx, t) for t in (grad64, g_err + U * grad64.abs()))
        size = torch.zeros(V, V, dtype=torch.float64).index_add_(0, ctx, grad64.abs())
        # torch adds a token's rows in fp32, at most 96 of them
        assert ((table.grad.cpu().double() - want).abs() <= lim + 96 * U * size + 1e-30).all()
        assert (table.grad[ctx[:-7].unique().cuda()].abs().sum(1) > 0).all()


def _draft(table, tokens, n, params, generator):
    """n drafts for each sequence, one token at a time, and the distributions they were drawn from."""
    S = len(tokens)
    out, probs = [], []
    cur = torch.tensor(tokens, device=table.device)
    for _ in range(n):
        rec = ops.pack_params(*zip(*[(p.temperature, p.top_p, p.top_k) for p in params]),
                              torch.rand(S, dtype=torch.float64, generator=generator).numpy())
        cur, _, p = ops.sample(table[cur], ops.params_tensor(rec, table.device), with_probs=True)
        out.append(cur)
        probs.append(p)
    return torch.stack(out, 1), torch.stack(probs, 1).reshape(S * n, V)


def _rows(table, tokens, drafts):
    """The target's rows of every sequence: at its last token and after each of its drafts."""
    first = torch.tensor(tokens, device=table.device)[:, None]
    return table[torch.cat([first, drafts], 1).reshape(-1)]


def test_greedy_decoding_is_the_targets(cuda):
    """Greedy sequences decoded through drafts are those decoded one token a step."""
    target, draft = (t.cuda() for t in _models())
    S, n, steps = 9, 4, 12
    params, gens = [SamplingParams(temperature=0.0)] * S, [None] * S
    want = [[s] for s in range(S)]
    for _ in range(steps * (n + 1)):
        got = sample_tokens(target[torch.tensor([w[-1] for w in want], device="cuda")], params, gens)
        for w, t in zip(want, got, strict=True):
            w.append(t)
    out, taken = [[s] for s in range(S)], 0
    for _ in range(steps):
        last = [o[-1] for o in out]
        drafts, _ = _draft(draft, last, n, params, torch.Generator().manual_seed(0))
        got = pb.verify_tokens(_rows(target, last, drafts), drafts.tolist(), params, gens)
        for o, t in zip(out, got, strict=True):
            o += t
            taken += len(t) - 1
    assert 0 < taken < S * n * steps
    for o, w in zip(out, want, strict=True):
        assert o == w[: len(o)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sampled_decoding(cuda, dtype):
    """Sampled drafts with their distributions, sequences of every kind: the tokens of the rule."""
    target, draft = (t.cuda() for t in _models(dtype))
    kinds = [(1.0, 1.0, 0), (0.8, 0.9, 0), (1.0, 1.0, 40), (0.7, 0.8, 20), (0.0, 1.0, 0), (1.3, 1.0, 300)]
    S, n = 12, 3
    params = [SamplingParams(temperature=t, top_p=p, top_k=k) for t, p, k in (kinds * 2)]
    last = list(range(S))
    gen = torch.Generator().manual_seed(5)
    for step in range(6):
        drafts, probs = _draft(draft, last, n, params, gen)
        rows = _rows(target, last, drafts)
        gens = [torch.Generator().manual_seed(100 * step + s) for s in range(S)]
        got = pb.verify_tokens(rows, drafts.tolist(), params, gens, probs)
        u = np.zeros(S * (n + 1))
        for s, p in enumerate(params):
            if p.temperature != 0:
                g = torch.Generator().manual_seed(100 * step + s)
                u[s * (n + 1) : (s + 1) * (n + 1)] = torch.rand(n + 1, dtype=torch.float64, generator=g).numpy()
        flat = torch.cat([drafts, torch.zeros_like(drafts[:, :1])], 1).reshape(-1).cpu().numpy()
        tok, acc, st = oracle.verify.verify(rows.cpu(), kinds * 2, [n] * S, flat, u, probs.cpu().numpy())
        assert not st.any()
        assert got == [tok[s * (n + 1) : s * (n + 1) + acc[s] + 1].tolist() for s in range(S)]
        last = [t[-1] for t in got]


def test_one_graph_for_the_step(cuda):
    """Record, loss, gradient, drafts and verification captured together; replays follow their inputs."""
    target, draft = (t.cuda() for t in _models())
    S, n = 8, 2
    params = ops.params_tensor(ops.pack_params([1.0] * S, [0.95] * S, [50] * S, np.linspace(0.05, 0.95, S)), "cuda")
    offsets = torch.arange(0, S * (n + 1) + 1, n + 1, dtype=torch.int32, device="cuda")
    last = torch.arange(S, device="cuda")
    u = torch.rand(S * (n + 1), dtype=torch.float64, device="cuda")
    z = draft[:S].clone().requires_grad_()

    def step():
        cur, drafts, probs = last, [], []
        for _ in range(n):
            cur, _, p = ops.sample(draft[cur], params, with_probs=True)
            drafts.append(cur)
            probs.append(p)
        ids = torch.stack([last, *drafts], 1)
        flat = torch.cat([ids[:, 1:], ids[:, :1]], 1).reshape(-1)
        rows = target[ids.reshape(-1)]
        tok, acc = pb.verify(rows, params, flat, offsets, u, torch.stack(probs, 1).reshape(S * n, V))
        rec = pb.top_logprobs(target[last], 16)
        loss = pb.distill_loss(z, rec.logprobs, rec.indices, reduction="sum")
        return tok, acc, loss.detach(), torch.autograd.grad(loss, z)[0]  # (no graph of z outlives the call)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        g = torch.Generator(device="cuda").manual_seed(seed)
        last.copy_(torch.randint(0, V, (S,), generator=g, device="cuda"))
        u.copy_(torch.rand(S * (n + 1), generator=g, dtype=torch.float64, device="cuda"))
        graph.replay()
        captured = [t.detach().clone() for t in got]
        for a, b in zip(captured, step(), strict=True):
            assert torch.equal(a, b)
