"""Verification of drafted tokens on a B200 against its restatement in whole numbers (oracle/verify.py),
token for token: every kind of parameters, element type and draft distribution, ragged sequences, odd
and unaligned rows, ties cut by top-p, invalid rows, drafts and random numbers, and the distribution
of the emitted tokens."""

import numpy as np
import pytest
import torch
from scipy import stats

import oracle.verify
import pagedbatch_b200 as pb
from pagedbatch_b200 import SamplingParams, _lib, ops, workloads

pytestmark = pytest.mark.gpu

KINDS = {
    "greedy": lambda i: (0.0, 1.0, 0),
    "whole": lambda i: ((1.0, 0.7, 2.0)[i % 3], 1.0, 0),
    "topk": lambda i: ((0.7, 1.0)[i % 2], (1.0, 0.95, 0.5)[i % 3], (1, 20, 50, 128)[i % 4]),
    "topp": lambda i: ((1.0, 0.6)[i % 2], (0.9, 0.3, 0.999)[i % 3], 0),
    "bigk": lambda i: (1.0, (1.0, 0.9)[i % 2], (200, 1500)[i % 2]),
}
KINDS["mixed"] = lambda i: list(KINDS.values())[i % 5](i // 5)


def _params(rows_params, device="cuda"):
    t, p, k = zip(*rows_params)
    return ops.params_tensor(ops.pack_params(t, p, k, np.zeros(len(t))), device)


def _offsets(lens):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(np.asarray(lens) + 1)]).astype(np.int32)).cuda()


def _drafts(x, lens, seed, favourite=0.6):
    """A draft per row: mostly the row's largest logit, else a likely or any token."""
    rng = np.random.default_rng(seed)
    R, V = x.shape
    best = x.float().argmax(1).numpy()
    top = torch.topk(x.float(), min(8, V), dim=1).indices.numpy()
    d = np.where(rng.random(R) < favourite, best, top[np.arange(R), rng.integers(0, top.shape[1], R)])
    return np.where(rng.random(R) < 0.1, rng.integers(0, V, R), d).astype(np.int64)


def _probs(x, lens, params, seed, dtype=torch.float32):
    """Draft distributions: the target's softmax with noise, cut to a few tokens on some rows."""
    g = torch.Generator().manual_seed(seed)
    rows, seq, r = [], [], 0
    for s, n in enumerate(lens):
        rows += list(range(r, r + n))
        seq += [s] * n
        r += n + 1
    t = torch.tensor([params[s][0] or 1.0 for s in seq], dtype=torch.float32).reshape(-1, 1)
    y = (x[rows].float() + torch.randn(len(rows), x.shape[1], generator=g)) / t
    cut = torch.rand(len(rows), 1, generator=g) < 0.5
    if len(rows):
        floor = torch.topk(y, min(30, x.shape[1]), dim=1).values[:, -1:]
        y = torch.where(cut & (y < floor), -torch.inf, y)
    return torch.softmax(y, 1).to(dtype)


def _check(x, params, lens, drafts, u, probs=None, view=None, marks=True):
    """The kernel against the oracle on CPU logits x (or `view`, the same values on the device)."""
    dev = x.cuda() if view is None else view
    pt = _params(params)
    if not marks:
        pt = pt.clone()  # without the host's note of which kinds of sequences it holds
    got = pb.verify(dev, pt, torch.from_numpy(drafts).cuda(), _offsets(lens), torch.from_numpy(u).cuda(),
                    draft_probs=None if probs is None else probs.cuda(), with_status=True)
    tok, acc, st = (t.cpu().numpy() for t in got)
    o_tok, o_acc, o_st = oracle.verify.verify(x, params, lens, drafts, u, None if probs is None else probs.float().numpy())
    assert np.array_equal(st, o_st), (np.flatnonzero(st != o_st)[:8], st[st != o_st][:8], o_st[st != o_st][:8])
    assert np.array_equal(acc, o_acc), (np.flatnonzero(acc != o_acc)[:8], acc[acc != o_acc][:8], o_acc[acc != o_acc][:8])
    assert np.array_equal(tok, o_tok), (np.flatnonzero(tok != o_tok)[:8], tok[tok != o_tok][:8], o_tok[tok != o_tok][:8])
    return tok, acc, st


def _lens(S, most, seed):
    return np.random.default_rng(seed).integers(0, most + 1, S).tolist()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sampled", [False, True])
def test_kinds_and_types(cuda, kind, dtype, sampled):
    S, V = 13, 4099
    lens = _lens(S, 6, 1)
    R = sum(lens) + S
    x = workloads.head_boosted(R, V, seed=5, dtype=dtype)
    params = [KINDS[kind](i) for i in range(S)]
    u = np.random.default_rng(2).random(R)
    probs = _probs(x, lens, params, 3) if sampled else None
    _check(x, params, lens, _drafts(x, lens, 4), u, probs)
    _check(x, params, lens, _drafts(x, lens, 4), u, probs, marks=False)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 31, 33, 127, 1000, 50021])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies(cuda, V, dtype):
    S = 10
    lens = _lens(S, 4, V)
    R = sum(lens) + S
    x = workloads.head_boosted(R, V, seed=V, dtype=dtype)
    params = [KINDS["mixed"](i) for i in range(S)]
    u = np.random.default_rng(V).random(R)
    _check(x, params, lens, _drafts(x, lens, V), u, _probs(x, lens, params, V))
    _check(x, params, lens, _drafts(x, lens, V), u)


@pytest.mark.parametrize("S,most", [(1, 0), (1, 7), (200, 0), (300, 3), (2, 700)])
def test_batches(cuda, S, most):
    """One row alone, no drafts at all, more sequences than SMs, and more drafts than a CTA's threads."""
    V = 512
    lens = [most] * S
    R = sum(lens) + S
    x = workloads.head_boosted(R, V, seed=S + most)
    params = [KINDS["mixed"](i + (most == 700)) for i in range(S)]
    if most == 700:  # long runs of accepted drafts
        params = [(0.0, 1.0, 0), (1.0, 1.0, 1)]
    u = np.random.default_rng(S).random(R) * (1e-3 if most == 700 else 1.0)
    d = _drafts(x, lens, S, favourite=0.999 if most == 700 else 0.6)
    if most == 700:
        d = x.argmax(1).numpy().astype(np.int64)
        d[650] = (d[650] + 1) % V
    tok, acc, _ = _check(x, params, lens, d, u)
    if most == 700:
        assert acc[0] == 650 and acc[1] == 700


def test_full_vocabulary(cuda):
    S, V = 12, workloads.LLAMA3_VOCAB
    lens = _lens(S, 3, 8)
    R = sum(lens) + S
    x = workloads.head_boosted(R, V, seed=9, dtype=torch.bfloat16)
    params = [KINDS["mixed"](i) for i in range(S)]
    u = np.random.default_rng(10).random(R)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        _check(x, params, lens, _drafts(x, lens, 11), u, _probs(x, lens, params, 12, dtype))


def test_flat_rows(cuda):
    """Every weight matters: the kept set is nearly the whole row."""
    S, V = 8, 50021
    lens = [2] * S
    x = workloads.flat(3 * S, V, seed=3)
    params = [(1.0, 1.0, 0), (0.7, 0.999, 0)] * (S // 2)
    u = np.random.default_rng(4).random(3 * S)
    _check(x, params, lens, _drafts(x, lens, 5), u, _probs(x, lens, params, 6))
    _check(x, params, lens, _drafts(x, lens, 5), u)


def test_kinds_named_wrongly(cuda):
    """A kind that the params' note leaves out is not settled (status 8), and nothing else is disturbed."""
    S, V = 12, 1000
    x = workloads.head_boosted(S, V, seed=1)
    params = [((0.0, 1.0, 0), (1.0, 1.0, 0), (1.0, 0.9, 0), (1.0, 1.0, 500))[i % 4] for i in range(S)]
    d, off = torch.zeros(S, dtype=torch.int64).cuda(), _offsets([0] * S)
    u = np.random.default_rng(1).random(S)
    want, _, _ = oracle.verify.verify(x, params, [0] * S, np.zeros(S, np.int64), u)
    bit = [_lib.VERIFY_SMALL, _lib.VERIFY_WHOLE, _lib.VERIFY_TOPP, _lib.VERIFY_OTHER]
    for kinds in range(1, 16):
        pt = _params(params)
        pt._pb_kinds = (kinds, 0)
        tok, _, st = pb.verify(x.cuda(), pt, d, off, torch.from_numpy(u).cuda(), with_status=True)
        for i in range(S):
            # (the launch for other kinds takes top-p rows too)
            named = kinds & bit[i % 4] or (i % 4 == 2 and kinds & _lib.VERIFY_OTHER)
            assert (tok[i] == want[i] and st[i] == 0) if named else (tok[i] == -1 and st[i] == _lib.ROW_INTERNAL)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_top_p_steps(cuda, dtype):
    """Top-p cuts in every part of a row: near the top, in the body, at the end, among many equals, in
    rows so flat that one step of the histogram holds them, and with temperatures at the ends."""
    V = 20011
    rows = [workloads.head_boosted(6, V, seed=1), workloads.flat(4, V, seed=2), torch.zeros(2, V),
            workloads.head_boosted(4, V, seed=3).round(), workloads.head_boosted(4, V, seed=4) * 1e-3]
    x = torch.cat(rows).to(dtype)
    S = len(x)
    for k, p in enumerate((1e-6, 0.1, 0.5, 0.9, 0.999, 1.0 - 1e-7)):
        params = [((1.0, 0.3, 2.5, 1e-3)[(i + k) % 4], p, 0) for i in range(S)]
        u = np.random.default_rng(k).random(S)
        _check(x, params, [0] * S, np.zeros(S, np.int64), u)


def test_weights_whose_reduction_is_a_tie(cuda):
    """Distances d from the maximum whose d log2(e), rounded, is a half: the weight's reduction must round
    the product before it rounds to a whole number. One rounding for both takes another whole number at
    some of them and ends in another last bit, so the draws are made where that bit decides."""
    log2e = np.float32(float.fromhex("0x1.715476p+0"))
    rows, us = [], []
    for k in range(3, 24):
        near = np.float32(-(k + 0.5) / float(log2e))
        for step in range(-3, 4):
            d = near
            for _ in range(abs(step)):
                d = np.nextafter(d, np.float32(np.inf if step > 0 else -np.inf))
            x = np.float32(1.0) + d
            if d * log2e != -(k + 0.5) or x - np.float32(1.0) != d:
                continue
            n = min(int(np.exp(float(-d))), 200000)
            q = oracle.verify.weights(np.array([d], dtype=np.float32), 0.0)[0]
            edge = n * int(q) / (n * int(q) + 2**40)  # where the draw passes from the tied values to the maximum
            rows += [np.append(np.full(n, x, dtype=np.float32), np.float32(1.0))] * 2
            us += [edge * (1 - 2e-9), edge * (1 + 2e-9)]
    assert len(rows) > 20
    for row, u in zip(rows, us, strict=True):
        x = torch.from_numpy(row)[None]
        _check(x, [(1.0, 1.0, 0)], [0], np.zeros(1, dtype=np.int64), np.array([u]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [7, 4099, 50021])
def test_random_numbers_at_the_edge(cuda, dtype, V):
    """Random numbers a few roundings around the draft's probability: the exact masses decide."""
    n = 24
    params = [((1.0, 0.7, 3.0, 1e-3)[s % 4], 1.0, 0) for s in range(8)]
    S = len(params)
    x = workloads.head_boosted(S * (n + 1), V, seed=V, dtype=dtype)
    x[n + 1 : 2 * (n + 1)] -= x[n + 1 : 2 * (n + 1)].max(1, keepdim=True).values  # largest value 0
    x[2 * (n + 1) : 3 * (n + 1)] += 500.0
    d = _drafts(x, [n] * S, 1, favourite=0.5)
    probs = _probs(x, [n] * S, params, 2).clamp(min=1e-6)
    u, row = np.zeros(len(x)), 0
    for s, (T, _, _) in enumerate(params):
        keys = (x[s * (n + 1) : (s + 1) * (n + 1)].float() / torch.tensor(T)).numpy()
        for j in range(n):
            r = s * (n + 1) + j
            w = oracle.verify.weights(keys[j], float(keys[j].max()))
            share = float(w[d[r]]) / float(w.sum())
            # mostly just inside, so that a sequence goes on; the last few wherever they fall
            off = (-1, -3, -1e-12 * 2**53, -1e-6 * 2**53)[j % 4] if j < n - 4 else (-1, 0, 1, 2)[(s + j) % 4]
            u[r] = min(max(share / float(probs[row, d[r]]) * (1 + off * 2.0**-53), 0.0), 1 - 2.0**-53)
            row += 1
    _check(x, params, [n] * S, d, u, probs)
    _check(x, params, [n] * S, d, u, probs, marks=False)


def test_strides_and_offsets(cuda):
    """Rows that start anywhere, rows apart, and draft distributions with rows apart."""
    S, V = 9, 1003
    lens = _lens(S, 4, 2)
    R = sum(lens) + S
    params = [KINDS["mixed"](i) for i in range(S)]
    u = np.random.default_rng(3).random(R)
    for dtype in (torch.float32, torch.float16):
        x = workloads.head_boosted(R, V, seed=4, dtype=dtype)
        probs = _probs(x, lens, params, 5)
        for shift, stride in ((1, 1009), (3, 1011), (0, 1024), (5, V + 5)):
            buf = torch.full((R * stride + 16,), float("nan"), dtype=dtype, device="cuda")
            view = buf[shift:].as_strided((R, V), (stride, 1))
            view.copy_(x)
            pbuf = torch.full((R - S, 1100), float("nan"), device="cuda")
            pbuf[:, 7 : 7 + V] = probs.cuda()
            dev = pb.verify(view, _params(params), torch.from_numpy(_drafts(x, lens, 6)).cuda(), _offsets(lens),
                            torch.from_numpy(u).cuda(), draft_probs=pbuf[:, 7 : 7 + V])
            ref = oracle.verify.verify(x, params, lens, _drafts(x, lens, 6), u, probs.numpy())
            assert np.array_equal(dev[0].cpu().numpy(), ref[0]) and np.array_equal(dev[1].cpu().numpy(), ref[1])


def test_ties_cut_by_top_p(cuda):
    """Equal values at the last kept key, of which top-p keeps those of lowest index: drafts on both
    sides of the cut, and draws over the cut group."""
    rng = np.random.default_rng(0)
    S, V, n = 60, 700, 3
    x = torch.from_numpy(rng.integers(-3, 4, (S * (n + 1), V)).astype(np.float32))
    lens = [n] * S
    params = [(1.0, (0.3, 0.5, 0.8, 0.97)[i % 4], (0, 0, 100, 60)[i % 4]) for i in range(S)]
    drafts = x.argmax(1).numpy()
    ties = [np.flatnonzero(r == r.max()) for r in x.numpy()]
    drafts = np.array([t[rng.integers(0, len(t))] for t in ties], dtype=np.int64)
    u = rng.random(len(x)) * 0.02
    tok, acc, _ = _check(x, params, lens, drafts, u)
    assert 0 < acc.sum() < S * n  # some were kept, some cut
    u = rng.random(len(x))
    _check(x, params, lens, drafts, u, _probs(x, lens, params, 1))


def test_masked_rows(cuda):
    """Vocabulary masked with -inf and with the type's lowest value; a single value left."""
    S, V = 12, 2000
    lens = [2] * S
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = workloads.head_boosted(3 * S, V, seed=1, dtype=dtype)
        for r in range(3 * S):
            x[r, (r % 7) :: 2] = -torch.inf if r % 2 else torch.finfo(dtype).min
        x[3, :] = -torch.inf
        x[3, 77] = 1.0
        x[6, :] = torch.finfo(dtype).min
        x[6, 1999] = 2.0
        params = [KINDS["mixed"](i) for i in range(S)]
        u = np.random.default_rng(2).random(3 * S)
        _check(x, params, lens, _drafts(x, lens, 3), u, _probs(x.clamp(min=-1e4), lens, params, 4))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,shift", [(50024, 0), (50021, 3)])
def test_few_allowed_tokens(cuda, dtype, V, shift):
    """Rows of which a mask leaves fewer tokens than top_k keeps, or one: masked ones are never drawn."""
    g = torch.Generator().manual_seed(V)
    S, n = 10, 2
    x = torch.empty(S * (n + 1), V, dtype=dtype)
    for r in range(len(x)):
        few = (1, 5, 30, 200)[r % 4]
        x[r] = (-torch.inf, torch.finfo(dtype).min, -60.0)[r % 3]
        x[r, torch.randperm(V, generator=g)[:few]] = torch.randn(few, generator=g).to(dtype)
    buf = torch.zeros(len(x), V + 8, dtype=dtype, device="cuda")
    view = buf[:, shift : shift + V]
    view.copy_(x)
    for kind in ("topk", "topp", "mixed"):
        params = [KINDS[kind](i) for i in range(S)]
        for seed in range(2):
            u = np.random.default_rng(seed).random(len(x))
            probs = _probs(x.clamp(min=-1e4), [n] * S, params, seed) if seed else None
            tok, _, st = _check(x, params, [n] * S, _drafts(x, [n] * S, seed), u, probs, view=view)
            assert not st.any()
            drawn = torch.from_numpy(tok)
            at = drawn >= 0
            assert (x[at, drawn[at]] > -20).all()


def test_invalid_rows_and_numbers(cuda):
    """A row without a distribution fails its sequence only where the sequence reaches it; so does a
    random number outside [0, 1); a draft outside the vocabulary is rejected."""
    S, V, n = 12, 300, 2
    lens = [n] * S
    x = workloads.head_boosted(S * 3, V, seed=2)
    params = [(1.0, 1.0, (0, 20, 200)[i % 3]) for i in range(S)]
    best = x.argmax(1).numpy().astype(np.int64)
    drafts, u = best.copy(), np.full(S * 3, 1e-9)
    x[0, 5] = torch.nan           # sequence 0 fails at once
    x[4, 5] = torch.inf           # sequence 1 after one draft
    x[8, :] = -torch.inf          # sequence 2 at its last row
    drafts[9], u[9] = (best[9] + 1) % V, 0.999
    x[10, 3] = torch.nan          # sequence 3 stops before it
    drafts[12] = -1
    drafts[15] = V
    drafts[18] = 1 << 40
    u[21], u[25], u[29] = 1.0, -0.25, np.nan
    tok, acc, st = _check(x, params, lens, drafts, u)
    assert st[:4].tolist() == [1, 1, 1, 0] and st[7:10].tolist() == [2, 2, 2]
    assert acc[:3].tolist() == [0, 1, 2] and acc[4:7].tolist() == [0, 0, 0] and (tok[[12, 15, 18]] >= 0).all()
    probs = _probs(x.nan_to_num(0.0, 0.0, 0.0), lens, params, 3)
    _check(x, params, lens, drafts, u, probs)


def test_rejected_parameters(cuda):
    x = workloads.head_boosted(4, 300, seed=3)
    rec = ops.pack_params([1.0, 1.0, 1.0, -1.0], [0.9, 0.0, 1.5, 1.0], [-1, 0, 0, 0], np.zeros(4))
    out = pb.verify(x.cuda(), ops.params_tensor(rec, "cuda"), torch.zeros(4, dtype=torch.int64).cuda(), _offsets([0] * 4),
                    torch.zeros(4, dtype=torch.float64).cuda(), with_status=True)
    assert out[2].tolist() == [_lib.ROW_BAD_PARAMS] * 4 and out[0].tolist() == [-1] * 4


def test_edges_of_the_draft_distribution(cuda):
    """No draft mass, all of it, more than all of it, NaN and negative values; the ends of [0, 1)."""
    S, V, n = 16, 257, 1
    lens = [n] * S
    x = workloads.head_boosted(2 * S, V, seed=6)
    params = [KINDS["mixed"](i) for i in range(S)]
    probs = _probs(x, lens, params, 7)
    probs[0:4] = 0.0
    probs[4:8] = 1.0        # empty residual: the draw is from the target
    probs[8] = torch.inf
    probs[9] = torch.nan
    probs[10] = -0.5
    probs[11] = 1e-45
    for val in (0.0, 1.0 - 2.0**-53, 2.0**-53, 0.5):
        _check(x, params, lens, _drafts(x, lens, 8), np.full(2 * S, val), probs)
        _check(x, params, lens, _drafts(x, lens, 8), np.full(2 * S, val))


def test_draft_from_the_target_itself_is_accepted(cuda):
    """Drafts drawn from the target's own probabilities (ops.sample with_probs) are all but always
    accepted: d = P / Z up to one rounding."""
    S, V, n = 64, 4099, 3
    R = S * (n + 1)
    x = workloads.head_boosted(R, V, seed=1).cuda()
    p = [KINDS["topk"](s) if s % 2 else (1.0, 1.0, 0) for s in range(S)]
    per_row = [p[r // (n + 1)] for r in range(R)]
    rng = np.random.default_rng(3)
    rec = ops.pack_params(*zip(*[(a, b, c) for a, b, c in per_row]), rng.random(R))
    tok, _, probs = ops.sample(x, ops.params_tensor(rec, x.device), None, with_probs=True)
    keep = torch.from_numpy(np.arange(R) % (n + 1) != n).cuda()
    u = torch.from_numpy(rng.random(R) * (1 - 1e-6)).cuda()
    out, acc = pb.verify(x, _params(p), tok, _offsets([n] * S), u, draft_probs=probs[keep])
    assert acc.tolist() == [n] * S
    assert torch.equal(out[keep], tok[keep])


@pytest.mark.parametrize("with_probs", [True, False])
@pytest.mark.parametrize("params", [(1.0, 1.0, 0), (0.8, 0.9, 0), (1.2, 0.95, 12)])
def test_emitted_tokens_follow_the_target(cuda, params, with_probs):
    """The first emitted token of 200000 one-draft sequences over one row has the target's distribution
    (chi-square at 1e-4, expected counts below 5 pooled), whatever the draft's."""
    S, V = 200_000, 48
    rng = np.random.default_rng(5)
    g = torch.Generator().manual_seed(1)
    row = torch.randn(1, V, generator=g) * 2
    x = row.expand(2 * S, V).contiguous().cuda()
    draft_p = torch.softmax(row + torch.randn(1, V, generator=g), 1).float()
    d = rng.choice(V, S, p=(draft_p[0].double() / draft_p.double().sum()).numpy()) if with_probs else np.full(S, 3)
    drafts = np.zeros(2 * S, np.int64)
    drafts[0::2] = d
    u = rng.random(2 * S)
    out, acc = pb.verify(x, _params([params] * S), torch.from_numpy(drafts).cuda(), _offsets([1] * S),
                         torch.from_numpy(u).cuda(), draft_probs=draft_p.expand(S, V).cuda() if with_probs else None)
    first, second, acc = out[0::2].cpu().numpy(), out[1::2].cpu().numpy(), acc.cpu().numpy()
    # the target's distribution of this row: the sampler's own probabilities
    rec = ops.pack_params([params[0]], [params[1]], [params[2]], [0.0])
    _, _, probs = ops.sample(row.cuda(), ops.params_tensor(rec, "cuda"), None, with_probs=True)
    p = probs[0].double().cpu().numpy()
    p /= p.sum()
    # a draft is accepted with probability sum_i min(p_i, d_i) over the drafts' distribution d
    d = draft_p[0].double().numpy() / draft_p.double().sum().item() if with_probs else np.eye(V)[3]
    assert stats.binomtest(int(acc.sum()), S, min(1.0, np.minimum(p, d).sum())).pvalue > 1e-6
    for tok in (first, second[acc == 1]):
        if not tok.size:
            continue
        seen = np.bincount(tok, minlength=V).astype(float)
        assert seen[p == 0].sum() == 0
        want = p * tok.size
        small = want < 5
        seen, want = np.append(seen[~small], seen[small].sum()), np.append(want[~small], want[small].sum())
        ok = want > 0
        assert stats.chisquare(seen[ok], want[ok] * seen.sum() / want.sum()).pvalue > 1e-4


def test_verify_tokens(cuda):
    """The host-level call against the device-level one, and its use of the generators."""
    S, V = 6, 4099
    drafts = [[], [5], [7, 8, 9], [1, 2], [], [3]]
    lens = [len(d) for d in drafts]
    R = sum(lens) + S
    x = workloads.head_boosted(R, V, seed=11)
    best = x.argmax(1).tolist()
    off = np.concatenate([[0], np.cumsum(np.array(lens) + 1)])
    drafts = [[best[off[s] + j] for j in range(lens[s])] for s in range(S)]
    params = [SamplingParams(temperature=t, top_p=p, top_k=k) for t, p, k in (KINDS["mixed"](i) for i in range(S))]
    got = pb.verify_tokens(x, drafts, params, [torch.Generator().manual_seed(s) for s in range(S)])
    u = np.zeros(R)
    for s in range(S):
        if params[s].temperature:
            u[off[s] : off[s + 1]] = torch.rand(lens[s] + 1, dtype=torch.float64, generator=torch.Generator().manual_seed(s))
    flat = np.zeros(R, np.int64)
    for s in range(S):
        flat[off[s] : off[s] + lens[s]] = drafts[s]
    tok, acc, _ = oracle.verify.verify(x, [(p.temperature, p.top_p, p.top_k) for p in params], lens, flat, u)
    assert got == [tok[off[s] : off[s] + acc[s] + 1].tolist() for s in range(S)]
    assert got == pb.verify_tokens(x.cuda(), drafts, params, [torch.Generator().manual_seed(s) for s in range(S)])
    x[2, 9] = torch.nan
    with pytest.raises(RuntimeError, match="probability tensor contains"):
        pb.verify_tokens(x, drafts, [SamplingParams()] * S, [torch.Generator().manual_seed(s) for s in range(S)])
    assert pb.verify_tokens(x[:0], [], [], []) == []


def test_streams_graphs_and_repeats(cuda):
    """Another stream, the custom op, two captured graphs replayed in turn, and the same bits each time."""
    S, V = 20, 4099
    lens = _lens(S, 5, 1)
    R = sum(lens) + S
    params = [KINDS["mixed"](i) for i in range(S)]
    pt, off = _params(params), _offsets(lens)
    cases = []
    for seed in (1, 2):
        x = workloads.head_boosted(R, V, seed=seed)
        d, u = _drafts(x, lens, seed), np.random.default_rng(seed).random(R)
        probs = _probs(x, lens, params, seed)
        cases.append((x.cuda(), torch.from_numpy(d).cuda(), torch.from_numpy(u).cuda(), probs.cuda(),
                      oracle.verify.verify(x, params, lens, d, u, probs.numpy())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, d, u, probs, want in cases:
            out = torch.ops.pagedbatch_b200.verify(x, pt, d, off, u, probs)
            assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])
    torch.cuda.synchronize()
    graphs = []
    for x, d, u, probs, want in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pb.verify(x, pt, d, off, u, draft_probs=probs)
        graphs.append((g, out, want))
    for _ in range(3):
        for g, out, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out, want in graphs:
            assert np.array_equal(out[0].cpu().numpy(), want[0]) and np.array_equal(out[1].cpu().numpy(), want[1])


def test_rows_far_apart(cuda):
    """Row starts past 2^31 elements."""
    V, stride = 1000, (1 << 30) + 8
    x = workloads.head_boosted(3, V, seed=1, dtype=torch.bfloat16)
    buf = torch.empty(2 * stride + V, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((3, V), (stride, 1))
    view.copy_(x)
    for params in ((1.0, 1.0, 0), (1.0, 0.9, 50), (0.0, 1.0, 0)):
        d = x.float().argmax(1).numpy().astype(np.int64)
        _check(x, [params], [2], d, np.array([1e-3, 0.3, 0.5]), view=view)
