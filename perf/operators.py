"""The cases of the drafted-decoding operators: drafted tokens verified against the target's rows,
the top log-probabilities of a row (what a teacher records), and the distillation loss that trains
a draft model on such records.

``run`` computes one pass: with ``own`` the package's entry points, else the plain form in torch
operations. Logits are shaped like the sampling workloads' (3 N(0,1) plus a Zipf-like head on a
permutation of the ids), vocabularies and row counts like theirs too (49152 and 128256; 1 to 1024
rows), with odd ones among them.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
SMALL_VOCAB, LARGE_VOCAB = 49152, 128256


# ---- cases -------------------------------------------------------------------------------------


def listed():
    return [
        # one sequence with four drafts of a draft model: a lone user's decode step, all latency
        dict(name="verify_1x4_f32_topk", op="verify", seqs=1, most=4, ragged=False, vocab=SMALL_VOCAB, dtype="f32",
             kind="topk", temperature=0.8, top_k=50, top_p=0.9, sampled=True),
        # a small mixed batch (greedy, temperature, top-k and top-p requests) with drafts looked up
        # in the prompt (no draft distribution), 0 to 7 a sequence, and a vocabulary of odd size
        dict(name="verify_16_f16_mixed", op="verify", seqs=16, most=7, ragged=True, vocab=50021, dtype="f16",
             kind="mixed", temperature=0.8, top_k=40, top_p=0.9, sampled=False),
        # an ordinary serving batch: top-k 50 and top-p 0.95 requests, four drafts each
        dict(name="verify_64x4_f32_topk", op="verify", seqs=64, most=4, ragged=False, vocab=LARGE_VOCAB, dtype="f32",
             kind="topk", temperature=0.7, top_k=50, top_p=0.95, sampled=True),
        # a full batch of requests that sample the whole distribution (as reinforcement learning
        # does), one to five drafts each: every row's mass is summed over the vocabulary
        dict(name="verify_256_bf16_temp", op="verify", seqs=256, most=5, ragged=True, vocab=LARGE_VOCAB, dtype="bf16",
             kind="temp", temperature=1.0, top_k=0, top_p=1.0, sampled=True),
        # top-p without top-k, three drafts each: the kept set is cut by mass over the whole row
        dict(name="verify_64x3_bf16_topp", op="verify", seqs=64, most=3, ragged=False, vocab=SMALL_VOCAB, dtype="bf16",
             kind="topp", temperature=1.0, top_k=0, top_p=0.9, sampled=True),
        # the log-probabilities a server returns beside one request's token
        dict(name="top_1_f16_k7", op="top", rows=1, vocab=50021, dtype="f16", k=7, temperature=0.8),
        # a decode step of a served batch recorded as a teacher
        dict(name="top_256_f32_k50", op="top", rows=256, vocab=LARGE_VOCAB, dtype="f32", k=50, temperature=1.0),
        # a prefill or scoring pass recorded as a teacher
        dict(name="top_1024_bf16_k128", op="top", rows=1024, vocab=LARGE_VOCAB, dtype="bf16", k=128, temperature=1.0),
        # one small training step, a weight for each row
        dict(name="distill_32_f32_k20", op="distill", rows=32, vocab=SMALL_VOCAB, dtype="f32", k=20, tail=False,
             temperature=1.0, reduction="none", backward=True),
        # a batch of odd sizes with padded rows, records of differing length, the tail kept as a bucket
        dict(name="distill_1001_f16_tail", op="distill", rows=1001, vocab=50021, dtype="f16", k=33, tail=True,
             temperature=2.0, reduction="none", backward=True),
        # evaluation: the loss alone
        dict(name="distill_2048_bf16_eval", op="distill", rows=2048, vocab=SMALL_VOCAB, dtype="bf16", k=100, tail=True,
             temperature=1.0, reduction="none", backward=False),
        # a full training step at the large vocabulary
        dict(name="distill_4096_bf16_sum", op="distill", rows=4096, vocab=LARGE_VOCAB, dtype="bf16", k=64, tail=True,
             temperature=1.0, reduction="sum", backward=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["verify", "verify", "top", "distill", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "verify":
        kind = rng.choice(["topk", "mixed", "temp", "topp"])
        vocab = _log_int(rng, 1000, LARGE_VOCAB)
        most = rng.randint(0, 7)
        seqs = min(_log_int(rng, 1, 256), max(1, (1024 * LARGE_VOCAB) // (vocab * (most + 1))), 1024 // (most + 1))
        return dict(op=op, seqs=seqs, most=most, ragged=rng.random() < 0.5, vocab=vocab, dtype=dtype, kind=kind,
                    temperature=round(rng.uniform(0.5, 1.5), 2), top_k=0 if kind in ("temp", "topp") else _log_int(rng, 1, 200),
                    top_p=1.0 if kind == "temp" else round(rng.uniform(0.5, 0.99), 3), sampled=rng.random() < 0.6)
    if op == "top":
        vocab = _log_int(rng, 300, LARGE_VOCAB)
        return dict(op=op, rows=_log_int(rng, 1, 1024), vocab=vocab, dtype=dtype, k=min(vocab, _log_int(rng, 1, 256)),
                    temperature=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)]))
    vocab = _log_int(rng, 300, LARGE_VOCAB)
    return dict(op=op, rows=min(_log_int(rng, 1, 4096), 4096 * 2 // BYTES[dtype]), vocab=vocab, dtype=dtype,
                k=min(vocab // 2, _log_int(rng, 4, 256)), tail=rng.random() < 0.5,
                temperature=rng.choice([1.0, round(rng.uniform(0.7, 3.0), 2)]),
                reduction=rng.choice(["none", "sum"]), backward=rng.random() < 0.8)


def _lengths(case):
    """Drafts of each sequence: `most`, or (ragged) spread over 0..most."""
    if not case["ragged"]:
        return [case["most"]] * case["seqs"]
    return [(7 * s + 3) % (case["most"] + 1) for s in range(case["seqs"])]


def work(case):
    n, v, es = case.get("rows"), case["vocab"], BYTES[case["dtype"]]
    if case["op"] == "verify":
        rows = sum(_lengths(case)) + case["seqs"]
        # every row of logits once, the draft and the random number of each row, the tokens; of the
        # draft's distribution only its value at each drafted token is certain to be needed
        per_row = v * es + 8 + 8 + 8 + (4 if case["sampled"] else 0)
        return {"bytes": rows * per_row + case["seqs"] * 12, "flops": 3 * rows * v}
    if case["op"] == "top":
        return {"bytes": n * (v * es + case["k"] * 8 + 4), "flops": 3 * n * v}
    passes = 2 if case["backward"] else 1  # the logits read once, the gradient written once
    return {"bytes": n * (passes * v * es + case["k"] * 8 + 8), "flops": (6 if case["backward"] else 3) * n * v}


# ---- inputs ------------------------------------------------------------------------------------


def _logits(g, rows, vocab, dtype):
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(3.0)
    shift = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    rank = (torch.arange(vocab, device="cuda") * 1000003 + shift) % vocab  # a permutation of 0..vocab-1
    x += 8.0 * (rank + 1).float().pow(-0.7)
    return x.to(DTYPES[dtype])


def _verify_params(case):
    """Per sequence: temperature, top_k, top_p."""
    s = case["seqs"]
    if case["kind"] != "mixed":
        return [case["temperature"]] * s, [case["top_k"]] * s, [case["top_p"]] * s
    t, k, p = case["temperature"], case["top_k"], case["top_p"]
    modes = [(0.0, 0, 1.0), (t, 0, 1.0), (t, k, 1.0), (t, 0, p)]
    return tuple(list(c) for c in zip(*(modes[i % 4] for i in range(s))))


def _prepare_verify(case, g):
    lens = np.array(_lengths(case))
    s, v = case["seqs"], case["vocab"]
    offsets = np.concatenate([[0], np.cumsum(lens + 1)])
    rows = int(offsets[-1])
    temps, ks, ps = _verify_params(case)
    x = _logits(g, rows, v, case["dtype"])
    seq_of = torch.from_numpy(np.repeat(np.arange(s), lens + 1)).cuda()
    last = torch.zeros(rows, dtype=torch.bool)
    last[torch.from_numpy(offsets[1:] - 1)] = True
    draft_rows = torch.nonzero(~last.cuda()).flatten()
    t = torch.tensor([a if a > 0 else 1.0 for a in temps], dtype=torch.float32, device="cuda")
    drafts = torch.zeros(rows, dtype=torch.int64, device="cuda")
    probs = None
    if case["sampled"]:
        # the draft model: the target's logits with noise, its own top-k cut, tokens drawn from it
        y = x[draft_rows].float()
        y += 0.8 * torch.randn(y.shape, generator=g, device="cuda")
        y /= t[seq_of[draft_rows], None]
        if max(ks) > 0 and y.numel():
            k = min(max(ks), v)
            floor = torch.topk(y, k, dim=1).values[:, -1:]
            y.masked_fill_(y < floor, -math.inf)
        probs = torch.softmax(y, dim=1) if y.numel() else torch.zeros(0, v, device="cuda")
        u = torch.rand(len(draft_rows), 1, generator=g, device="cuda")
        cum = torch.cumsum(probs, 1)
        drafts[draft_rows] = (cum < u * cum[:, -1:]).sum(1).clamp(max=v - 1) if y.numel() else drafts[draft_rows]
    else:
        # looked-up drafts: mostly the target's favourite, sometimes anything
        best = x[draft_rows].float().argmax(1) if len(draft_rows) else drafts[draft_rows]
        any_ = torch.randint(0, v, (len(draft_rows),), generator=g, device="cuda")
        drafts[draft_rows] = torch.where(torch.rand(len(draft_rows), generator=g, device="cuda") < 0.7, best, any_)
    u53 = torch.randint(0, 1 << 53, (rows,), generator=g, device="cuda")
    st = dict(logits=x, drafts=drafts, offsets=torch.from_numpy(offsets.astype(np.int32)).cuda(),
              uniforms=u53.double() * 2.0**-53, draft_probs=probs, temps=temps, ks=ks, ps=ps)
    if own:
        # the requests' packed parameters, which a serving loop keeps while the batch stays the same
        from pagedbatch_b200 import ops

        rec = ops.pack_params(temps, ps, ks, np.zeros(s))
        st["params"] = ops.params_tensor(rec, "cuda")
    else:
        st["sorted"] = case["kind"] != "temp"
        st["seq_of"] = seq_of
        st["params_t"] = (torch.tensor(temps, dtype=torch.float64).float().cuda(), torch.tensor(ks).cuda(),
                          torch.tensor(ps, dtype=torch.float64).float().cuda())
    return st


def _prepare_distill(case, g):
    n, v, k = case["rows"], case["vocab"], case["k"]
    z = _logits(g, n, v, case["dtype"])
    # a teacher that the student is still far from, at the loss's temperature
    y = z.float() / case["temperature"] + 2.0 * torch.randn(n, v, generator=g, device="cuda")
    top = torch.topk(y, k, dim=1)
    lp = top.values - torch.logsumexp(y, 1, keepdim=True)
    del y
    idx = top.indices.to(torch.int32)
    if k > 1:  # records of differing length, and padded rows
        short = torch.rand(n, 1, generator=g, device="cuda") < 0.2
        length = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
        idx = torch.where(short & (torch.arange(k, device="cuda") >= length), -1, idx)
        idx = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.05, -1, idx)
    w = torch.rand(n, generator=g, device="cuda") + 0.5
    return dict(student=z, lp=lp, idx=idx, weight=w)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        st = _prepare_verify(case, g)
    elif case["op"] == "top":
        st = dict(logits=_logits(g, case["rows"], case["vocab"], case["dtype"]))
    else:
        st = _prepare_distill(case, g)
    st["case"] = dict(case)
    return st


# ---- plain forms -------------------------------------------------------------------------------


def _fma(a, b, c):
    """fp32 fused multiply-add: the product is exact in 64 bits."""
    return (a.double() * b.double() + c).float()


def _weights(d):
    """The framework's weight of a key d = key - max <= 0: e^d by its fixed polynomial, in fp32."""
    log2e, ln2_hi, ln2_lo = float.fromhex("0x1.715476p+0"), float.fromhex("0x1.62e43p-1"), float.fromhex("-0x1.05c61p-29")
    n = torch.round(d * np.float32(log2e).item())
    r = (d.double() - n.double() * ln2_hi).float()
    r = (r.double() - n.double() * ln2_lo).float()
    p = torch.full_like(r, float.fromhex("0x1.a01a02p-13"))
    p = _fma(p, r, float.fromhex("0x1.6c16c2p-10"))
    p = _fma(p, r, float.fromhex("0x1.111112p-7"))
    p = _fma(p, r, float.fromhex("0x1.555556p-5"))
    p = _fma(p, r, float.fromhex("0x1.555556p-3"))
    p = _fma(p, r, 0.5)
    p = _fma(p, r, 1.0)
    p = _fma(p, r, 1.0)
    w = torch.ldexp(p.double(), n.clamp(min=-200).double())
    return torch.where(d >= -87.0, w, 0.0)


def _scale_draw(u53, z):
    """floor(u53 * z / 2^53) in whole numbers (u53 < 2^53, z < 2^58)."""
    uh, ul = u53 >> 27, u53 & ((1 << 27) - 1)
    zh, zl = z >> 29, z & ((1 << 29) - 1)
    a, b, c, d = uh * zh, uh * zl, ul * zh, ul * zl
    low = ((b & ((1 << 26) - 1)) << 27) + ((c & ((1 << 24) - 1)) << 29) + d
    return a * 8 + (b >> 26) + (c >> 24) + (low >> 53)


def _plain_verify(st):
    x = st["logits"].float()
    rows, v = x.shape
    seq_of, off = st["seq_of"], st["offsets"].long()
    temp, top_k, top_p = (a[seq_of, None] for a in st["params_t"])
    greedy = temp[:, 0] == 0
    key = x / torch.where(temp == 0, 1.0, temp)
    q = torch.floor(_weights(key - key.amax(1, keepdim=True)) * 2.0**40).long()
    if st["sorted"]:
        sk, si = torch.sort(key, dim=1, descending=True, stable=True)
        sq = q.gather(1, si)
        k = torch.where((top_k > 0) & (top_k < v), top_k, v)
        sq = torch.where(sk >= sk.gather(1, k - 1), sq, 0)
        z = sq.sum(1, keepdim=True)
        m = (top_p.double() * 2.0**24).long()  # top_p in [0.5, 1]: 24 bits
        cut = m * (z >> 24) + ((m * (z & 0xFFFFFF)) >> 24)
        keep = (torch.cumsum(sq, 1) - sq <= cut) | (top_p >= 1.0)
        q = torch.zeros_like(q).scatter_(1, si, torch.where(keep, sq, 0))
    z = q.sum(1)
    ids = torch.arange(v, device=x.device)
    best = torch.where(x == x.amax(1, keepdim=True), ids, v).amin(1)
    row = torch.arange(rows, device=x.device)
    drafts, u, dp = st["drafts"], st["uniforms"], st["draft_probs"]
    px = q.gather(1, drafts[:, None])[:, 0]
    drow = row - seq_of
    if dp is None or not len(dp):
        d = torch.ones_like(u)
    else:
        d = dp[drow.clamp(max=len(dp) - 1), drafts].double()
    ok = torch.where(greedy, drafts == best, (u * d) * z.double() < px.double())
    stop = (row == off[seq_of + 1] - 1) | ~ok
    first = torch.full((len(off) - 1,), rows, device=x.device).scatter_reduce_(
        0, seq_of, torch.where(stop, row, rows), "amin")
    # the last token: from the residual at a rejected row, from the target itself at the last row
    p, zf, bonus = q[first], z[first], first == off[1:] - 1
    if dp is None or not len(dp):
        taken = torch.where(ids == drafts[first][:, None], p, 0)
    else:
        df = dp[drow[first].clamp(max=len(dp) - 1)].double()
        taken = torch.where(df > 0, torch.floor(df * zf.double()[:, None]), 0.0).long()
    res = torch.where(bonus[:, None], p, (p - taken).clamp(min=0))
    total = res.sum(1)
    res = torch.where(total[:, None] == 0, p, res)
    total = torch.where(total == 0, zf, total)
    t = _scale_draw((u[off[1:] - 1] * 2.0**53).long(), total)  # the last row's number draws
    tok = (torch.cumsum(res, 1) <= t[:, None]).sum(1)
    tok = torch.where(greedy[first], best[first], tok)
    here = first[seq_of]
    tokens = torch.where(row < here, drafts, torch.where(row == here, tok[seq_of], -1))
    return tokens, (first - off[:-1]).int()


def _plain_top(st):
    case = st["case"]
    x = st["logits"].float()
    # whole numbers in the order of (value descending, index ascending)
    bits = x.view(torch.int32).long()
    order = torch.where(x == 0, 0, torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits))
    order = (order << 32) - torch.arange(x.shape[1], device=x.device)
    idx = torch.topk(order, case["k"], dim=1).indices
    y = x / case["temperature"]
    m = y.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(y - m).sum(1, keepdim=True))
    return y.gather(1, idx) - lse, idx.int(), lse[:, 0]


def _plain_distill(st):
    case = st["case"]
    z, lp, idx = st["student"], st["lp"], st["idx"].long()
    y = z.float() / case["temperature"]
    there = idx >= 0
    at = idx.clamp(min=0)
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    lse = m + torch.log(e.sum(1, keepdim=True))
    zl = y.gather(1, at) - lse
    if case["tail"]:
        t = torch.where(there, torch.exp(lp), 0.0)
        rest = torch.where(there.any(1, keepdim=True), (1 - t.sum(1, keepdim=True)).clamp(min=0), 0.0)
        member = torch.zeros_like(y).scatter_reduce_(1, at, there.float(), "amax")
        out = torch.where(member > 0, 0.0, e)
        tail = out.sum(1, keepdim=True)
        rest = torch.where(tail > 0, rest, 0.0)
    else:
        lm = torch.where(there, lp, -math.inf).amax(1, keepdim=True).clamp(min=-3e38)
        t = torch.where(there, torch.exp(lp - lm), 0.0)
        t = t / t.sum(1, keepdim=True).clamp(min=1e-38)
        rest = torch.zeros_like(m)
    loss = torch.where(t > 0, t * (torch.log(t) - zl), 0.0).sum(1)
    if case["tail"]:
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - (m + torch.log(tail) - lse)), 0.0)[:, 0]
    w = st["weight"] if case["reduction"] == "sum" else torch.ones_like(loss)
    out_loss = (w * loss).sum() if case["reduction"] == "sum" else loss
    if not case["backward"]:
        return out_loss
    total = t.sum(1, keepdim=True) + rest
    grad = e * (total / e.sum(1, keepdim=True))
    if case["tail"]:
        grad -= out * torch.where(rest > 0, rest / tail, 0.0)
    grad.scatter_add_(1, at, torch.where(there, -t, 0.0))
    grad *= (st["weight"] / case["temperature"])[:, None]
    return out_loss, grad.to(z.dtype)


# ---- one pass ----------------------------------------------------------------------------------


def _own_distill(st):
    from pagedbatch_b200 import distill_loss

    case = st["case"]
    kw = dict(temperature=case["temperature"], tail=case["tail"], reduction=case["reduction"])
    if case["reduction"] == "sum":
        kw["row_weight"] = st["weight"]
    if not case["backward"]:
        with torch.no_grad():
            return distill_loss(st["student"], st["lp"], st["idx"], **kw)
    z = st["student"].detach().requires_grad_()
    loss = distill_loss(z, st["lp"], st["idx"], **kw)
    (grad,) = torch.autograd.grad(loss, z, None if case["reduction"] == "sum" else st["weight"])
    return loss.detach(), grad


def run(state):
    op = state["case"]["op"]
    if own:
        import pagedbatch_b200 as pb

        if op == "verify":
            return pb.verify(state["logits"], state["params"], state["drafts"], state["offsets"], state["uniforms"],
                             draft_probs=state["draft_probs"])
        if op == "top":
            return tuple(pb.top_logprobs(state["logits"], state["case"]["k"], temperature=state["case"]["temperature"]))
        return _own_distill(state)
    return {"verify": _plain_verify, "top": _plain_top, "distill": _plain_distill}[op](state)


# ---- the definition in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    """None for the verification, whose outputs are whole numbers."""
    if case["op"] == "verify":
        return None
    st = prepare(case, seed)
    if case["op"] == "top":
        y = st["logits"].double() / case["temperature"]
        lse = torch.logsumexp(y, 1, keepdim=True)
        return torch.topk(y, case["k"], dim=1).values - lse, None, lse[:, 0]
    y = st["student"].double() / case["temperature"]
    lp, idx = st["lp"].double(), st["idx"].long()
    n, k = idx.shape
    logs = torch.log_softmax(y, 1)
    row = torch.arange(n, device=y.device)[:, None].expand(n, k)
    used = idx >= 0
    # the teacher as a full row: probabilities of the entries, and for the tail one number a row
    target = torch.zeros_like(y)
    if case["tail"]:
        target[row[used], idx[used]] = lp[used].exp()
        rest = (1 - target.sum(1)).clamp(min=0) * used.any(1)
    else:
        target[row[used], idx[used]] = torch.softmax(torch.where(used, lp, -math.inf), 1)[used]
        rest = torch.zeros(n, dtype=torch.float64, device=y.device)
    loss = (torch.xlogy(target, target) - target * logs).sum(1)
    grad = logs.exp() * (target.sum(1) + rest)[:, None] - target
    if case["tail"]:
        outside = logs.clone()
        outside[row[used], idx[used]] = -math.inf
        log_tail = torch.logsumexp(outside, 1)
        loss += torch.xlogy(rest, rest) - rest * log_tail
        grad -= rest[:, None] * (outside - log_tail[:, None]).exp()
    out = (st["weight"].double() * loss).sum() if case["reduction"] == "sum" else loss
    if not case["backward"]:
        return out
    return out, grad * (st["weight"].double() / case["temperature"])[:, None]
