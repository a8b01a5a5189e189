"""Refusals of the drafted-decoding operators (CPU only): every argument is checked before any device
work, in Python and at the C ABI; and the oracle of the verification on small cases worked by hand."""

import numpy as np
import pytest
import torch

import oracle.verify
import pagedbatch_b200 as pb
from pagedbatch_b200 import SamplingParams, _lib, build, ops


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_cpu_tensors_are_refused():
    z = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        pb.top_logprobs(z, 2)
    with pytest.raises(ValueError, match="CUDA"):
        pb.distill_loss(z, torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32))
    rec = torch.zeros(64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        pb.verify(z, rec, torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.float64))


def test_verify_tokens_checks_its_lists():
    p, g = SamplingParams(), torch.Generator()
    z = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="params"):
        pb.verify_tokens(z, [[1, 2]], [], [g])
    with pytest.raises(ValueError, match="rows"):
        pb.verify_tokens(z, [[1]], [p], [g])
    with pytest.raises(ValueError, match=r"\[0, 8\)"):
        pb.verify_tokens(z, [[1, 8]], [p], [g])
    with pytest.raises(ValueError, match=r"\[0, 8\)"):
        pb.verify_tokens(z, [[-1, 0]], [p], [g])
    with pytest.raises(ValueError, match="logits"):
        pb.verify_tokens(z[0], [[1, 2]], [p], [g])
    bad = SamplingParams()
    bad.top_k = -1
    with pytest.raises(ValueError, match="top_k"):
        pb.verify_tokens(z, [[1, 2]], [bad], [g])


class _Fake:
    """A tensor that says it is on a CUDA device, for the checks that come after that one."""

    def __init__(self, t):
        self._t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


def test_shapes_and_types_are_refused():
    z = _Fake(torch.zeros(3, 8))
    rec = ops.mark_rows(torch.from_numpy(ops.pack_params([1.0], [1.0], [0], [0.0]).view(np.uint8).copy()),
                        ops.pack_params([1.0], [1.0], [0], [0.0]))
    d, o, u = torch.zeros(3, dtype=torch.int64), torch.tensor([0, 3], dtype=torch.int32), torch.zeros(3, dtype=torch.float64)
    from pagedbatch_b200 import distill, logprobs, speculative

    for bad in (dict(d=d[:2]), dict(d=d.int()), dict(o=o[:1]), dict(o=o.long()), dict(u=u.float()), dict(u=u[:1]),
                dict(rec=rec[:7]), dict(rec=rec.view(torch.int8)), dict(p=torch.zeros(1, 8)), dict(p=torch.zeros(2, 7)),
                dict(p=torch.zeros(2, 8, dtype=torch.float64)), dict(p=torch.zeros(8, 2).T),
                dict(z=_Fake(torch.zeros(3, 8, dtype=torch.float64))), dict(z=_Fake(torch.zeros(8, 3).T)),
                dict(z=_Fake(torch.zeros(3)))):
        a = dict(z=z, rec=rec, d=d, o=o, u=u, p=None) | bad
        with pytest.raises(ValueError):
            speculative._launch(a["z"], a["rec"], a["d"], a["o"], a["u"], a["p"])
    for k, t in ((0, 1.0), (9, 1.0), (257, 1.0), (-1, 1.0), (2, 0.0), (2, -1.0), (2, float("nan")), (2, float("inf")), (2, 1e-9)):
        with pytest.raises(ValueError):
            logprobs._launch(z, k, t)
    with pytest.raises(ValueError):
        logprobs._launch(_Fake(torch.zeros(8, 3).T), 2, 1.0)
    lp, idx = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    for a, kw in (((lp[:2], idx), {}), ((lp, idx[:, :1]), {}), ((lp, idx.short()), {}), ((lp.double(), idx), {}),
                  ((lp.requires_grad_(), idx), {}), ((torch.zeros(3, 1025), torch.zeros(3, 1025, dtype=torch.int32)), {}),
                  ((torch.zeros(3, 0), torch.zeros(3, 0, dtype=torch.int32)), {}),
                  ((torch.zeros(3, 2), idx), dict(temperature=0.0)), ((torch.zeros(3, 2), idx), dict(reduction="mean")),
                  ((torch.zeros(3, 2), idx), dict(row_weight=torch.ones(2))),
                  ((torch.zeros(3, 2), idx), dict(row_weight=torch.ones(3).double())),
                  ((torch.zeros(3, 2), idx), dict(row_weight=torch.ones(3).requires_grad_()))):
        with pytest.raises(ValueError):
            distill.distill_loss(z, *a, **kw)


def test_c_abi_refusals(lib):
    b = np.zeros(4096, np.uint8)
    base = (b.ctypes.data + 255) & ~255  # an address that passes the alignment checks; nothing reads it

    def verify(**kw):
        a = dict(logits=base, dtype=0, n_rows=2, vocab=8, stride=8, params=base, n_seqs=1, offsets=base, drafts=base,
                 uniforms=base, probs=None, pdtype=0, n_probs=1, pstride=8, kinds=0, tokens=base, accepted=base, status=None,
                 ws=base, ws_bytes=lib.pb_verify_ws_bytes(2, 1, 8, 0, 0), stream=None) | kw
        return lib.pb_verify(*a.values())

    for kw in (dict(dtype=9), dict(n_rows=-1), dict(vocab=0), dict(stride=7), dict(logits=None), dict(params=None),
               dict(offsets=None), dict(drafts=None), dict(uniforms=None), dict(tokens=None), dict(accepted=None),
               dict(ws=None), dict(ws=base + 8), dict(ws_bytes=0), dict(n_seqs=0), dict(n_seqs=3), dict(kinds=16),
               dict(kinds=-1), dict(probs=base, pdtype=5), dict(probs=base, pstride=7), dict(probs=base + 1),
               dict(logits=base + 2)):
        assert verify(**kw) == -1, kw
    assert verify(vocab=1 << 24, stride=1 << 24) == -2
    assert verify(n_rows=0, n_seqs=0) == 0
    assert lib.pb_verify_ws_bytes(-1, 1, 8, 0, 0) == -1 and lib.pb_verify_ws_bytes(1, 1, 8, 7, 0) == -1 and lib.pb_verify_ws_bytes(1, 1, 8, 0, 16) == -1

    def top(**kw):
        a = dict(logits=base, dtype=0, n_rows=2, vocab=8, stride=8, k=2, t=1.0, lp=base, idx=base, lse=base, ws=base, ws_bytes=1 << 20, stream=None) | kw
        return lib.pb_top_logprobs(*a.values())

    for kw in (dict(dtype=9), dict(n_rows=-1), dict(vocab=0), dict(stride=-1), dict(k=0), dict(k=9), dict(vocab=999, k=257),
               dict(t=0.0), dict(t=float("nan")), dict(t=float("inf")), dict(logits=None), dict(lp=None), dict(idx=None),
               dict(lse=None), dict(logits=base + 1), dict(ws=None), dict(ws=base + 16), dict(ws_bytes=64)):
        assert top(**kw) == -1, kw
    assert top(vocab=1 << 24) == -2 and top(n_rows=0, logits=None) == 0

    def forward(**kw):
        a = dict(z=base, dtype=0, n=2, vocab=8, stride=8, lp=base, ls=2, idx=base, xs=2, xb=4, k=2, t=1.0, tail=0, w=None,
                 loss=base, stats=base, ws=base, ws_bytes=1 << 20, stream=None) | kw
        return lib.pb_distill_forward(*a.values())

    def backward(**kw):
        a = dict(z=base, dtype=0, n=2, vocab=8, stride=8, lp=base, ls=2, idx=base, xs=2, xb=4, k=2, t=1.0, w=None,
                 stats=base, grad=base, gs=1, dz=base, stream=None) | kw
        return lib.pb_distill_backward(*a.values())

    common = (dict(dtype=9), dict(n=-1), dict(vocab=0), dict(stride=-1), dict(ls=-1), dict(xs=-1), dict(xb=2), dict(k=0),
              dict(k=1025), dict(t=0.0), dict(t=float("nan")), dict(z=None), dict(lp=None), dict(idx=None), dict(stats=None),
              dict(stats=base + 4), dict(z=base + 1), dict(lp=base + 2), dict(idx=base + 4, xb=8))
    for kw in (*common, dict(loss=None), dict(ws=None), dict(ws=base + 8), dict(ws_bytes=0)):
        assert forward(**kw) == -1, kw
    for kw in (*common, dict(grad=None), dict(dz=None), dict(gs=-1), dict(dz=base + 2)):
        assert backward(**kw) == -1, kw
    assert forward(vocab=(1 << 20) + 1) == -2 and backward(vocab=(1 << 20) + 1) == -2
    assert forward(n=0, z=None) == 0 and backward(n=0, z=None) == 0
    assert lib.pb_distill_ws_bytes(1, 8, 9) == -1 and lib.pb_distill_ws_bytes(1, (1 << 20) + 1, 0) == -1
    assert lib.pb_top_ws_bytes(1, 8, 9) == -1 and lib.pb_top_ws_bytes(-1, 8, 0) == -1
    assert lib.pb_distill_sum(None, 1, base, None) == -1 and lib.pb_distill_sum(base, 1, None, None) == -1
    assert lib.pb_distill_stats_bytes(-1) == -1 and lib.pb_distill_stats_bytes(3) == 96


def test_misaligned_arrays_are_refused(lib):
    """Arrays that do not start on their elements' size, as a slice of a byte buffer may."""
    b = np.zeros(4096, np.uint8)
    base = (b.ctypes.data + 255) & ~255  # nothing reads it
    ws = lib.pb_verify_ws_bytes(2, 1, 8, 0, 0)
    ok = [base, 0, 2, 8, 8, base, 1, base, base, base, None, 0, 1, 8, 0, base, base, None, base, ws, None]
    for at, off in ((5, 1), (5, 4), (7, 2), (8, 4), (9, 4), (15, 4), (16, 1), (17, 2)):
        a = list(ok)
        a[at] = base + off
        assert lib.pb_verify(*a) == -1, at
    ok = [base, 0, 2, 8, 8, 2, 1.0, base, base, base, base, 1 << 20, None]
    for at in (7, 8, 9):
        a = list(ok)
        a[at] = base + 2
        assert lib.pb_top_logprobs(*a) == -1, at
    ok = [base, 0, 2, 8, 8, base, 2, base, 2, 4, 2, 1.0, 0, None, base, base, base, 1 << 20, None]
    for at in (5, 7, 13, 14, 15, 16):
        a = list(ok)
        a[at] = base + 2
        assert lib.pb_distill_forward(*a) == -1, at
    ok = [base, 0, 2, 8, 8, base, 2, base, 2, 4, 2, 1.0, None, base, base, 1, base, None]
    for at in (5, 7, 12, 13, 14, 16):
        a = list(ok)
        a[at] = base + 2
        assert lib.pb_distill_backward(*a) == -1, at
    assert lib.pb_distill_sum(base + 2, 2, base, None) == -1 and lib.pb_distill_sum(base, 2, base + 1, None) == -1


def test_kinds_of_sequences():
    def kinds(t, p, k):
        return ops.row_kinds(ops.pack_params(t, p, k, [0.0] * len(t)))

    assert kinds([0.0, 1.0], [1.0, 0.9], [0, 50]) == (_lib.VERIFY_SMALL, 50)
    assert kinds([1.0], [1.0], [0]) == (_lib.VERIFY_WHOLE, 0)
    assert kinds([1.0], [1.0 - 1e-12], [0]) == (_lib.VERIFY_WHOLE, 0)  # rounds to 1 in fp32: no filter
    assert kinds([1.0], [0.9], [0]) == (_lib.VERIFY_TOPP, 0)
    assert kinds([1.0], [1.0], [129]) == (_lib.VERIFY_OTHER, 129)
    assert kinds([0.0, 1.0, 1.0, 1.0], [1.0, 1.0, 0.5, 1.0], [0, 0, 0, 500]) == (_lib.VERIFY_ANY, 500)
    assert kinds([-1.0], [1.0], [0])[0] == _lib.VERIFY_OTHER


def test_oracle_by_hand():
    """Two tokens of weights 2^40 and about 2^39: acceptance at the quotient of the probabilities, the
    residual's only token, and the fallback to the target."""
    x = torch.tensor([[0.0, -np.log(2.0)]] * 2, dtype=torch.float32)
    p1 = 1 / 3
    for u, ok in ((p1 * 0.99, True), (p1 * 1.01, False)):
        tok, acc, st = oracle.verify.verify(x, [(1.0, 1.0, 0)], [1], [1, 0], [u, 0.0])
        assert acc[0] == int(ok) and tok[0] == (1 if ok else 0) and st[0] == 0
    # the draft model gives token 1 half: accepted up to p / d = 2 / 3
    d = np.array([[0.5, 0.5]], np.float32)
    for u, ok in ((0.66, True), (0.67, False)):
        tok, acc, _ = oracle.verify.verify(x, [(1.0, 1.0, 0)], [1], [1, 0], [u, 0.99], d)
        assert acc[0] == int(ok) and tok[0] == (1 if ok else 0)
    # a draft distribution above the target everywhere leaves no residual: the target is drawn from
    d = np.array([[1.0, 1.0]], np.float32)
    for u, t in ((0.6, 0), (0.7, 1)):
        assert oracle.verify.verify(x, [(1.0, 1.0, 0)], [1], [1, 0], [0.9, u], d)[0][0] == t
