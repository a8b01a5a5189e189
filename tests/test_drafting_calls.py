"""What the calls of drafted decoding do on the host (CPU only)."""

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import pagedbatch_b200 as pb
from pagedbatch_b200 import SamplingParams, _lib, build, ops


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _records():
    return ops.pack_params([0.0, 1.0, 1.0], [1.0, 0.9, 1.0], [0, 50, 0], np.zeros(3))


def test_the_sampler_does_not_look_for_kinds_of_sequences(monkeypatch):
    """Uploads and marks of the sampler's records, made every step, leave the verification's note to it; the
    note is of the records as they were."""
    asked = []
    kinds = ops.row_kinds
    monkeypatch.setattr(ops, "row_kinds", lambda rec: asked.append(1) or kinds(rec))
    rec = _records()
    ops.mark_rows(torch.from_numpy(rec.view(np.uint8).copy()), rec)
    params = ops.params_tensor(rec, "cpu", pinned=False)
    assert not asked
    rec["top_k"] = 0
    for _ in range(2):
        assert ops.noted_kinds(params) == (_lib.VERIFY_SMALL | _lib.VERIFY_WHOLE, 50)
    assert len(asked) == 1
    assert ops.noted_kinds(params.clone()) == (0, 0)


@pytest.mark.parametrize("inference", [False, True])
def test_records_written_to_are_known_as_such(inference):
    with torch.inference_mode(inference):
        params = ops.params_tensor(_records(), "cpu", pinned=False)
        assert ops.unchanged(params)
        assert not ops.unchanged(params.clone())
        params[32:64].zero_()
        assert not ops.unchanged(params)
    assert not ops.unchanged(params)


def test_kinds_beside_others(lib):
    """PB_VERIFY_REST goes with some kind, and needs no more memory than the kinds do."""
    for kinds in range(1, 16):
        assert lib.pb_verify_ws_bytes(7, 3, 1000, 1, kinds | _lib.VERIFY_REST) == lib.pb_verify_ws_bytes(7, 3, 1000, 1, kinds)
    for kinds in (_lib.VERIFY_REST, 32, 32 | 1, -16):
        assert lib.pb_verify_ws_bytes(7, 3, 1000, 1, kinds) == -1


def test_refused_calls_leave_the_generators(monkeypatch):
    """verify_tokens draws random numbers when every check is behind it, the device's among them."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    g = [torch.Generator().manual_seed(s) for s in range(2)]
    before = [x.get_state() for x in g]
    params, drafts, z = [SamplingParams()] * 2, [[1], [2, 3]], torch.zeros(5, 8)
    ok = torch.zeros(3, 8)
    for logits, probs, error in ((z, ok[:2], ValueError), (z, ok[:, :7], ValueError), (z, ok.double(), ValueError),
                                 (z, torch.zeros(8, 3).T, ValueError), (z, ok[0], ValueError), (z.double(), None, ValueError),
                                 (z, ok, RuntimeError), (z, None, RuntimeError)):
        with pytest.raises(error):
            pb.verify_tokens(logits, drafts, params, g, draft_probs=probs)
        assert all(torch.equal(a, b.get_state()) for a, b in zip(before, g, strict=True))


def test_fake_tensors():
    """Shapes and types of the results without data, and the same refusals."""
    with FakeTensorMode():
        z = torch.empty(5, 100, device="cuda", dtype=torch.bfloat16)
        lp, idx, lse = pb.top_logprobs(z, 7, temperature=0.5)
        assert lp.shape == idx.shape == (5, 7) and lse.shape == (5,)
        assert (lp.dtype, idx.dtype, lse.dtype) == (torch.float32, torch.int32, torch.float32) and lp.is_cuda
        with pytest.raises(ValueError, match="k must be"):
            pb.top_logprobs(z, 101)
        params = torch.empty(64, dtype=torch.uint8, device="cuda")
        d, u = torch.empty(5, dtype=torch.int64, device="cuda"), torch.empty(5, dtype=torch.float64, device="cuda")
        off = torch.empty(3, dtype=torch.int32, device="cuda")
        for probs in (None, torch.empty(3, 100, device="cuda")):
            tok, acc, st = pb.verify(z, params, d, off, u, draft_probs=probs, with_status=True)
            assert tok.shape == (5,) and acc.shape == st.shape == (2,)
            assert (tok.dtype, acc.dtype, st.dtype) == (torch.int64, torch.int32, torch.int32)
            assert len(pb.verify(z, params, d, off, u, draft_probs=probs)) == 2
        with pytest.raises(ValueError, match="draft_probs"):
            pb.verify(z, params, d, off, u, draft_probs=torch.empty(2, 100, device="cuda"))
        z.requires_grad_()
        for reduction, shape in (("none", (5,)), ("sum", ())):
            loss = pb.distill_loss(z, lp, idx, reduction=reduction, row_weight=torch.empty(5, device="cuda"))
            assert loss.shape == shape and loss.dtype == torch.float32
            assert loss.requires_grad


def test_ops_refuse_what_the_calls_refuse():
    """The registered ops check their arguments themselves."""
    op, back = torch.ops.pagedbatch_b200.distill_loss, torch.ops.pagedbatch_b200.distill_loss_backward
    with FakeTensorMode():
        z, lp, w = (torch.empty(s, device="cuda") for s in ((3, 50), (3, 4), (3,)))
        idx = torch.empty(3, 4, dtype=torch.int32, device="cuda")
        stats, g = torch.empty(96, dtype=torch.uint8, device="cuda"), torch.empty(3, device="cuda")
        ok = dict(z=z, lp=lp, idx=idx, w=w, t=1.0)
        for bad in (dict(lp=lp[:2]), dict(idx=idx[:, :2]), dict(idx=idx.short()), dict(w=w[:1]), dict(t=0.0), dict(z=z.double()),
                    dict(z=torch.empty(50, 3, device="cuda").T), dict(lp=torch.empty(3, 4))):
            a = list((ok | bad).values())
            with pytest.raises(ValueError):
                op(*a, False, False)
            with pytest.raises(ValueError):
                back(*a[:4], stats, a[4], g)
        for st, gr in ((stats[:64], g), (stats.float(), g), (stats, g[:1]), (stats, g.double()), (stats, g[None])):
            with pytest.raises(ValueError):
                back(z, lp, idx, w, st, 1.0, gr)
        assert back(z, lp, idx, None, stats, 1.0, g[0]).shape == z.shape


def test_workspace_of_small_vocabularies(lib):
    """What top-p sequences need of a row's step is no more than the row."""
    for V in (1, 48, 1000, 5000):
        more = lib.pb_verify_ws_bytes(4096, 64, V, 0, _lib.VERIFY_TOPP) - lib.pb_verify_ws_bytes(4096, 64, V, 0, _lib.VERIFY_OTHER)
        assert more == 4096 * 8 * (512 + min(V, 2048))
