"""What the calls of drafted decoding do on the host (CPU only)."""

import numpy as np
import pytest
import torch

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
