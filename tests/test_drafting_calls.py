"""What the calls of drafted decoding do on the host (CPU only)."""

import numpy as np
import torch

from pagedbatch_b200 import _lib, ops


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
