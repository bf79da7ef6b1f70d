"""Sizes that the C entry points' 32-bit arguments do not hold: refused, not cut to their lower bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("helper", [True, False])
def test_sizes_past_31_bits_are_refused(cuda_device, monkeypatch, helper):
    from hsn_amd import sampling, scan

    if not helper:
        for module in (scan, sampling):
            monkeypatch.setattr(module, "native_calls", lambda *names: None)
    many = 2 ** 32 + 2  # whose lower 32 bits are 2
    y = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device=cuda_device)
    rows, long = y.expand(many, 1, 1), y.expand(1, many, 1)
    marks = torch.zeros(1, 1, 1, device=cuda_device)
    for t in (rows, long):
        with pytest.raises(ValueError, match="2\\^31"):
            scan.forward(t, t)
        with pytest.raises(ValueError, match="2\\^31"):
            scan.backward(t, t, marks, None, t)
    with pytest.raises(ValueError, match="2\\^31"):
        scan.step(rows[:, 0], rows[:, 0], marks[0])
    with pytest.raises(ValueError, match="2\\^31"):
        sampling.sample(rows[:, 0], marks[0, 0])
    pool = torch.empty(2 ** 31, 1, device=cuda_device)
    with pytest.raises(ValueError, match="2\\^31"):
        scan.step(y[0], y[0], pool, rows=torch.zeros(1, dtype=torch.int32, device=cuda_device))
