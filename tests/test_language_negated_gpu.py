"""Views whose memory holds the negated values, given to the scan, the unit layer and the sampling: refused by name, and
resolved where they are a node's cotangents."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _negated(*shape):
    """A float32 view that counts as its memory's negative; elements of a last dimension of one are dense."""
    t = torch.complex(torch.ones(shape), torch.ones(shape)).cuda().conj().imag
    assert t.is_neg() and t.dtype == torch.float32 and bool((t == -1).all())
    return t


@pytest.mark.parametrize("helper", [True, False])
def test_negated_views_are_refused(cuda_device, monkeypatch, helper):
    from hsn_amd import sampling, scan, unit_layer

    if not helper:
        for module in (sampling, scan, unit_layer):
            monkeypatch.setattr(module, "native_calls", lambda *names: None)
    y = torch.ones(2, 5, 1, device=cuda_device)
    marks = scan.forward(y, y)["marks"]
    state = torch.zeros(2, 1, device=cuda_device)
    x, router, W = (torch.ones(s, device=cuda_device) for s in ((3, 1), (2, 1), (2, 1, 1)))
    calls = [lambda: scan.forward(_negated(2, 5, 1), y), lambda: scan.forward(y, _negated(2, 5, 1)),
             lambda: scan.backward(y, y, marks, None, _negated(2, 5, 1)),
             lambda: scan.step(_negated(2, 1), state.clone(), state),
             lambda: unit_layer.unit_layer(_negated(3, 1), router, W, None, W, None, 1),
             lambda: sampling.sample(_negated(3, 1), torch.zeros(3, device=cuda_device)),
             lambda: sampling.sample(torch.zeros(1, 4, device=cuda_device), _negated(1))]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="negated"):
            call()
            pytest.fail(f"call {i} is not refused")


def test_a_negated_cotangent_of_the_scan(cuda_device):
    from hsn_amd import scan

    g = torch.Generator().manual_seed(0)
    y = torch.randn(2, 7, 1, generator=g).cuda().requires_grad_()
    gate = torch.randn(2, 7, 1, generator=g).cuda()

    class Negate(torch.autograd.Function):
        """The same values, whose cotangent comes negated."""

        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, d):
            d = torch.complex(torch.zeros_like(d), -d).conj().imag
            assert d.is_neg()
            return d

    for which in (0, 1):
        a, = torch.autograd.grad(Negate.apply(scan.gated_scan(y, gate)[which]).square().sum(), y)
        b, = torch.autograd.grad(scan.gated_scan(y, gate)[which].square().sum(), y)
        assert torch.equal(a, b) and bool(a.any())
