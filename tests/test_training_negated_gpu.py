"""Views whose memory holds the negated values (the imaginary part of a conjugated tensor): the kernels read memory,
so the training step's operators refuse them by name."""

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
    from hsn_amd import embedding, grad_clip, scoring, unit_router

    if not helper:
        for module in (embedding, grad_clip, scoring, unit_router):
            monkeypatch.setattr(module, "native_calls", lambda *names: None)
    tokens = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    logits = torch.zeros(4, 10, device=cuda_device)
    stats = scoring.forward(logits, tokens)["stats"]
    out = unit_router.forward(logits, 1)
    one = torch.ones(4, 1, device=cuda_device)
    calls = [lambda: scoring.forward(_negated(4, 1), tokens),
             lambda: scoring.backward(logits, tokens, stats, _negated(4)),
             lambda: scoring.backward(logits, tokens, stats, None, _negated(4)),
             lambda: embedding.forward(tokens, _negated(3, 1)),
             lambda: embedding.backward(tokens, _negated(4, 1), 3),
             lambda: unit_router.forward(_negated(4, 1), 1),
             lambda: unit_router.backward(logits, out["units"], out["tally"], _negated(4, 1)),
             lambda: unit_router.backward(logits, out["units"], out["tally"], one, _negated()),
             lambda: grad_clip.norm([one, _negated(1)]),
             lambda: grad_clip.clip([_negated(1)], 1.0),
             lambda: grad_clip.clip([torch.ones(1, device=cuda_device)], 1.0, out=[_negated(1)])]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="negated"):
            call()
            pytest.fail(f"call {i} is not refused")
    # resolved, they are tensors like others
    d = scoring.backward(logits, tokens, stats, _negated(4).resolve_neg())
    assert torch.equal(d, scoring.backward(logits, tokens, stats, -torch.ones(4, device=cuda_device)))


def test_negated_cotangents_of_the_nodes(cuda_device):
    """A cotangent that reaches a node through complex numbers may be such a view."""
    from hsn_amd import embedding, scoring, unit_router

    g = torch.Generator().manual_seed(0)
    logits = torch.randn(4, 10, generator=g).cuda().requires_grad_()
    tokens = torch.arange(4, device=cuda_device)
    met = []

    def through(real):
        """The same values, whose cotangent comes negated."""
        real.register_hook(lambda d: met.append(d.is_neg()))
        return Negate.apply(real)

    class Negate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, d):
            return torch.complex(torch.zeros_like(d), -d).conj().imag

    def check(loss, leaf):
        a, = torch.autograd.grad(loss(through), leaf)
        b, = torch.autograd.grad(loss(lambda t: t), leaf)
        assert torch.equal(a, b) and bool(a.any())

    check(lambda f: f(scoring.token_logprobs(logits, tokens)[0]).sum(), logits)
    check(lambda f: f(scoring.token_logprobs(logits, tokens)[1]).sum(), logits)
    check(lambda f: f(unit_router.choose_units(logits, 3)[1]).square().sum(), logits)
    check(lambda f: f(unit_router.choose_units(logits, 3)[2]), logits)
    table = torch.randn(10, 1, generator=g).cuda().requires_grad_()
    check(lambda f: f(embedding.embed(tokens, table)).sum(), table)
    assert met == [True] * 5
