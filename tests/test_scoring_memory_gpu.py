"""What the scoring's node allocates: of logits whose rows have one distance nothing of their size but the gradient."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_next_tokens_without_a_copy(cuda_device):
    """All positions with the tokens moved up and -1 behind the last: the slice's values and gradient, without the
    slice's copies."""
    from hsn_amd import scoring

    B, T, V = 8, 129, 32001
    g = torch.Generator("cuda").manual_seed(0)
    leaf = torch.randn(B, T, V, generator=g, device=cuda_device).to(torch.bfloat16).requires_grad_()
    tokens = torch.randint(0, V, (B, T), generator=g, device=cuda_device)
    moved = torch.cat([tokens[:, 1:], torch.full((B, 1), -1, device=cuda_device)], dim=1)
    size = B * T * V * 2

    def peak(f):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = f()
        return out, torch.cuda.max_memory_allocated() - before

    (logprob, entropy), more = peak(lambda: scoring.token_logprobs(leaf, moved))
    assert more < size // 16
    weight = torch.rand(B, T, generator=g, device=cuda_device)
    (grad,), more = peak(lambda: torch.autograd.grad((logprob * weight).sum(), leaf))
    assert more < size + size // 16
    assert not logprob[:, -1].any() and not grad[:, -1].any()
    sliced, _ = scoring.token_logprobs(leaf[:, :-1], tokens[:, 1:])
    # the copy's rows lie elsewhere, so their sums' order differs: within 2 (2^-22) of 16 at most
    assert bool(((logprob[:, :-1] - sliced).abs() <= 2.0 ** -17).all())
    other, = torch.autograd.grad((sliced * weight[:, :-1]).sum(), leaf)
    # a probability by 2 (2^-21 + 2^-23 16) of itself, and half a step of bf16 each
    off = (grad.double() - other.double()).abs()
    assert bool((off <= other.double().abs() * (2.0 ** -17 + 2.0 ** -7)).all())
