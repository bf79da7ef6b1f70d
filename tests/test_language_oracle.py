"""The float64 oracle of the language-model operators against autograd, differences and closed
forms (CPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import language as L

F64 = torch.float64


def _scan_problem(B=2, T=7, D=3, seed=0, resets=True):
    g = torch.Generator().manual_seed(seed)
    y, gate, d_h = (torch.randn(B, T, D, generator=g, dtype=F64) for _ in range(3))
    h0, d_h_T = (torch.randn(B, D, generator=g, dtype=F64) for _ in range(2))
    reset = (torch.rand(B, T, generator=g) < 0.3) if resets else None
    return y, gate, reset, h0, d_h, d_h_T


@pytest.mark.parametrize("candidate", ["tanh", "linear"])
@pytest.mark.parametrize("resets", [False, True])
def test_scan_gradient_is_autograds_and_the_differences(candidate, resets):
    y, gate, reset, h0, d_h, d_h_T = _scan_problem(resets=resets)
    leaves = [t.clone().requires_grad_() for t in (y, gate, h0)]

    def loss(y, gate, h0):
        c = torch.tanh(y) if candidate == "tanh" else y
        b = torch.sigmoid(gate)
        now, total = h0, 0.0
        for t in range(y.shape[1]):
            if reset is not None:
                now = now * (~reset[:, t, None])
            now = now + b[:, t] * (c[:, t] - now)
            total = total + (d_h[:, t] * now).sum()
        return total + (d_h_T * now).sum()

    want = torch.autograd.grad(loss(*leaves), leaves)
    got = L.scan_backward(y, gate, reset, h0, d_h, d_h_T, candidate)
    for w, g in zip(want, got):
        torch.testing.assert_close(g, w, rtol=1e-12, atol=1e-12)
    # central differences of the loss in a few places: error h^2 ~ 1e-10 and rounding 1e-16 / h
    step = 1e-5
    for k, at in ((0, (1, 2, 1)), (1, (0, 0, 2)), (2, (1, 0))):
        ends = []
        for sign in (1, -1):
            moved = [t.clone() for t in (y, gate, h0)]
            moved[k][at] += sign * step
            ends.append(float(loss(*moved)))
        assert abs((ends[0] - ends[1]) / (2 * step) - float(got[k][at])) < 1e-8


def test_scan_closed_forms():
    """A constant gate of 0 halves the distance to the candidate at every position; a reset starts
    from zero; the step is the scan's position."""
    y = torch.full((1, 5, 2), 0.75, dtype=F64)
    h, h_T = L.scan_forward(y, torch.zeros_like(y), h0=torch.zeros(1, 2, dtype=F64),
                            candidate="linear")
    want = 0.75 * (1 - 0.5 ** torch.arange(1, 6, dtype=F64))
    torch.testing.assert_close(h[0, :, 0], want, rtol=1e-14, atol=0)
    reset = torch.tensor([[False, False, False, True, False]])
    again, _ = L.scan_forward(y, torch.zeros_like(y), reset, candidate="linear")
    torch.testing.assert_close(again[0, 3:, 0], want[:2], rtol=1e-14, atol=0)
    step, pool = L.scan_step(y[:, 0].expand(3, 2), torch.zeros(3, 2), torch.ones(4, 2),
                             torch.tensor([2, -1, 0]), torch.tensor([False, False, True]),
                             "linear")
    assert step.tolist() == [[0.875] * 2, [0.0] * 2, [0.375] * 2]
    assert pool.tolist() == [[0.375] * 2, [1.0] * 2, [0.875] * 2, [1.0] * 2]


def test_unit_layer_is_the_dense_sum_where_every_unit_is_chosen():
    g = torch.Generator().manual_seed(3)
    M, d, H, n = 4, 5, 6, 3
    x, router = torch.randn(n, d, generator=g, dtype=F64), torch.randn(M, d, generator=g, dtype=F64)
    W1 = torch.randn(M, d, H, generator=g, dtype=F64)
    W2 = torch.randn(M, H, d, generator=g, dtype=F64)
    got = L.unit_layer(x, router, W1, None, W2, None, M)
    share = torch.softmax(x @ router.t(), dim=1)
    hidden = torch.nn.functional.gelu(torch.einsum("nd,mdh->nmh", x, W1))
    want = torch.einsum("nmh,mhd,nm->nd", hidden, W2, share)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)


def test_unit_layer_ties_go_to_the_lowest_unit():
    x = torch.ones(1, 2)
    router = torch.ones(3, 2)
    W1 = torch.zeros(3, 2, 1)
    b1 = torch.full((3, 1), 2.0)
    W2 = torch.tensor([1.0, 10.0, 100.0]).view(3, 1, 1)
    got = L.unit_layer(x, router, W1, b1, W2, None, 2)
    act = 0.5 * 2 * (1 + math.erf(math.sqrt(2)))
    assert abs(float(got) - 0.5 * act * 11) < 1e-12


def test_kept_tokens():
    logits = torch.tensor([math.log(v) for v in (0.1, 0.4, 0.2, 0.3)])
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 0, 1.0, 0.0)] == [1, 3, 2, 0]
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 2, 1.0, 0.0)] == [1, 3]
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 0, 0.6, 0.0)] == [1, 3]
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 3, 0.8, 0.0)] == [1, 3, 2]
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 0, 1.0, 0.6)] == [1, 3]
    assert [j for j, _ in L.kept_tokens(logits, 1.0, 0, 0.0, 2.0)] == [1]
    equal = torch.zeros(5)
    assert [j for j, _ in L.kept_tokens(equal, 1.0, 3, 1.0, 0.0)] == [0, 1, 2]
    assert L.sample(equal, 0.5)[0] == 2
    assert L.sample(torch.tensor([-math.inf, 1.0, math.nan, 1.0]), 0.9, 0.0)[0] == 1
    assert L.sample(torch.full((3,), -math.inf), 0.3) == (-1, 1.0)
