"""The float64 oracle of the training step's operators against autograd, differences and closed forms."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training as R

F64 = torch.float64


def _rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def test_embedding_is_indexing_and_its_gradient_autograds():
    table = _rnd(6, 4).requires_grad_()
    tokens = torch.tensor([[0, 5, 5], [2, 0, 5]])
    d = _rnd(2, 3, 4, seed=1)
    out = table[tokens] * 1.5
    assert torch.equal(R.embed(tokens, table.detach(), 1.5), out.detach())
    grad, = torch.autograd.grad((out * d).sum(), table)
    got, size = R.embed_backward(tokens, d, 6, 1.5)
    torch.testing.assert_close(got, grad, rtol=1e-14, atol=1e-14)
    assert bool((size >= got.abs()).all())


def test_padding_has_a_row_of_zeros_and_no_gradient():
    table, tokens = _rnd(3, 2), torch.tensor([-1, 3, 1, 2 ** 40])
    assert torch.equal(R.embed(tokens, table)[[0, 1, 3]], torch.zeros(3, 2, dtype=F64))
    got, _ = R.embed_backward(tokens, torch.ones(4, 2), 3)
    assert got.sum() == 2 and bool((got[1] == 1).all())


def test_score_is_log_softmax():
    logits = (_rnd(5, 9) * 3).requires_grad_()
    tokens = torch.tensor([0, 8, 3, -1, 4])
    logp = torch.log_softmax(logits, dim=1)
    entropy = -(logp.exp() * logp).sum(1)
    got = R.score(logits.detach(), tokens, 9)
    want = torch.stack([logp[i, t] if t >= 0 else logp[i, 0] * 0 for i, t in enumerate(tokens.tolist())])
    torch.testing.assert_close(got[0], want.detach(), rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(got[1], entropy.detach(), rtol=1e-13, atol=1e-13)
    order = torch.sort(logits.detach(), dim=1, descending=True, stable=True).indices
    assert torch.equal(got[2], order)
    torch.testing.assert_close(got[3], logp.detach().gather(1, order), rtol=1e-13, atol=1e-13)
    g, h = _rnd(5, seed=2), _rnd(5, seed=3)
    grad, = torch.autograd.grad((want * g).sum() + (entropy * h).sum(), logits)
    torch.testing.assert_close(R.score_backward(logits.detach(), tokens, g, h), grad, rtol=1e-12, atol=1e-12)


def test_score_closed_forms():
    """Equal logits: log V each; a row of one logit: 0; a masked logit has no mass."""
    logits = torch.tensor([[2.0] * 8, [-math.inf] * 7 + [3.0], [0.0, 0.0] + [-math.inf] * 6,
                           [-math.inf] * 8])
    logprob, entropy, best, best_logprob = R.score(logits, torch.tensor([3, 7, 2, 0]), 3)
    torch.testing.assert_close(entropy, torch.tensor([math.log(8), 0.0, math.log(2), 0.0], dtype=F64))
    torch.testing.assert_close(logprob, torch.tensor([-math.log(8), 0.0, -math.inf, -math.inf], dtype=F64))
    assert best.tolist() == [[0, 1, 2], [7, -1, -1], [0, 1, -1], [-1, -1, -1]]
    assert best_logprob[3].tolist() == [-math.inf] * 3
    d = R.score_backward(logits, torch.tensor([3, 7, 2, 0]), torch.ones(4), torch.ones(4))
    assert not d[3].any() and not d[2, 2 + 1:].any()


@pytest.mark.parametrize("valid", [None, torch.tensor([True, False, True, True, True, False])])
def test_choice_against_autograd(valid):
    logits = (_rnd(6, 5, seed=4) * 2).requires_grad_()
    rows = torch.arange(6) if valid is None else torch.nonzero(valid)[:, 0]
    best, units = torch.topk(logits[rows], 2, dim=1)
    shares = torch.softmax(best, dim=1)
    counts = torch.bincount(units.reshape(-1), minlength=5)
    load = counts.to(F64) / counts.sum()  # (whole numbers divide to fp32)
    probs = torch.softmax(logits[rows], dim=1).mean(0)
    balance = 5 * (load * probs).sum()
    got = R.choose_units(logits.detach(), 2, valid)
    assert torch.equal(got[0][rows], units) and torch.equal(got[3], counts) and got[5] == len(rows)
    torch.testing.assert_close(got[1][rows], shares.detach(), rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(got[2], balance.detach(), rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(got[4], probs.detach(), rtol=1e-13, atol=1e-13)
    g = _rnd(6, 2, seed=5)
    grad, = torch.autograd.grad((shares * g[rows]).sum() + 0.3 * balance, logits)
    torch.testing.assert_close(R.choose_units_backward(logits.detach(), 2, g, 0.3, valid), grad,
                               rtol=1e-12, atol=1e-12)


def test_choice_closed_forms():
    """The balance is 1 where units are chosen alike, M where one takes all with certainty, 0 for none."""
    alike = torch.full((4, 4), -1e3) + 1e3 * torch.eye(4)
    assert abs(float(R.choose_units(alike, 1)[2]) - 1) < 1e-12
    one = torch.tensor([[1e3, 0.0, 0.0, 0.0]] * 5)
    assert abs(float(R.choose_units(one, 1)[2]) - 4) < 1e-12
    none = torch.full((3, 4), -math.inf)
    units, shares, balance, counts, probs, rows = R.choose_units(none, 2)
    assert bool((units == -1).all()) and not shares.any() and float(balance) == 0 and rows == 0
    ties = torch.tensor([[1.0, 2.0, 2.0, 2.0]])
    assert R.choose_units(ties, 2)[0].tolist() == [[1, 2]]
    few = torch.tensor([[-math.inf, 2.0, -math.inf, -math.inf]])
    assert R.choose_units(few, 2)[0].tolist() == [[1, -1]]


def test_norm_and_coefficient():
    grads = [torch.tensor([3.0, 0.0]), torch.tensor([[4.0]]), torch.zeros(0)]
    assert R.grad_norm(grads) == 5.0
    assert R.clip_coefficient(5.0, 10.0) == 1.0
    assert abs(R.clip_coefficient(5.0, 1.0) - 0.2) < 1e-6
    assert R.clip_coefficient(math.inf, 1.0) == 1.0 and R.clip_coefficient(math.nan, 1.0) == 1.0
