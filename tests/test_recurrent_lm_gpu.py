"""The language-model operators together, as the example runs them: training lowers the loss, and
answering token by token agrees with the training forward."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    from examples.recurrent_lm import RecurrentLM, train

    torch.manual_seed(0)
    model = RecurrentLM(32).cuda()
    losses = train(model, 40)
    # 30 tokens in 6 phrases: log 32 = 3.5 at the start; a phrase's next token is known once its first
    # two are, so about log(6) / 5 = 0.36 nats and the documents' starts remain
    assert losses[0] > 2.5 and losses[-1] < 1.3, losses
    return model


@torch.no_grad()
def test_answering_agrees_with_the_training_forward(model):
    """Greedy answers, and the logits behind them: the whole text through the training forward gives
    every position's logits to 1e-3 (the scan joins spans, the products split their sums
    otherwise), and the answered token is its largest."""
    from examples.recurrent_lm import Answerer, phrases

    n, steps = 5, 24
    prompt = phrases(n, 40, 32, 99)[0].cuda()
    answerer = Answerer(model, n, temperature=0.0)
    answer = answerer.answer(prompt, torch.zeros(steps, n, device="cuda"))
    text = torch.cat([prompt, answer], dim=1)
    reset = torch.zeros(text.shape, dtype=torch.bool, device="cuda")
    logits, _ = model(text, reset, torch.zeros(n, model.D, device="cuda"))
    at = logits[:, prompt.shape[1] - 1:-1]
    taken = at.gather(2, answer[..., None])[..., 0]
    assert bool((taken >= at.amax(dim=2) - 1e-3).all())
    torch.testing.assert_close(answerer.logits, logits[:, -2], rtol=1e-3, atol=1e-3)


@torch.no_grad()
def test_the_same_random_numbers_give_the_same_answer(model):
    from examples.recurrent_lm import Answerer, phrases

    n = 6
    prompt = phrases(n, 30, 32, 5)[0].cuda()
    u = torch.rand(12, n, device="cuda")
    settings = dict(temperature=0.9, top_k=10, top_p=0.9, min_p=0.01)
    first = Answerer(model, n, **settings).answer(prompt, u)
    again = Answerer(model, n, **settings)
    again.answer(prompt, torch.rand(3, n, device="cuda"))
    assert torch.equal(again.answer(prompt, u), first)
