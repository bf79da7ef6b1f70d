"""Scoring in every way in which a launch divides long rows and many rows, with several batches of a row to a
thread, against the oracle and float64.

Bars, with u = 2^-24 and x = l - max l: an exponential is off by (3 |x| + 4) u of itself (the difference, its product
with log2 e and the constant, the instruction's 2 u). A sum of a batch is off by 7 u of itself (three steps of
pairs or four of a chain, two of packs, two to spare), a thread's sums of batches are float64. 64 threads' sums are
rounded to fp32 and joined by 6 steps, 4 or 16 waves' by 2 or 4 and up to 64 parts' by 6: 17 u. While a thread reads
on, its reference is up to 4 below its largest logit, and each of the at most 4 changes of reference that matter
multiplies by an exponential: where logits rise within a thread, 3 * 8 + 4 * 4 = 40 u more."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _rows(n, V, io, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    logits = (torch.randn(n, V, generator=g, device="cuda") * 2).to(IO[io])
    logits[1, : V - 3] = -math.inf  # little is left
    logits[2] = logits[2].round()  # equal logits in every batch
    logits[3, V // 3:] = torch.finfo(IO[io]).min
    tokens = torch.randint(0, V, (n,), generator=g, device="cuda")
    tokens[4] = -1
    tokens[1] = V - 2
    return logits, tokens


@pytest.mark.parametrize("top", [0, 5, 32])
@pytest.mark.parametrize("n,V,io", [
    (300, 60001, "bf16"),    # four waves a row, several batches, odd addresses
    (300, 60001, "f32"),
    (200, 140001, "bf16"),   # 16 waves a row, five batches
    (129, 262144, "f32"),    # 16 waves, two batches to each noted maximum
    (300, 262144, "f16"),    # four waves, a row in three parts
    (2000, 131071, "bf16"),  # four waves, 16 batches
    (20000, 4001, "bf16"),   # one wave a row, two batches; a gradient past the cache
])
def test_rows_of_many_batches(cuda_device, n, V, io, top):
    """Sampled rows against the oracle; every row's values against float64 sums of torch's."""
    from hsn_amd import scoring

    logits, tokens = _rows(n, V, io, n + V)
    out = scoring.forward(logits, tokens, top=top)
    some = sorted({0, 1, 2, 3, 4, 5, n // 2, n - 2, n - 1})
    logprob, entropy, best, best_logprob = R.score(logits[some].cpu(), tokens[some].cpu(), top)
    # |x| is about 4 where the mass is: 3 * 4 + 4 + 7 + 17 + 40 u and the logarithm's 2 u of 14
    log_bar = (80 + 28) * U
    _near(out["logprob"][some], logprob, log_bar + 2 * U * _size(logprob))
    _near(out["entropy"][some], entropy, 5 * log_bar)  # W / S with |x| about 4, and log S
    if top:
        assert torch.equal(out["top_tokens"][some].cpu(), best)
        _near(out["top_logprobs"][some], best_logprob, log_bar + 2 * U * _size(best_logprob))
        # and the other rows' are a descending list of logits, none of which is left out
        values = logits.gather(1, out["top_tokens"].clamp(min=0)).float()
        least = torch.topk(logits.float(), top, dim=1).values
        there = out["top_tokens"] >= 0
        assert torch.equal(there, least > -math.inf)
        assert torch.equal(values[there], least[there])
    d = torch.randn(n, generator=torch.Generator().manual_seed(0)).to(cuda_device)
    h = d.flip(0)
    step = max(1, (1 << 27) // V)
    for i in range(0, n, step):
        l = logits[i:i + step].double()
        rest = torch.logsumexp(l, 1)
        logp = l - rest[:, None]
        p = torch.exp(logp)
        H = -torch.where(p > 0, p * logp, 0.0).sum(1)
        t = tokens[i:i + step]
        want = torch.where(t >= 0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
        _near(out["logprob"][i:i + step], want.cpu(), log_bar + 2 * U * _size(want.cpu()))
        _near(out["entropy"][i:i + step], H.cpu(), 5 * log_bar)
    back = scoring.backward(logits, tokens, out["stats"], d, h)
    for i in some:
        t = int(tokens[i])
        l = logits[i].double()
        logp = torch.log_softmax(l, 0)
        p = torch.exp(logp)
        H = -torch.where(p > 0, p * logp, 0.0).sum()
        want = -p * ((float(d[i]) if t >= 0 else 0.0) + float(h[i]) * torch.where(p > 0, logp + H, 0.0))
        if t >= 0:
            want[t] += float(d[i])
        x = (l.max() - l).clamp(max=200)
        # p off by (3 |x| + 4) u and the sum's error of itself, log p + H by log S's and the entropy's
        size = abs(float(d[i])) + abs(float(h[i])) * (x + 20)
        bar = p * (size * ((3 * x + 12) * U + log_bar) + abs(float(h[i])) * 6 * log_bar)
        # (a probability below fp32's smallest normal number is 0) and the rounding
        bar = bar + size * 2.0 ** -125 + want.abs() * (torch.finfo(IO[io]).eps / 2 + 2 * U)
        bar = bar + (2.0 ** -25 if io == "f16" else 0.0)
        if t >= 0:
            bar[t] += abs(float(d[i])) * 2 * U
        assert bool(((back[i].double() - want).abs() <= bar).all()), i


def _size(t):
    return t.nan_to_num(0.0).clamp(min=-1e30).abs() + 1


def _near(got, want, bar):
    got, want = got.double().cpu(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine])
    bar = (torch.as_tensor(bar, dtype=torch.float64) + torch.zeros_like(want))[fine]
    off = (got - want)[fine].abs()
    assert bool((off <= bar).all()), float((off - bar).max())
