"""Scoring's sums over many logits that are alike, or that rise slowly, against float64.

Bars, with u = 2^-24 and x = l - max l: an exponential is off by (3 |x| + 4) u of itself (the difference, its product
with log2 e and the constant, the instruction's 2 u). A sum of a batch is off by 7 u of itself (three steps of
pairs or four of a chain, two of packs, two to spare), a thread's sums of batches are float64. 64 threads' sums are
rounded to fp32 and joined by 6 steps, 4 or 16 waves' by 2 or 4 and up to 64 parts' by 6: 17 u. While a thread reads
on, its reference is up to 4 below its largest logit, and each of the at most 4 changes of reference that matter
multiplies by an exponential: where logits rise within a thread, 3 * 8 + 4 * 4 = 40 u more."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _statistics(row):
    """The log of the sum, the entropy and the mean of |x| of one row, in float64."""
    x = row.double() - row.double().max()
    e = torch.exp(x)
    p = e / e.sum()
    rest = torch.log(e.sum())
    return float(rest), float(rest - (p * x).sum()), float((p * -x).sum())


def _check_row(row, token, rows, changes, gradient):
    """``row`` as ``rows`` rows of one launch (the same memory), its values and gradient against float64."""
    from hsn_amd import scoring

    logits = row[None].expand(rows, -1)
    tokens = torch.full((rows,), token, device=row.device)
    out = scoring.forward(logits, tokens)
    rest, entropy, mean = _statistics(row)
    x = float(row[token].double() - row.double().max())
    # a sum, and its logarithm rounded
    off = (3 * mean + 4 + 7 + 17 + changes) * U
    log_bar = off + 2 * U * abs(rest)
    assert bool((out["logprob"].double() - (x - rest)).abs().max() <= log_bar + 2 * U * (abs(x) + abs(x - rest)))
    # W adds the products' and its own like errors, each of at most (3 |x| + 4 + 7 + 17 + 2) u of e |x|
    # (not torch.softmax: of more than 1024 numbers in float64 it is right to 2^-24 only)
    p = torch.exp(torch.log_softmax(row.double(), 0))
    square = float((p * (row.double() - row.double().max()) ** 2).sum())
    bar = log_bar + (3 * square + 30 * mean + changes * (mean + 1)) * U + mean * (off + 4 * U) + 2 * U * abs(entropy)
    assert bool((out["entropy"].double() - entropy).abs().max() <= bar)
    if gradient:
        d = scoring.backward(logits, tokens, out["stats"], torch.ones(rows, device=row.device))
        want = -p
        want[token] += 1
        x = (row.double().max() - row.double())
        bar = (3 * x + 4 + 8) * U * (want - (torch.arange(row.numel(), device=row.device) == token).double()).abs()
        bar = bar + off * p + 2 * U * want.abs()
        for i in (0, rows // 2, rows - 1):
            assert bool(((d[i].double() - want).abs() <= bar).all())


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("V", [131072, 1 << 20, 1 << 24])
def test_a_flat_background(cuda_device, V, io):
    """Every thread's first batch has the row's largest logits, and all others are alike: each addition of a
    background's exponential rounds the same way."""
    for below in (0.7, 1.1, 2.3, 3.9, 5.2):
        row = torch.full((V,), -below, device=cuda_device).to(IO[io])
        row[:16384] = 0.0
        _check_row(row, V - 1, 1024, 0, gradient=io == "f32" and V == 131072)


@pytest.mark.parametrize("V", [131072, 1 << 20, 1 << 24])
@pytest.mark.parametrize("up", [1.0, -1.0])
def test_a_slow_ramp(cuda_device, up, V):
    """Every batch has a new largest logit, by little (or none has)."""
    for height in (0.25, 1.0, 6.0, 40.0):
        row = torch.arange(V, device=cuda_device, dtype=torch.float64) * (up * height / V)
        _check_row(row.float(), V // 2, 1024, 40, gradient=V == 131072)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("V", [131072, 1 << 22])
def test_one_peak(cuda_device, V, io):
    """A single large logit: the thread that has it adds numbers of 1e-7 to one of 1."""
    for below in (9.1, 16.3):
        row = torch.full((V,), -below, device=cuda_device).to(IO[io])
        row[77] = 0.0
        _check_row(row, V - 1, 1024, 0, gradient=io == "f32" and V == 131072)


def test_probabilities_of_every_size(cuda_device):
    """A probability is off by its exponential's (3 |x| + 4) u and its sum's share, down to the smallest normal
    numbers: the gradient of one row, but for its own token."""
    from hsn_amd import scoring

    x = -84 * torch.rand(1 << 16, generator=torch.Generator().manual_seed(0))
    x[0] = 0.0
    tokens = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    on = x[None].to(cuda_device)
    d = scoring.backward(on, tokens, scoring.forward(on, tokens)["stats"], -torch.ones(1, device=cuda_device))
    p = torch.softmax(x.double(), 0)
    # the mean of |x| is about 1; the reciprocal and the product round too
    off = (d[0].cpu().double() - p).abs()[1:]
    assert bool((off <= ((-3 * x + 4 + 3 + 4 + 24 + 4) * U * p + 2.0 ** -126)[1:]).all())
