"""The choice of units where a wave takes several turns: stepped addresses, LDS slots written again, sums of many
turns, against float64.

Bars as beside the other tests of the choice: with u = 2^-24 and |x| < 32, a share or a probability is off by at most
140 u, a mean of probabilities by 170 u of itself, a gradient by four such errors of its terms' sizes and
half a step of a 16-bit type."""

from __future__ import annotations

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _reference(logits, k, valid, d_shares, d_balance):
    """The oracle's values for many tokens at once, on the logits' device; no token is without a logit."""
    l = logits.double()
    n, M = l.shape
    live = torch.ones(n, dtype=torch.bool, device=l.device) if valid is None else valid
    order = torch.sort(l, dim=1, descending=True, stable=True)
    units = order.indices[:, :k]
    shares = torch.softmax(order.values[:, :k], dim=1) * live[:, None]
    p = torch.softmax(l, dim=1) * live[:, None]
    counts = torch.bincount(units[live].reshape(-1), minlength=M)
    rows = int(live.sum())
    load = counts.double() / max(1, int(counts.sum()))
    probs = p.sum(dim=0) / max(1, rows)
    g = d_shares.double()
    d = torch.zeros_like(l).scatter_(1, units, shares * (g - (shares * g).sum(dim=1, keepdim=True)))
    d += d_balance * M / max(1, rows) * p * (load - p @ load[:, None])
    return torch.where(live[:, None], units, -1), shares, M * (load * probs).sum(), counts, probs, rows, d


def _off(got, want, bar):
    off = (got.double() - want).abs()
    assert bool((off <= bar).all()), float((off - bar).max())


def _check(n, M, k, io, dev, padded, stride=0):
    from hsn_amd import unit_router

    g = torch.Generator("cuda").manual_seed(n + M)
    wide = (torch.randn(n, M + stride, generator=g, device=dev) * 2).to(IO[io])
    logits = wide[:, stride:]
    valid = torch.rand(n, generator=g, device=dev) < 0.8 if padded else None
    d_shares = torch.randn(n, 2 * k + 1, generator=g, device=dev)[:, 1:k + 1]
    d_balance = torch.tensor(1.7, device=dev) * n / 50  # so that it is as large as the shares' part
    out = unit_router.forward(logits, k, valid=valid)
    units, shares, balance, counts, probs, rows, want = _reference(logits, k, valid, d_shares, float(d_balance))
    assert torch.equal(out["units"], units) and torch.equal(out["counts"], counts)
    assert torch.equal(out["tally"][:M], counts) and int(out["tally"][M]) == rows
    _off(out["shares"], shares, 140 * U)
    _off(out["probs"], probs, 170 * U * probs)
    _off(out["balance"], balance, 170 * U * max(1.0, float(balance)))
    d = unit_router.backward(logits, out["units"], out["tally"], d_shares, d_balance, valid=valid)
    scale = 2 * d_shares.double().abs().amax(dim=1, keepdim=True)
    p = torch.softmax(logits.double(), dim=1)
    bar = 4 * 140 * U * (scale + float(d_balance) * M / max(1, rows) * 2 * p)
    if io != "f32":
        bar = bar + want.abs() * torch.finfo(IO[io]).eps / 2 + (2.0 ** -25 if io == "f16" else 0.0)
    _off(d, want, bar)
    if valid is not None:
        assert not d[~valid].any()


def test_the_reference_is_the_oracle():
    n, M, k = 60, 21, 5
    g = torch.Generator().manual_seed(0)
    logits, d = torch.randn(n, M, generator=g), torch.randn(n, k, generator=g)
    valid = torch.rand(n, generator=g) < 0.7
    for v in (None, valid):
        got = _reference(logits, k, v, d, 0.9)
        want = (*R.choose_units(logits, k, v), R.choose_units_backward(logits, k, d, torch.tensor(0.9, dtype=torch.float64), v))
        assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3]) and got[5] == want[5]
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("n,M,k,io,stride", [
    (70001, 64, 8, "bf16", 3),    # 16 lanes a token, four turns of the forward's 16 waves, three of the backward's
    (70001, 64, 8, "f32", 1),
    (20001, 250, 16, "bf16", 1),  # a wave a token, the last units shared by two lanes
    (20001, 250, 16, "f32", 0),
    (20003, 256, 7, "f16", 0),
    (40001, 70, 13, "f16", 2),    # 32 lanes a token
    (300007, 8, 3, "f32", 0),     # two lanes a token
    (90001, 30, 16, "bf16", 5),   # eight lanes a token, two slots a lane
    (140003, 3, 2, "f16", 1),     # a lane a unit
    (600011, 4, 2, "bf16", 0),    # a lane a token
    (160001, 13, 9, "f32", 0),    # four lanes a token
])
def test_turns(cuda_device, n, M, k, io, stride, padded):
    _check(n, M, k, io, cuda_device, padded, stride)


def test_slots_and_cotangents_past_32_bits(cuda_device):
    """2^29 + 5 tokens of 8 units, 5 chosen: 2.7e9 slots; sampled tokens against float64."""
    from hsn_amd import unit_router

    if torch.cuda.get_device_properties(cuda_device).total_memory < 150 << 30:
        pytest.skip("needs 150 GiB of device memory")
    n, M, k = (1 << 29) + 5, 8, 5
    g = torch.Generator("cuda").manual_seed(0)
    logits = torch.empty(n, M, dtype=torch.bfloat16, device=cuda_device)
    d_shares = torch.empty(n, k, device=cuda_device)
    for i in range(0, n, 1 << 26):
        end = min(n, i + (1 << 26))
        logits[i:end] = torch.randn(end - i, M, generator=g, device=cuda_device).to(torch.bfloat16)
        d_shares[i:end] = torch.randn(end - i, k, generator=g, device=cuda_device)
    out = unit_router.forward(logits, k)
    tally = out["tally"]
    assert int(tally[M]) == n and int(tally[:M].sum()) == n * k
    d_balance = torch.tensor(float(n), device=cuda_device)
    d = unit_router.backward(logits, out["units"], tally, d_shares, d_balance)
    load = tally[:M].double() / (n * k)
    at = torch.tensor([0, 1, (1 << 28) + 3, n // 2, 429496729, 429496731, n - 2, n - 1], device=cuda_device)
    # (2^31 / 5 is 429496729.6)
    l = logits[at].double()
    order = torch.sort(l, dim=1, descending=True, stable=True)
    assert torch.equal(out["units"][at], order.indices[:, :k])
    shares = torch.softmax(order.values[:, :k], dim=1)
    _off(out["shares"][at], shares, 140 * U)
    p = torch.softmax(l, dim=1)
    c = d_shares[at].double()
    want = torch.zeros_like(l).scatter_(1, order.indices[:, :k], shares * (c - (shares * c).sum(dim=1, keepdim=True)))
    want += M * p * (load - p @ load[:, None])
    scale = 2 * c.abs().amax(dim=1, keepdim=True)
    _off(d[at], want, 4 * 140 * U * (scale + 2 * M * p) + want.abs() * 2.0 ** -8)
    torch.cuda.empty_cache()
