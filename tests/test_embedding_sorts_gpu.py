"""The embedding's gradient by sorted lists of every length: the border of the short sort, tiles of all three
sizes with one to three digits, lists whose tokens are alike, neighbours or in any order.

A sum of m cotangents over spans of at most 1024 one by one and then over the spans is off by at most
min(m, 1100) + m / 1024 + 4 steps of 2^-24 of the sum of their sizes."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _tokens(n, V, seed, kind="any"):
    g = torch.Generator("cuda").manual_seed(seed)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if kind == "alike":
        t = (u * V).long()
    else:  # the r-th most frequent has a share of about 1 / r; as they are, these are neighbours
        t = ((V + 1.0) ** u - 1).long().clamp(0, V - 1)
        if kind == "any":
            t = torch.randperm(V, generator=g, device="cuda")[t]
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.1, -1, t)


def _check(tokens, V, D, dtype=torch.float32):
    from hsn_amd import embedding

    n = tokens.numel()
    d = torch.randn(n, D, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(dtype)
    got = embedding.backward(tokens, d, V, dtype=torch.float32)
    keep = tokens >= 0
    order = torch.sort(torch.where(keep, tokens, V), stable=True).indices
    # the sums in float64, as differences of running sums (off by less than 2^-30)
    count = torch.bincount(tokens[keep], minlength=V)[:, None]
    end = count.cumsum(0)[:, 0]
    want, size = (torch.cat([zero, x.double().cumsum(0)])[torch.stack([end - count[:, 0], end])].diff(dim=0)[0]
                  for zero in [torch.zeros(1, D, dtype=torch.float64, device="cuda")]
                  for x in (d[order], d[order].abs()))
    bar = size * (count.clamp(max=1100) + count / 1024 + 4) * U + want.abs() * U + 2.0 ** -30
    assert bool(((got.double() - want).abs() <= bar).all())
    assert not got[count[:, 0] == 0].any()
    # the sums go by the sorted list alone: the list sorted beforehand, with its positions' order kept, gives the
    # same bits
    assert torch.equal(embedding.backward(tokens[order], d[order], V, dtype=torch.float32), got)


@pytest.mark.parametrize("n", [1023, 1025, 2048, 2049, 4097, 8191, 8192, 8193, 8256])
@pytest.mark.parametrize("V", [3, 1000, 70001])
def test_around_the_short_sort(cuda_device, n, V):
    for kind in ("any", "alike"):
        _check(_tokens(n, V, n, kind), V, 9)


@pytest.mark.parametrize("n", [60001, 65536, 65537, 524288, 524289, 600001, 1100003])
@pytest.mark.parametrize("V", [700, 5003, 100003, (1 << 20) + 1])
def test_tiles_and_digits(cuda_device, n, V):
    """Tiles of four, eight and 32 entries a thread; one digit, two, two, three."""
    for kind in ("any", "neighbours"):
        _check(_tokens(n, V, n, kind), V, 3, torch.bfloat16)


@pytest.mark.parametrize("n", [8193, 70001, 600001])
def test_one_token(cuda_device, n):
    V = 2000
    tokens = torch.full((n,), 1777, device=cuda_device)
    _check(tokens, V, 20)
    tokens[::3] = -1
    _check(tokens, V, 20)
    tokens[::2] = 1778
    _check(tokens, V, 20)
