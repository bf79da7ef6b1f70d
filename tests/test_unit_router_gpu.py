"""The choice of units, its balance and their gradient on the GPU against the float64 oracle.

Bars, with u = 2^-24 and |x| < 32 (x = l - max l): an exponential is off by (3 |x| + 4) u of itself, a sum
of up to 256 of them by 12 u more, so a share or a probability by (3 |x| + 40) u of itself, at most 140 u
of 1 where it is largest over e (p |x| e < 1 / e) and below. A mean of probabilities averages that: 40 u of itself
and 128 u for the fp32 sums of 128 tokens; the balance likewise. A gradient is off by four such errors of
its terms' sizes, and outputs of 16 bits by half a step."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _near(got, want, bar):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert bool(torch.isfinite(got[fine]).all())
    off = (got - want).abs()[fine]
    bar = (torch.as_tensor(bar, dtype=torch.float64) + torch.zeros_like(want))[fine]
    assert bool((off <= bar).all()), float((off - bar).max())


def _problem(n, M, io, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, M, generator=g) * spread).to(IO[io])


def _check(logits, k, dev, valid=None, seed=0, parts=("shares", "balance")):
    from hsn_amd import unit_router

    n, M = logits.shape
    g = torch.Generator().manual_seed(seed)
    d_shares = torch.randn(n, k, generator=g) if "shares" in parts else None
    d_balance = torch.tensor(1.7) if "balance" in parts else None
    on = logits.to(dev)
    v = None if valid is None else valid.to(dev)
    out = unit_router.forward(on, k, valid=v)
    units, shares, balance, counts, probs, rows = R.choose_units(logits, k, valid)
    assert torch.equal(out["units"].cpu(), units)
    assert torch.equal(out["counts"].cpu(), counts) and torch.equal(out["tally"].cpu()[:M], counts)
    assert int(out["tally"][M]) == rows
    _near(out["shares"], shares, 140 * U)
    _near(out["probs"], probs, 170 * U * probs.nan_to_num(0.0) + 1e-12)
    assert out["balance"].shape == ()
    _near(out["balance"], balance, 170 * U * max(1.0, float(balance.nan_to_num(1.0))))
    d = unit_router.backward(on, out["units"], out["tally"], None if d_shares is None else d_shares.to(dev),
                             None if d_balance is None else d_balance.to(dev), valid=v)
    assert d.shape == (n, M) and d.dtype == logits.dtype and d.is_contiguous()
    want = R.choose_units_backward(logits, k, d_shares, d_balance, valid)
    p = torch.softmax(logits.double(), dim=1).nan_to_num(0.0)
    scale = 0.0 if d_shares is None else 2 * d_shares.double().abs().amax(dim=1, keepdim=True)
    bar = 4 * 140 * U * scale
    bar = bar + (0.0 if d_balance is None else 4 * 140 * U * 1.7 * M / max(1, rows) * p * 2) + 1e-30
    if logits.dtype != torch.float32:
        bar = bar + want.abs().nan_to_num(0.0) * torch.finfo(logits.dtype).eps / 2
        bar = bar + (2.0 ** -25 if logits.dtype == torch.float16 else 0.0)  # half of the smallest step
    _near(d, want, bar)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,k", [(3, 2), (8, 3), (17, 16), (64, 8), (250, 16)])
def test_the_smallest_and_largest_logits(cuda_device, M, k, io):
    """Logits below the smallest normal one keep their order, of both signs and beside zeros; the type's
    lowest value is chosen like any other, and -inf is not."""
    info = torch.finfo(IO[io])
    rows = 37
    g = torch.Generator().manual_seed(M + k)
    step = info.smallest_normal * info.eps  # the smallest step there is
    small = (torch.randint(-100, 100, (rows, M), generator=g).double() * step).to(IO[io])
    assert int(torch.unique(small).numel()) > 30 or rows * M < 200
    small[::3, 0] = -0.0
    edges = torch.tensor([info.min, -math.inf, info.min / 2, -1.0, 0.0]).to(IO[io])
    edge = edges[torch.randint(0, 5, (rows, M), generator=g)]
    edge[0] = info.min
    edge[1] = -math.inf
    edge[2] = -math.inf
    edge[2, M // 2] = info.min
    _check(torch.cat([small, edge]), k, cuda_device, seed=k)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,M,k", [(1, 1, 1), (1, 8, 2), (5, 3, 3), (33, 4, 4), (70, 8, 2), (130, 16, 5),
                                   (65, 17, 16), (40, 33, 7), (37, 64, 8), (21, 100, 3), (19, 129, 16),
                                   (9, 256, 8), (12, 255, 1)])
def test_values_and_gradient(cuda_device, n, M, k, io):
    logits = _problem(n, M, io, n + M)
    valid = torch.rand(n, generator=torch.Generator().manual_seed(k)) < 0.8
    _check(logits, k, cuda_device)
    _check(logits, k, cuda_device, valid)
    _check(logits, k, cuda_device, valid, parts=("shares",))
    _check(logits, k, cuda_device, None, parts=("balance",))


@pytest.mark.parametrize("M,k", [(8, 3), (100, 8), (256, 16)])
def test_ties_go_to_the_lowest_unit(cuda_device, M, k):
    g = torch.Generator().manual_seed(M)
    logits = torch.randint(0, 3, (50, M), generator=g).float()
    logits[0] = 1.0
    logits[1] = -0.0
    logits[1, M // 2] = 0.0  # equal to -0
    _check(logits, k, cuda_device)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,k", [(3, 2), (8, 8), (64, 6), (200, 16)])
def test_masked_units(cuda_device, M, k, io):
    """Tokens with fewer units than slots, one, or none; a mask of the type's lowest value."""
    logits = _problem(12, M, io, M)
    logits[0] = -math.inf
    logits[1, 1:] = -math.inf
    logits[2, : M - 2] = -math.inf
    logits[3] = torch.finfo(logits.dtype).min
    logits[4, 1:] = torch.finfo(logits.dtype).min
    logits[5, ::2] = -math.inf
    _check(logits, k, cuda_device)
    valid = torch.ones(12, dtype=torch.bool)
    valid[4:] = False
    _check(logits, k, cuda_device, valid)
    _check(logits[:1], k, cuda_device)  # no live token at all
    _check(logits, k, cuda_device, torch.zeros(12, dtype=torch.bool))


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("M", [2, 8, 100])
def test_nan_and_infinity(cuda_device, M, bad, io):
    """Their own token's shares and gradient, and the means; not another token's."""
    from hsn_amd import unit_router

    logits = _problem(6, M, io, 3)
    logits[2, M - 1] = bad
    if math.isnan(bad):
        logits[4] = bad
    k = 2
    on = logits.to(cuda_device)
    out = unit_router.forward(on, k)
    assert torch.equal(out["units"].cpu(), R.choose_units(logits, k)[0])
    strange = torch.tensor([False, False, True, False, math.isnan(bad), False])
    assert bool(out["shares"].cpu()[strange].isnan().all())
    assert math.isnan(float(out["balance"])) and bool(out["probs"].isnan().all())
    d = unit_router.backward(on, out["units"], out["tally"], torch.ones(6, k, device=cuda_device),
                             torch.ones((), device=cuda_device)).cpu()
    assert bool(d[strange].isnan().all()) and bool(torch.isfinite(d[~strange]).all())
    # a token that is not valid leaves the means alone
    _check(logits, k, cuda_device, ~strange)


def test_many_tokens(cuda_device):
    """More tokens than one round of the workgroups, and sums that leave fp32 behind."""
    from hsn_amd import unit_router

    n, M, k = 300001, 4, 2
    logits = _problem(n, M, "f32", 0)
    out = unit_router.forward(logits.to(cuda_device), k)
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    assert torch.equal(out["units"].cpu(), order.indices[:, :k])
    counts = torch.bincount(order.indices[:, :k].reshape(-1), minlength=M)
    assert torch.equal(out["counts"].cpu(), counts) and int(out["tally"][M]) == n
    probs = torch.softmax(logits.double(), dim=1).mean(dim=0)
    _near(out["probs"], probs, 170 * U * probs)
    shares = torch.softmax(order.values[:, :k].double(), dim=1)
    _near(out["shares"], shares, 140 * U)


def test_strides(cuda_device):
    from hsn_amd import unit_router

    for io in ("f32", "bf16"):
        wide = _problem(40, 90, io, 1).to(cuda_device)
        d = torch.randn(40, 9, device=cuda_device)
        b = torch.ones((), device=cuda_device)
        for start, M, k in ((0, 64, 4), (1, 33, 3), (7, 64, 8), (3, 2, 1)):
            view = wide[:, start:start + M]
            out, ref = unit_router.forward(view, k), unit_router.forward(view.contiguous(), k)
            for name in out:
                assert torch.equal(out[name], ref[name]), name
            got = unit_router.backward(view, out["units"], out["tally"], d[:, 1:1 + k], b)
            want = unit_router.backward(view.contiguous(), out["units"], out["tally"],
                                        d[:, 1:1 + k].contiguous(), b)
            assert torch.equal(got, want)
        assert torch.equal(unit_router.forward(wide[::3], 5)["units"],
                           unit_router.forward(wide[::3].contiguous(), 5)["units"])


def test_the_gradient_against_differences(cuda_device):
    from hsn_amd import unit_router

    logits = _problem(4, 12, "f32", 9).to(cuda_device).requires_grad_()
    w = torch.randn(4, 3, generator=torch.Generator().manual_seed(2)).to(cuda_device)

    def loss(l):
        _, shares, balance, _ = unit_router.choose_units(l, 3)
        return (shares * w).sum() + 0.7 * balance

    grad, = torch.autograd.grad(loss(logits), logits)
    for i in range(4):
        for j in range(12):
            step = torch.zeros_like(logits)
            step[i, j] = 2.0 ** -7
            with torch.no_grad():
                ahead, behind = (unit_router.choose_units(logits + s, 3) for s in (step, -step))
                if not torch.equal(ahead[0], behind[0]):
                    continue  # another choice
                slope = (loss(logits + step) - loss(logits - step)) / 2.0 ** -6
            # a third derivative below 6 (the sizes of w), a loss off by 2^-20 each side
            assert abs(float(slope - grad[i, j])) <= 2.0 ** -14 + 2.0 ** -20 * 2 ** 6


def test_the_autograd_node(cuda_device):
    from hsn_amd import unit_router

    logits = _problem(30, 10, "bf16", 4).to(cuda_device).requires_grad_()
    units, shares, balance, counts = unit_router.choose_units(logits, 2)
    assert not units.requires_grad and not counts.requires_grad
    out = unit_router.forward(logits.detach(), 2)
    one = torch.ones((), device=cuda_device)
    grad, = torch.autograd.grad(shares.sum() + 0.5 * balance, logits, create_graph=True)
    assert torch.equal(grad.detach(), unit_router.backward(
        logits.detach(), out["units"], out["tally"], torch.ones(30, 2, device=cuda_device), 0.5 * one))
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    grad, = torch.autograd.grad(unit_router.choose_units(logits, 2)[2], logits)
    assert torch.equal(grad, unit_router.backward(logits.detach(), out["units"], out["tally"], None, one))


def test_it_chooses_as_the_unit_layer(cuda_device):
    """The training choice, applied by plain products, gives what the unit layer answers: its bar there
    is 1e-5 of the values' size for fp32."""
    from hsn_amd import unit_router
    from hsn_amd.unit_layer import unit_layer

    g = torch.Generator().manual_seed(5)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(cuda_device)

    n, M, k, d, H = 7, 12, 3, 24, 16
    x, router = rnd(n, d), rnd(M, d, scale=d ** -0.5)
    W1, W2 = rnd(M, d, H, scale=d ** -0.5), rnd(M, H, d, scale=H ** -0.5)
    units, shares, _, _ = unit_router.choose_units(x @ router.t(), k)
    want = torch.zeros(n, d, dtype=torch.float64, device=cuda_device)
    for i in range(n):
        for r in range(k):
            z = x[i].double() @ W1[units[i, r]].double()
            z = 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
            want[i] += shares[i, r].double() * (z @ W2[units[i, r]].double())
    got = unit_layer(x, router, W1, None, W2, None, k)
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)


def test_no_token(cuda_device):
    from hsn_amd import unit_router

    logits = torch.zeros(0, 8, device=cuda_device)
    out = unit_router.forward(logits, 2)
    assert out["units"].shape == (0, 2) and float(out["balance"]) == 0.0
    assert not out["tally"].any() and not out["probs"].any()
    assert unit_router.backward(logits, out["units"], out["tally"], None, out["balance"]).shape == (0, 8)


def test_units_outside_are_empty_slots(cuda_device):
    from hsn_amd import unit_router

    logits = _problem(5, 6, "f32", 0).to(cuda_device)
    out = unit_router.forward(logits, 2)
    d = torch.randn(5, 2, device=cuda_device)
    units = out["units"].clone()
    units[:, 1] = torch.tensor([-1, 6, 2 ** 40, -2 ** 63, 7], device=cuda_device)
    got = unit_router.backward(logits, units, out["tally"], d)
    # one unit alone has the share 1, and g - (p g) (1 / p) is left: the product, the reciprocal and the
    # second product round by u each, the difference is then exact, and the share in front of it is
    # 1 within 2 u, so at most 4 u |g| of the formula's 0
    assert bool((got.abs() <= 4 * U * d[:, :1].abs()).all())
    assert int((got != 0).sum()) <= 5


def test_the_same_bits_every_time_and_from_graphs(cuda_device):
    from hsn_amd import unit_router

    source = [_problem(5000, 70, "bf16", seed).to(cuda_device) for seed in range(3)]
    logits = source[0].clone()
    d = torch.randn(5000, 6, device=cuda_device)
    one = torch.ones((), device=cuda_device)

    def both():
        out = unit_router.forward(logits, 6)
        return [*(out[k] for k in sorted(out)),
                unit_router.backward(logits, out["units"], out["tally"], d, one)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(both())
    for i in range(4):
        logits.copy_(source[i % 3])
        for graph in graphs:
            graph.replay()
        eager = both()
        torch.cuda.synchronize()
        for results in held:
            for a, b in zip(results, eager):
                assert torch.equal(a, b)


@pytest.mark.parametrize("helper", [True, False])
def test_refusals(cuda_device, monkeypatch, helper):
    from hsn_amd import unit_router

    if not helper:
        monkeypatch.setattr(unit_router, "native_calls", lambda *names: None)
    logits = torch.zeros(4, 10, device=cuda_device)
    out = unit_router.forward(logits, 2)
    units, tally = out["units"], out["tally"]
    d = torch.zeros(4, 2, device=cuda_device)
    for bad in (logits.double(), logits[0]):
        with pytest.raises(ValueError, match="logits must be"):
            unit_router.forward(bad, 1)
    with pytest.raises(ValueError, match="cpu"):
        unit_router.forward(logits.cpu(), 1)
    for bad in (logits[:, :0], logits[:, :1].expand(4, 257)):
        with pytest.raises(ValueError, match="M must be"):
            unit_router.forward(bad, 1)
    for bad in (0, 11, 17):
        with pytest.raises(ValueError, match="k must be"):
            unit_router.forward(logits, bad)
    with pytest.raises(ValueError, match="contiguous"):
        unit_router.forward(logits.t(), 1)
    for bad in (torch.ones(3, dtype=torch.bool, device=cuda_device), torch.ones(4, device=cuda_device)):
        with pytest.raises(ValueError, match="valid must be"):
            unit_router.forward(logits, 1, valid=bad)
    with pytest.raises(ValueError, match="valid must be contiguous"):
        unit_router.forward(logits, 1, valid=torch.ones(8, dtype=torch.bool, device=cuda_device)[::2])
    with pytest.raises(ValueError, match="units must be"):
        unit_router.backward(logits, units[0], tally, d)
    with pytest.raises(ValueError, match="units must be"):
        unit_router.backward(logits, units.int(), tally, d)
    with pytest.raises(ValueError, match="tally must be"):
        unit_router.backward(logits, units, tally[:10], d)
    for bad in (d[:3], d.double(), d.t().contiguous().t()):
        with pytest.raises(ValueError, match="d_shares must be"):
            unit_router.backward(logits, units, tally, bad)
    for bad in (d, d[0, 0].double(), d[0, 0].cpu()):
        with pytest.raises(ValueError, match="d_balance must be"):
            unit_router.backward(logits, units, tally, d, bad)


def test_both_ways_of_calling_give_the_same(cuda_device, monkeypatch):
    from hsn_amd import unit_router

    logits = _problem(500, 20, "f16", 8).to(cuda_device)
    d, one = torch.randn(500, 4, device=cuda_device), torch.ones(1, device=cuda_device)
    valid = torch.rand(500, device=cuda_device) < 0.5

    def everything():
        out = unit_router.forward(logits, 4, valid=valid)
        return [out[k] for k in sorted(out)] + [
            unit_router.backward(logits, out["units"], out["tally"], d, one, valid=valid)]

    with_it = everything()
    monkeypatch.setattr(unit_router, "native_calls", lambda *names: None)
    for a, b in zip(with_it, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype
