"""The unit layer on the GPU against the float64 oracle.

Tolerance. With x of order 1 and weights of order width^-1/2 every product sum is of order 1 and an
fp32 sum of up to 4096 products is off by at most about sqrt(4096) 2^-24 times its terms' size in
the mean, 2^-24 4096 2^-6 ~ 4e-6 in all but one of millions; three sums and the activation follow one
another, so 2e-5 of the largest |y|. A 16-bit output adds half a unit in its last place. A choice
that the oracle's router decides by less than 1e-4 is moved apart before the call."""

from __future__ import annotations

import pytest
import torch

from oracle import language as L

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FP32 = 2e-5


def _problem(n, M, K, d_in, H, d_out, io, activation, bias, seed=0, like_one=False):
    g = torch.Generator().manual_seed(seed)
    io = IO[io]
    H1 = 2 * H if activation == "swiglu" else H

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(io)

    x, router = rnd(n, d_in), rnd(M, d_in, scale=d_in ** -0.5)
    if like_one:  # every token chooses alike
        x = (rnd(1, d_in).float() + 1e-2 * rnd(n, d_in).float()).to(io)
    for _ in range(100):  # no choice by a hair
        best = (x.double() @ router.double().t()).sort(1, descending=True).values
        if M > K:
            near = (best[:, K - 1] - best[:, K]) < 1e-4
            if not bool(near.any()):
                break
            x[near] = rnd(int(near.sum()), d_in)
        else:
            break
    W1, W2 = rnd(M, d_in, H1, scale=d_in ** -0.5), rnd(M, H, d_out, scale=H ** -0.5)
    b1, b2 = (rnd(M, H1, scale=0.3), rnd(M, d_out, scale=0.3)) if bias else (None, None)
    return x, router, W1, b1, W2, b2


def _check(got, want, io, floor=1.0):
    got = got.double().cpu()
    scale = max(floor, float(want.abs().max())) if want.numel() else 1.0
    room = FP32 * scale + HALF_ULP[io] * want.abs() * (1 + 1e-3) + (2.0 ** -24 if io == torch.float16 else 0)
    off = (got - want).abs()
    assert bool((off <= room).all()), f"off by {float((off - room).max()):.3g} over the bound"


def _run(p, K, activation, dev):
    from hsn_amd.unit_layer import unit_layer

    return unit_layer(*(None if t is None else t.to(dev) for t in p), K, activation=activation)


SIZES = [(1, 1, 1, 1, 1, 1), (1, 8, 2, 256, 512, 64), (3, 5, 5, 24, 77, 24), (7, 12, 3, 99, 123, 99),
         (16, 4, 2, 64, 128, 64), (64, 16, 4, 64, 96, 32), (2, 256, 16, 40, 24, 40),
         (5, 9, 2, 520, 264, 200), (33, 3, 1, 72, 64, 136), (4, 6, 3, 2056, 40, 16),
         (2, 4, 2, 16, 2056, 24)]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("activation,bias", [("gelu", True), ("swiglu", False), ("swiglu", True)])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(cuda_device, io, activation, bias, size):
    n, M, K, d_in, H, d_out = size
    p = _problem(n, M, K, d_in, H, d_out, io, activation, bias, seed=sum(size))
    got = _run(p, K, activation, cuda_device)
    assert got.dtype == IO[io] and got.shape == (n, d_out)
    _check(got, L.unit_layer(*p, K, activation), IO[io])


@pytest.mark.parametrize("n", [1, 2, 8, 9, 17, 64])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_tokens_that_choose_alike(cuda_device, n, io):
    """All tokens on the same units: one unit's tokens fill more than one group."""
    p = _problem(n, 10, 2, 128, 64, 72, io, "gelu", True, seed=n, like_one=True)
    _check(_run(p, 2, "gelu", cuda_device), L.unit_layer(*p, 2, "gelu"), IO[io])


def test_ties_go_to_the_lowest_units(cuda_device):
    x, router, W1, b1, W2, b2 = _problem(4, 70, 6, 32, 16, 8, "f32", "gelu", True, seed=1)
    router[:] = router[:1]
    for equal in (70, 3):
        if equal == 3:
            router[5:8] *= 0
            x = x.abs()
            router[:] = router.abs()
        p = (x, router, W1, b1, W2, b2)
        _check(_run(p, 6, "gelu", cuda_device), L.unit_layer(*p, 6, "gelu"), torch.float32)


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_rows_apart_and_at_any_address(cuda_device, io):
    from hsn_amd.unit_layer import unit_layer

    p = _problem(5, 6, 2, 64, 64, 64, io, "swiglu", False, seed=3)
    on = [None if t is None else t.to(cuda_device) for t in p]
    want = unit_layer(*on, 2, activation="swiglu")
    room = torch.zeros(5, 200, dtype=IO[io], device=cuda_device)
    view = room[:, 3:67]
    view.copy_(on[0])
    assert torch.equal(unit_layer(view, *on[1:], 2, activation="swiglu"), want)
    # weights that start one element past an aligned place
    moved = []
    for t in on[1:]:
        if t is not None:
            flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=cuda_device)
            flat[1:] = t.reshape(-1)
            t = flat[1:].view(t.shape)
        moved.append(t)
    _check(unit_layer(on[0], *moved, 2, activation="swiglu"), L.unit_layer(*p, 2, "swiglu"), IO[io])


def test_values_that_are_not_finite_stay_in_their_token(cuda_device):
    """A token with a NaN gives NaN; weights of units that nobody chose may hold anything; fp16
    values whose products pass 65504 are summed in fp32."""
    p = _problem(6, 8, 2, 64, 48, 32, "f32", "gelu", True, seed=8)
    x, router, W1, b1, W2, b2 = p
    want = L.unit_layer(*p, 2, "gelu")
    chosen = set((x @ router.t()).topk(2, dim=1).indices.reshape(-1).tolist())
    for e in set(range(8)) - chosen:
        W1[e], W2[e], b1[e], b2[e] = float("nan"), float("inf"), float("nan"), float("nan")
    got = _run(p, 2, "gelu", cuda_device)
    _check(got, want, torch.float32)
    x[3, 10] = float("nan")
    got = _run(p, 2, "gelu", cuda_device).cpu()
    assert bool(torch.isnan(got[3]).all())
    rest = [0, 1, 2, 4, 5]
    _check(got[rest], want[rest], torch.float32)
    q = _problem(3, 4, 2, 64, 64, 64, "f16", "swiglu", False, seed=9)
    q[0].mul_(100)
    q[2].mul_(30)
    q[4].mul_(1e-4)
    want = L.unit_layer(*q, 2, "swiglu")
    assert float(want.abs().max()) > 10
    _check(_run(q, 2, "swiglu", cuda_device), want, torch.float16)


def test_the_same_bits_in_every_run_and_in_a_graph(cuda_device):
    from hsn_amd.unit_layer import unit_layer

    p = _problem(9, 16, 4, 256, 128, 256, "bf16", "swiglu", True, seed=5)
    on = [t.to(cuda_device) for t in p]
    want = unit_layer(*on, 4, activation="swiglu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = unit_layer(*on, 4, activation="swiglu")
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = unit_layer(*on, 4, activation="swiglu")
    for k in range(3):
        on[0].copy_(torch.randn(9, 256, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, unit_layer(*on, 4, activation="swiglu"))


def test_weights_past_31_bits(cuda_device):
    """A bank whose last unit lies past 2^31 elements."""
    from hsn_amd.unit_layer import unit_layer

    M, d_in, H, d_out = 9, 16384, 16384, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, d_in, generator=g).bfloat16()
    router = torch.zeros(M, d_in, dtype=torch.bfloat16)
    router[M - 1] = x[0] * 0.01
    W1 = torch.empty(M, d_in, H, dtype=torch.bfloat16, device=cuda_device)
    assert W1[M - 1].data_ptr() - W1.data_ptr() >= 2 ** 32
    last = (torch.randn(d_in, H, generator=g) * d_in ** -0.5).bfloat16()
    W1[M - 1].copy_(last)
    W2 = (torch.randn(M, H, d_out, generator=g) * H ** -0.5).bfloat16()
    got = unit_layer(x.to(cuda_device), router.to(cuda_device), W1, None, W2.to(cuda_device), None, 1)
    z = x.double() @ last.double()
    want = (0.5 * z * (1 + torch.erf(z / 2 ** 0.5))) @ W2[M - 1].double()
    _check(got, want, torch.bfloat16)


def test_empty(cuda_device):
    p = _problem(0, 4, 2, 16, 8, 16, "f32", "gelu", True)
    assert _run(p, 2, "gelu", cuda_device).shape == (0, 16)


def test_refusals(cuda_device):
    from hsn_amd.unit_layer import unit_layer

    p = [t.to(cuda_device) for t in _problem(3, 6, 2, 16, 8, 16, "f32", "gelu", True)]
    x, router, W1, b1, W2, b2 = p
    many = torch.zeros(65, 16, device=cuda_device)
    bad = [
        lambda: unit_layer(*p, 0),
        lambda: unit_layer(*p, 7),
        lambda: unit_layer(*p, 2, activation="relu"),
        lambda: unit_layer(*p, 2, activation="swiglu"),
        lambda: unit_layer(many, *p[1:], 2),
        lambda: unit_layer(x.cpu(), *p[1:], 2),
        lambda: unit_layer(x.bfloat16(), *p[1:], 2),
        lambda: unit_layer(x.double(), *p[1:], 2),
        lambda: unit_layer(x[0], *p[1:], 2),
        lambda: unit_layer(x[:, ::2], *p[1:], 2),
        lambda: unit_layer(x, router[:, :8], W1, b1, W2, b2, 2),
        lambda: unit_layer(x, router, W1.transpose(1, 2), b1, W2, b2, 2),
        lambda: unit_layer(x, router, W1, b1[:3], W2, b2, 2),
        lambda: unit_layer(x, router, W1, b1, W2, b2.cpu(), 2),
        lambda: unit_layer(x, router, W1.clone().requires_grad_(), b1, W2, b2, 2),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("activation", ["gelu", "swiglu"])
def test_hidden_values_keep_their_bits(cuda_device, io, activation):
    """Two hidden values of 32 whose 20th significant bit differs, with the weights 1 and -1: the result
    is that bit. Every product and sum here is exact in fp32 (gelu(32) and silu(32) are 32), so no
    rounding is allowed for."""
    from hsn_amd.unit_layer import unit_layer

    dt = IO[io]
    x = torch.ones(1, 3, dtype=dt)
    router = torch.ones(1, 3, dtype=dt)
    W1 = torch.zeros(1, 3, 2 if activation == "gelu" else 4)
    if activation == "gelu":  # v = 32 + 2^-4 + 2^-14 and 32 + 2^-4
        W1[0, :, 0] = torch.tensor([32.0, 2.0 ** -4, 2.0 ** -14])
        W1[0, :, 1] = torch.tensor([32.0, 2.0 ** -4, 0.0])
    else:  # v = 32 (1 + 2^-9 + 2^-19) and 32 (1 + 2^-9)
        W1[0, 0, :2] = 32.0
        W1[0, :, 2] = torch.tensor([1.0, 2.0 ** -9, 2.0 ** -19])
        W1[0, :, 3] = torch.tensor([1.0, 2.0 ** -9, 0.0])
    W2 = torch.ones(1, 2, 24)
    W2[0, 1] = -1.0
    p = [t.to(dt).to(cuda_device) for t in (x, router, W1, W2)]
    assert float(p[2].float().cpu().sub(W1).abs().max()) == 0.0
    got = unit_layer(p[0], p[1], p[2], None, p[3], None, 1, activation=activation)
    assert bool((got.float() == 2.0 ** -14).all()), got


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("where", ["weight", "hidden"])
def test_an_infinity_of_a_chosen_unit_is_an_infinity(cuda_device, io, where):
    """An infinite weight W2 gives an infinity of the hidden value's sign, whatever bits that value has
    (one without low bits, one whose low bits round up or down, a small one); an infinite hidden
    value one of the weight's sign. Neither is a NaN."""
    from hsn_amd.unit_layer import unit_layer

    dt, inf = IO[io], float("inf")
    n, H, d_out = 16, 5, 20
    W1 = torch.zeros(1, n, H)  # token i picks row i
    x = torch.eye(n)
    W1[0, :, 2] = torch.cat([torch.tensor([32.0, 2.0 ** -8]), torch.linspace(0.5, 3.0, n - 2)])
    b1 = torch.zeros(1, H)
    W2 = torch.zeros(1, H, d_out)
    W2[0, 2, ::2], W2[0, 2, 1::2] = 3.0, -0.5
    if where == "weight":
        W2[0, 2, 4], W2[0, 2, 7] = inf, -inf
    else:
        b1[0, 2] = inf
    p = [t.to(dt) for t in (x, torch.ones(1, n), W1, b1, W2)]
    got = unit_layer(*(t.to(cuda_device) for t in p), None, 1).float().cpu()
    want = L.unit_layer(*p, None, 1)
    assert not bool(torch.isnan(want).any())
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not bool(torch.isnan(got).any())
    assert torch.equal(got[torch.isinf(want)].double(), want[torch.isinf(want)])
    if where == "weight":
        assert int(torch.isinf(want).sum()) == 2 * n
        finite = torch.isfinite(want)
        _check(got[finite], want[finite], dt)
    else:
        assert bool(torch.isinf(want).all())


def test_refusals_are_the_same_with_and_without_the_host_helper(cuda_device, monkeypatch):
    """More chosen units than the layer takes, where the bank has as many; wider than it takes."""
    import hsn_amd.unit_layer as module

    def refused():
        p = [t.to(cuda_device) for t in _problem(2, 32, 4, 8, 8, 8, "f32", "gelu", True)]
        with pytest.raises(ValueError, match="k must be in"):
            module.unit_layer(*p, 17)
        x, router = torch.zeros(1, 65537, device=cuda_device), torch.zeros(2, 65537, device=cuda_device)
        W1, W2 = torch.zeros(2, 65537, 4, device=cuda_device), torch.zeros(2, 4, 4, device=cuda_device)
        with pytest.raises(ValueError, match="65536"):
            module.unit_layer(x, router, W1, None, W2, None, 1)

    refused()
    monkeypatch.setattr(module, "native_calls", lambda *names: None)
    refused()


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("like_one", [False, True])
@pytest.mark.parametrize("activation,H,d_out", [("gelu", 1100, 1000), ("swiglu", 1024, 1032)])
def test_hidden_values_in_several_stages(cuda_device, io, like_one, activation, H, d_out):
    """40 units over 8 to 17 column tiles leave a workgroup all rows of W2: its hidden values pass
    through LDS 512 at a time, two or three times, with the next weights in flight over the refill.
    Alike, one unit has all 40 tokens, in three groups of up to 16."""
    p = _problem(40, 40, 2, 24, H, d_out, io, activation, True, seed=H, like_one=like_one)
    got = _run(p, 2, activation, cuda_device)
    _check(got, L.unit_layer(*p, 2, activation), IO[io])
