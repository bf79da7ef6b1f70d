"""The gradients' global norm and the clip on the GPU against the float64 oracle.

The norm: squares of fp32 (or narrower) numbers are exact in float64, N of them added in any order are off
by at most N 2^-53 of the sum, and the root halves that. The coefficient is then the oracle's to as much
and two roundings. What is scaled is one product in float64 rounded to fp32 and to the type, which the CPU
repeats bit for bit from the coefficient that the call returned."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _list(sizes, types, seed, scale=0.02, offset=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n + offset, generator=g) * scale).to(TYPES[types[i % len(types)]])[offset:]
            for i, n in enumerate(sizes)]


def _scaled(grads, coefficient):
    return [(g.double() * coefficient).float().to(g.dtype) for g in grads]


def _check(grads, dev, max_norm, where="in place"):
    from hsn_amd import grad_clip

    mine = [g.to(dev) for g in grads]
    assert all(m.data_ptr() for m in mine if m.numel())
    elements = sum(g.numel() for g in grads)
    want = R.grad_norm(grads)
    bar = (elements + 4) * 2.0 ** -53
    alone = grad_clip.norm(mine)
    assert alone.shape == (1,) and alone.dtype == torch.float64 and alone.device == dev
    assert abs(float(alone) - want) <= bar * want
    for a, b in zip(mine, grads):
        assert torch.equal(a.cpu(), b)
    out = None if where == "in place" else [torch.full_like(m, 7.0) for m in mine]
    norm, coefficient = grad_clip.clip(mine, max_norm, out=out)
    assert torch.equal(norm, alone)
    expect = R.clip_coefficient(want, max_norm)
    assert abs(float(coefficient) - expect) <= 2 * bar * expect
    for got, old, new in zip(mine if out is None else out, grads, _scaled(grads, float(coefficient))):
        assert torch.equal(got.cpu(), new), (old.shape, old.dtype)
    if out is not None:
        for a, b in zip(mine, grads):
            assert torch.equal(a.cpu(), b)


SIZES = {
    "one": [1],
    "chunk edges": [4095, 4096, 4097, 1, 8192, 8193, 12289],
    "empty ones": [0, 5, 0, 0, 4096, 0],
    "small": [64] * 48 + [4096] * 30 + [255] * 7,
    "several launches": [3] * 450,
    "long": [1, 300000, 17, 70001],
}


@pytest.mark.parametrize("where", ["in place", "out"])
@pytest.mark.parametrize("types", [("f32",), ("bf16",), ("f16",), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("sizes", SIZES)
def test_norm_and_clip(cuda_device, sizes, types, where):
    _check(_list(SIZES[sizes], types, len(sizes)), cuda_device, 0.05, where)


@pytest.mark.parametrize("max_norm", [0.0, 1e-9, 1.0, 1e9, math.inf])
def test_limits(cuda_device, max_norm):
    _check(_list([100, 5000], ("f32", "bf16"), 3), cuda_device, max_norm)
    _check(_list([100, 5000], ("f32", "f16"), 3), cuda_device, max_norm, "out")


@pytest.mark.parametrize("types", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_any_address(cuda_device, types, offset):
    """Views that begin off a 16-byte boundary, gradients and outputs differently."""
    from hsn_amd import grad_clip

    whole = _list([9001], (types,), 5)[0].to(cuda_device)
    to = torch.full_like(whole, 3.0)
    grads = [whole[offset:offset + 5000], whole[6000:]]
    out = [to[11 - offset:5011 - offset], to[6000:]]
    want = [g.cpu() for g in grads]
    _, coefficient = grad_clip.clip(grads, 0.01, out=out)
    for o, g in zip(out, _scaled(want, float(coefficient))):
        assert torch.equal(o.cpu(), g)
    # nothing beside them
    kept = torch.ones_like(to, dtype=torch.bool)
    kept[11 - offset:5011 - offset] = False
    kept[6000:] = False
    assert bool((to[kept] == 3.0).all())


def test_any_order_of_dimensions(cuda_device):
    from hsn_amd import grad_clip

    base = _list([6 * 50 * 70], ("f32",), 9)[0].view(6, 50, 70).to(cuda_device)
    turned = base.permute(2, 0, 1)
    want = turned.cpu()
    out = torch.empty(6, 50, 70, device=cuda_device).permute(2, 0, 1)
    _, coefficient = grad_clip.clip([turned], 0.1, out=[out])
    assert torch.equal(out.cpu(), (want.double() * float(coefficient)).float())
    # a dimension of one may have any stride
    row = base[0, :1].as_strided((1, 70), (999, 1))
    grad_clip.clip([row], 0.1, out=[torch.empty(1, 70, device=cuda_device)])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_not_finite_leaves_the_gradients(cuda_device, bad):
    from hsn_amd import grad_clip

    grads = [g.to(cuda_device) for g in _list([300, 4096], ("f32",), 2)]
    grads[1][4095] = bad
    before = [g.clone() for g in grads]
    norm, coefficient = grad_clip.clip(grads, 0.1)
    assert float(coefficient) == 1.0
    assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
    out = [torch.zeros_like(g) for g in grads]
    grad_clip.clip(grads, 0.1, out=out)
    for a, b, c in zip(grads, before, out):
        torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(c, b, rtol=0, atol=0, equal_nan=True)


def test_squares_beyond_fp32(cuda_device):
    """1e30 squared is above fp32's range and 1e-30 squared below it."""
    from hsn_amd import grad_clip

    for v in (1e30, 1e-30):
        g = torch.full((5000,), v, device=cuda_device)
        want = float(g[0].double()) * math.sqrt(5000)
        assert abs(float(grad_clip.norm([g])) - want) <= 1e-12 * want


def test_the_same_bits_every_time_and_from_graphs(cuda_device):
    from hsn_amd import grad_clip

    source = [g.to(cuda_device) for g in _list([64] * 20 + [30000] * 9, ("f32", "bf16"), 8)]
    grads = [g.clone() for g in source]
    first = grad_clip.clip(grads, 0.3)
    want = [g.clone() for g in grads]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        grad_clip.clip(grads, 0.3)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = grad_clip.clip(grads, 0.3)
    for i in range(4):
        for g, s in zip(grads, source):
            g.copy_(s * (i + 1))
        graph.replay()
        eager = [s * (i + 1) for s in source]
        got = grad_clip.clip(eager, 0.3)
        torch.cuda.synchronize()
        assert torch.equal(result[0], got[0]) and torch.equal(result[1], got[1])
        for a, b in zip(grads, eager):
            assert torch.equal(a, b)
        if i == 0:
            assert torch.equal(got[0], first[0])
            for a, b in zip(eager, want):
                assert torch.equal(a, b)


def test_a_clip_counts_as_an_update_in_place(cuda_device):
    from hsn_amd import grad_clip

    g = torch.ones(10, device=cuda_device)
    o = torch.ones(10, device=cuda_device)
    before = g._version, o._version
    grad_clip.norm([g])
    assert g._version == before[0]
    grad_clip.clip([g], 1.0, out=[o])
    assert (g._version, o._version) == (before[0], before[1] + 1)
    grad_clip.clip([g], 1.0)
    assert g._version == before[0] + 1


def test_the_coefficient_is_the_trainers(cuda_device):
    """What the clip scales equals the trainer's own scaling by the returned coefficient."""
    from hsn_amd import grad_clip, trainer

    grads = [g.to(cuda_device) for g in _list([5000, 64, 70000], ("f32",), 4)]
    other = [g.clone() for g in grads]
    _, coefficient = grad_clip.clip(grads, 0.2)
    assert trainer.scale64(other, coefficient)
    for a, b in zip(grads, other):
        assert torch.equal(a, b)


@pytest.mark.parametrize("helper", [True, False])
def test_refusals(cuda_device, monkeypatch, helper):
    from hsn_amd import grad_clip

    if not helper:
        monkeypatch.setattr(grad_clip, "native_calls", lambda *names: None)
    a = torch.ones(100, device=cuda_device)
    with pytest.raises(ValueError, match="empty"):
        grad_clip.norm([])
    with pytest.raises(ValueError, match="max_norm"):
        grad_clip.clip([a], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        grad_clip.clip([a], math.nan)
    with pytest.raises(ValueError, match="float64"):
        grad_clip.norm([a, a.double()])
    with pytest.raises(ValueError, match="cpu"):
        grad_clip.norm([a, a.cpu()])
    with pytest.raises(ValueError, match="must be a tensor"):
        grad_clip.norm([a, None])
    with pytest.raises(ValueError, match="dense"):
        grad_clip.norm([a[::2]])
    with pytest.raises(ValueError, match="dense"):
        grad_clip.norm([a[:1].expand(5)])
    with pytest.raises(ValueError, match="1 tensors"):
        grad_clip.clip([a], 1.0, out=[])
    with pytest.raises(ValueError, match="laid out"):
        grad_clip.clip([a], 1.0, out=[a[:50]])
    with pytest.raises(ValueError, match="laid out"):
        grad_clip.clip([a.view(10, 10)], 1.0, out=[torch.ones(10, 10, device=cuda_device).t()])
    with pytest.raises(ValueError, match="requires a gradient"):
        grad_clip.clip([a.clone().requires_grad_()], 1.0)
    # what is written overlaps: the same gradient twice, a part of one, another one's output
    with pytest.raises(RuntimeError, match="overlap"):
        grad_clip.clip([a, a], 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        grad_clip.clip([a[:60], a[59:]], 1.0)
    with pytest.raises(RuntimeError, match="overlaps gradient 1"):
        grad_clip.clip([a.clone(), a], 1.0, out=[a, torch.ones(100, device=cuda_device)])
    with pytest.raises(RuntimeError, match="overlaps gradient 0"):
        grad_clip.clip([a[:50]], 1.0, out=[a[1:51]])
    torch.cuda.synchronize()
    assert bool((a == 1.0).all())
    grad_clip.norm([a, a])  # only read: counted twice


def test_both_ways_of_calling_give_the_same(cuda_device, monkeypatch):
    from hsn_amd import grad_clip

    def everything():
        grads = [g.to(cuda_device) for g in _list([70, 0, 9000], ("f32", "bf16", "f16"), 6)]
        out = [torch.zeros_like(g) for g in grads]
        results = [grad_clip.norm(tuple(grads)), *grad_clip.clip(iter(grads), 0.1, out=out)]
        results += [*grad_clip.clip(grads, 0.2)]
        return results + grads + out + [torch.tensor(g._version) for g in grads]

    with_it = everything()
    monkeypatch.setattr(grad_clip, "native_calls", lambda *names: None)
    for a, b in zip(with_it, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype
