"""The embedding and its gradient on the GPU against the float64 oracle.

A row is one fp32 product rounded to its type. A sum of m cotangents is taken over spans of at most 1024
one by one and then over the spans, so it is off by at most (m + 2) 2^-24 of the sum of their sizes and
usually far less (bounded here by min(m, 1100) + m / 1024 + 4), the scale's product and the rounding to the
type by one step each."""

from __future__ import annotations

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}  # half of fp16's smallest step
U = 2.0 ** -24


def _tokens(shape, V, seed, padded=0.1, skew=True):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(shape, generator=g)
    t = ((V + 1.0) ** u - 1).long() if skew else (u * V).long()
    t = torch.randperm(V, generator=g)[t.clamp(0, V - 1)]
    strange = torch.tensor([-1, V, V + 5, -2 ** 40])[torch.randint(0, 4, shape, generator=g)]
    return torch.where(torch.rand(shape, generator=g) < padded, strange, t)


def _check(tokens, V, D, dev, table="f32", out="f32", scale=1.0, seed=0):
    from hsn_amd import embedding

    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g).to(IO[table])
    d = torch.randn(*tokens.shape, D, generator=g).to(IO[out])
    on = tokens.to(dev)
    got = embedding.forward(on, w.to(dev), scale=scale, dtype=IO[out])
    assert got.dtype == IO[out] and got.is_contiguous()
    assert got.shape == (*tokens.shape, D)
    outside = (tokens < 0) | (tokens >= V)
    rows = torch.where(outside[..., None], 0.0, w[tokens.masked_fill(outside, 0)].float() * scale)
    assert torch.equal(got.cpu(), rows.to(IO[out]))
    back = embedding.backward(on, d.to(dev), V, scale=scale, dtype=IO[table])
    assert back.shape == (V, D) and back.dtype == IO[table] and back.is_contiguous()
    want, size = R.embed_backward(tokens, d, V, scale)
    count = torch.bincount(tokens[~outside].reshape(-1), minlength=V)[:, None]
    bar = size * (count.clamp(max=1100) + count / 1024 + 4) * U
    bar = bar + want.abs() * torch.finfo(IO[table]).eps / 2 + TINY[table]
    off = (back.cpu().double() - want).abs()
    assert bool((off <= bar).all()), float((off - bar).max())
    assert not back.cpu()[count[:, 0] == 0].any()


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("table", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,V,D", [((1,), 1, 1), ((7,), 5, 3), ((3, 50), 40, 100), ((2, 33), 1000, 64),
                                       ((5, 101), 70, 520), ((60,), 20, 2055), ((40,), 9, 4), ((41,), 99, 5),
                                       ((42,), 80, 7), ((43,), 81, 8), ((44,), 65, 9)])
def test_rows_and_gradient(cuda_device, shape, V, D, table, out):
    _check(_tokens(shape, V, V + D), V, D, cuda_device, table, out, scale=1.0 if V % 2 else 2.5)


@pytest.mark.parametrize("n,V", [(4095, 700), (4096, 3), (4097, 50000), (2048 * 3, 1023), (2048 * 3 + 1, 1024),
                                 (12345, 262144), (9000, (1 << 20) + 1), (5000, 1 << 24), (16384, 900),
                                 (16385, 901), (20000, 262144), (17000, (1 << 20) + 1), (70000, 1023)])
@pytest.mark.parametrize("D", [1, 9])
def test_sorts(cuda_device, n, V, D):
    """Sizes around the sort's: one workgroup's list, whole tiles, one to three digits."""
    from hsn_amd import embedding

    if V * D > 1 << 24:
        tokens = _tokens((n,), 5000, n) + (V - 5000)  # the table's end
        d = torch.randn(n, D, generator=torch.Generator().manual_seed(1))
        back = embedding.backward(tokens.to(cuda_device), d.to(cuda_device), V)
        want, size = R.embed_backward(tokens - (V - 5000), d, 5000)
        inside = tokens < V
        assert not back[:V - 5000].any() or bool((tokens[inside] < V - 5000).any())
        off = (back[V - 5000:].cpu().double() - want).abs()
        assert bool((off <= size * 1000 * U).all())
    else:
        _check(_tokens((n,), V, n), V, D, cuda_device)


@pytest.mark.parametrize("kind", ["one token", "two tokens", "in order", "backwards", "all padding",
                                  "padding first", "all different"])
@pytest.mark.parametrize("n", [100, 5000, 40000])
def test_awkward_lists(cuda_device, n, kind):
    V = 60000 if kind in ("in order", "backwards", "all different") else 300
    tokens = {
        "one token": torch.full((n,), 299),
        "two tokens": torch.arange(n) % 2 * 299,
        "in order": torch.arange(n),
        "backwards": torch.arange(n).flip(0),
        "all padding": torch.full((n,), -1),
        "padding first": torch.where(torch.arange(n) < n // 2, -1, torch.arange(n) % 300),
        "all different": torch.randperm(V, generator=torch.Generator().manual_seed(n))[:n],
    }[kind]
    _check(tokens, V, 16, cuda_device, "bf16", "bf16")


@pytest.mark.parametrize("n", [1, 31, 127, 128, 129, 1000, 5000])
@pytest.mark.parametrize("V,D", [(2, 33), (40, 16), (40, 3), (700, 300)])
def test_runs_across_groups(cuda_device, n, V, D):
    """Short lists: runs within, across and over many of a workgroup's groups, and past its entries."""
    _check(_tokens((n,), V, n + D), V, D, cuda_device, "bf16" if D == 16 else "f32", "bf16")
    _check(_tokens((n,), V, n, padded=0.5, skew=False), V, D, cuda_device)


def test_short_lists_of_wide_rows(cuda_device):
    """More than 2^24 elements: chunks and joins after the short sort."""
    _check(_tokens((4200,), 30, 0), 30, 4100, cuda_device, "bf16", "bf16")


def test_a_long_list(cuda_device):
    """Large tiles and long chunks, wide rows; against sums in float64 on the GPU."""
    from hsn_amd import embedding

    for n, V, D in ((200001, 5000, 24), (150000, 100, 300)):
        tokens = _tokens((n,), V, n).to(cuda_device)
        d = torch.randn(n, D, generator=torch.Generator().manual_seed(0)).to(cuda_device)
        back = embedding.backward(tokens, d, V)
        keep = (tokens >= 0) & (tokens < V)
        want = torch.zeros(V, D, dtype=torch.float64, device=cuda_device)
        want.index_add_(0, tokens[keep], d[keep].double())
        size = torch.zeros_like(want).index_add_(0, tokens[keep], d[keep].double().abs())
        count = torch.bincount(tokens[keep], minlength=V)[:, None]
        bar = size * (count.clamp(max=1100) + count / 1024 + 4) * U
        assert bool(((back.double() - want).abs() <= bar).all())


def test_strides(cuda_device):
    """Slices of wider tensors, transposed batches, tables inside others, int32, more dimensions, none."""
    from hsn_amd import embedding

    V, D = 90, 40
    for io in ("f32", "bf16"):
        tokens = _tokens((6, 30), V, 1).to(cuda_device)
        wide = torch.randn(6, 30, 3 * D + 1, generator=torch.Generator().manual_seed(2)).to(IO[io]).to(cuda_device)
        table = torch.randn(V, 2 * D + 3, generator=torch.Generator().manual_seed(3)).to(IO[io]).to(cuda_device)
        for t, d in ((tokens, wide[..., D + 1:2 * D + 1]), (tokens[:, 3:20], wide[:, 3:20, 1:D + 1]),
                     (tokens.t(), wide.transpose(0, 1)[..., :D]), (tokens[::2, ::3], wide[::2, ::3, :D]),
                     (tokens[:, 4], wide[:, 7, 5:5 + D]), (tokens[2:3], wide[2:3, :, :D]),
                     (tokens[:, :1], wide[:, :1, :D]), (tokens, wide[:1, :1, :D].expand(6, 30, D)),
                     (tokens.view(2, 3, 30), wide.view(2, 3, 30, 3 * D + 1)[..., :D]),
                     (tokens.view(2, 3, 30).permute(2, 0, 1), wide.view(2, 3, 30, 3 * D + 1).permute(2, 0, 1, 3)[..., :D]),
                     (tokens[0, 0], wide[0, 0, :D])):
            for tt in (t, t.clamp(-9, V + 9).int()):  # -2^40 as int32 would be the token 0
                for w in (table[:, 1:D + 1], table[:, :D]):
                    got = embedding.forward(tt, w, scale=3.0)
                    assert torch.equal(got, embedding.forward(t.contiguous(), w.contiguous(), scale=3.0))
                    assert got.shape == (*t.shape, D)
                back = embedding.backward(tt, d, V)
                assert torch.equal(back, embedding.backward(t.contiguous(), d.contiguous(), V))


def test_no_token(cuda_device):
    from hsn_amd import embedding

    for shape in ((0,), (3, 0), (0, 5)):
        tokens = torch.zeros(shape, dtype=torch.int64, device=cuda_device)
        assert embedding.forward(tokens, torch.ones(4, 6, device=cuda_device)).shape == (*shape, 6)
        back = embedding.backward(tokens, torch.ones(*shape, 6, device=cuda_device), 70)
        assert back.shape == (70, 6) and not back.any()


def test_values_that_are_not_finite(cuda_device):
    """They reach their own token's row and column alone."""
    from hsn_amd import embedding

    tokens = torch.tensor([3, 1, 3, -1, 2], device=cuda_device)
    d = torch.ones(5, 8, device=cuda_device)
    d[0, 2], d[3], d[4, 5] = float("inf"), float("nan"), float("nan")
    back = embedding.backward(tokens, d, 5, scale=2.0).cpu()
    want = torch.zeros(5, 8)
    want[3], want[1], want[2] = 4.0, 2.0, 2.0
    want[3, 2], want[2, 5] = float("inf"), float("nan")
    torch.testing.assert_close(back, want, rtol=0, atol=0, equal_nan=True)
    table = torch.full((5, 8), float("nan"), device=cuda_device)
    assert not embedding.forward(tokens, table, scale=float("inf"))[3].any()


def test_the_autograd_node(cuda_device):
    from hsn_amd import embedding

    tokens = _tokens((4, 9), 20, 0).to(cuda_device)
    table = torch.randn(20, 12, device=cuda_device).requires_grad_()
    out = embedding.embed(tokens, table, scale=0.5, dtype=torch.bfloat16)
    assert out.dtype == torch.bfloat16
    grad, = torch.autograd.grad(out.sum(), table, create_graph=True)
    assert grad.dtype == torch.float32
    want = embedding.backward(tokens, torch.ones(4, 9, 12, dtype=torch.bfloat16, device=cuda_device), 20,
                              scale=0.5, dtype=torch.float32)
    assert torch.equal(grad.detach(), want)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    # the same table used twice: the gradients add
    (embedding.embed(tokens, table) * 2.0 + embedding.embed(tokens.flip(0), table)).sum().backward()
    inside = tokens[(tokens >= 0) & (tokens < 20)]
    count = torch.bincount(inside, minlength=20).float()
    assert torch.equal(table.grad, (3 * count)[:, None].expand(20, 12))


def test_the_gradient_against_differences(cuda_device):
    """The embedding is linear: a difference is the gradient up to the rounding of 9 sums of 27."""
    from hsn_amd import embedding

    tokens = torch.tensor([[1, 4, 1], [0, 1, 7], [4, 4, 4]], device=cuda_device)
    w = torch.randn(3, 3, 3, generator=torch.Generator().manual_seed(0)).to(cuda_device)
    table = torch.randn(6, 3, generator=torch.Generator().manual_seed(1)).to(cuda_device).requires_grad_()

    def loss(t):
        return (embedding.embed(tokens, t, scale=1.5).double() * w.double()).sum()

    grad, = torch.autograd.grad(loss(table), table)
    for i in range(6):
        for j in range(3):
            step = torch.zeros_like(table)
            step[i, j] = 0.5
            with torch.no_grad():
                slope = float(loss(table + step) - loss(table - step))
            # a row's product and the step each round by 2^-24 of at most 8, times at most 9 weights below 4
            assert abs(slope - float(grad[i, j])) <= 2 * 2 * 8 * 9 * 4 * U


def test_the_same_bits_every_time_and_from_graphs(cuda_device):
    from hsn_amd import embedding

    source = [_tokens((3, 2500), 900, seed).to(cuda_device) for seed in range(3)]
    tokens = source[0].clone()
    table = torch.randn(900, 72, device=cuda_device)
    d = torch.randn(3, 2500, 72, device=cuda_device)

    def both():
        return (embedding.forward(tokens, table), embedding.backward(tokens, d, 900),
                embedding.backward(tokens[:, :100], d[:, :100], 900))

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
        tokens.copy_(source[i % 3])
        for graph in graphs:
            graph.replay()
        eager = both()
        torch.cuda.synchronize()
        for results in held:
            for a, b in zip(results, eager):
                assert torch.equal(a, b)


@pytest.mark.parametrize("helper", [True, False])
def test_refusals(cuda_device, monkeypatch, helper):
    from hsn_amd import embedding

    if not helper:
        monkeypatch.setattr(embedding, "native_calls", lambda *names: None)
    table, tokens = torch.zeros(5, 8, device=cuda_device), torch.zeros(3, dtype=torch.int64, device=cuda_device)
    d = torch.zeros(3, 8, device=cuda_device)
    for bad in (table.double(), table[0]):
        with pytest.raises(ValueError, match="table must be"):
            embedding.forward(tokens, bad)
    with pytest.raises(ValueError, match="cpu"):
        embedding.forward(tokens, table.cpu())
    with pytest.raises(ValueError, match="row of the table"):
        embedding.forward(tokens, table.t())
    for bad in (table[:0], table[:, :0], table[:, :1].expand(5, 65537), table[:1].expand(2 ** 24 + 1, 8)):
        with pytest.raises(ValueError, match="V must be"):
            embedding.forward(tokens, bad)
    for bad in (tokens.float(), tokens.cpu()):
        with pytest.raises(ValueError, match="tokens must be"):
            embedding.forward(bad, table)
        with pytest.raises(ValueError, match="tokens must be"):
            embedding.backward(bad, d, 5)
    with pytest.raises(ValueError, match="2.26 tokens"):
        embedding.forward(tokens[:1].expand(2 ** 26), table)
    with pytest.raises(ValueError, match="2.26 tokens"):
        embedding.backward(tokens[:1].expand(2 ** 26), d[:1].expand(2 ** 26, 8), 5)
    for bad in (torch.float64, torch.int32):
        with pytest.raises(ValueError, match="dtype must be"):
            embedding.forward(tokens, table, dtype=bad)
        with pytest.raises(ValueError, match="dtype must be"):
            embedding.backward(tokens, d, 5, dtype=bad)
    for bad in (d[:2], d.double(), d[None]):
        with pytest.raises(ValueError, match="d_out must be"):
            embedding.backward(tokens, bad, 5)
    with pytest.raises(ValueError, match="cpu"):
        embedding.backward(tokens, d.cpu(), 5)
    with pytest.raises(ValueError, match="last dimension"):
        embedding.backward(tokens, torch.zeros(3, 16, device=cuda_device)[:, ::2], 5)
    for V in (0, -1, 2 ** 24 + 1):
        with pytest.raises(ValueError, match="V must be"):
            embedding.backward(tokens, d, V)


def test_both_ways_of_calling_give_the_same(cuda_device, monkeypatch):
    from hsn_amd import embedding

    tokens = _tokens((3, 700), 50, 4).to(cuda_device)
    table, d = torch.randn(50, 30, device=cuda_device).half(), torch.randn(3, 700, 30, device=cuda_device)

    def everything():
        return [embedding.forward(tokens, table, scale=0.3, dtype=torch.float32),
                embedding.forward(tokens[0, 0], table), embedding.forward(tokens[1].int(), table),
                embedding.backward(tokens, d, 50, scale=0.3, dtype=torch.float16),
                embedding.backward(tokens[:, 1], d[:, 1], 50), embedding.backward(tokens[0, 0], d[0, 0], 50)]

    with_it = everything()
    monkeypatch.setattr(embedding, "native_calls", lambda *names: None)
    for a, b in zip(with_it, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype
