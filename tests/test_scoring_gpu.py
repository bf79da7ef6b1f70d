"""Log probabilities, entropy, alternatives and the gradient on the GPU against the float64 oracle.

Bars, with u = 2^-24 and x = l - max l, |x| < 64 in these rows: x is rounded (u |x|), its product with
log2 e too (2 u |x| more, the constant among it), and the exponential is right to 2^-22, so an exponential
is off by (3 |x| + 4) u of itself, on the average over p by at most 13 u where the mass lies within |x| < 3
(the sums add at most 64 terms a thread one by one, then 8 joins: 40 u). So log S is off by 60 u, log p_t by
that and 2 u |x|. The entropy is log S - W / S: its error is at most 130 u of max(1, |x| at the mass). A
probability is off by (3 |x| + 64) u of itself, 2^-16 at |x| = 64. Outputs of 16 bits add half a step."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training as R

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _problem(n, V, io, seed, masked=0.1, skipped=0.2):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, V, generator=g) * 3
    logits[torch.rand(n, V, generator=g) < masked] = -math.inf
    tokens = torch.randint(0, V, (n,), generator=g)
    tokens[torch.rand(n, generator=g) < skipped] = -1
    return logits.to(IO[io]), tokens


def _near(got, want, bar):
    """Equal where the oracle's value is not finite, within ``bar`` elsewhere."""
    got, want = got.double().cpu(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine].nan_to_num(1.0), want[~fine].nan_to_num(1.0))
    off = (got - want).abs()[fine]
    bar = (torch.as_tensor(bar, dtype=torch.float64) + torch.zeros_like(want))[fine]
    assert bool((off <= bar).all()), float((off - bar).max())


def _check(logits, tokens, dev, top=0, d_logprob=None, d_entropy=None):
    from hsn_amd import scoring

    n, V = logits.shape
    on = logits.to(dev), tokens.to(dev)
    out = scoring.forward(*on, top=top)
    logprob, entropy, best, best_logprob = R.score(logits, tokens, top)
    spread = 2 * (logprob.nan_to_num(0.0).clamp(min=-1e30).abs() + 1)
    _near(out["logprob"], logprob, (60 + spread) * U)
    _near(out["entropy"], entropy, 130 * U * entropy.nan_to_num(0.0).clamp(min=1.0))
    if top:
        assert out["top_tokens"].dtype == torch.int64
        assert torch.equal(out["top_tokens"].cpu(), best)
        spread = 2 * (best_logprob.nan_to_num(0.0).clamp(min=-1e30).abs() + 1)
        _near(out["top_logprobs"], best_logprob, (60 + spread) * U)
    else:
        assert out["top_tokens"] is None and out["top_logprobs"] is None
    bare = scoring.forward(*on, save=False)
    assert bare["stats"] is None and torch.equal(bare["logprob"].nan_to_num(), out["logprob"].nan_to_num())
    if d_logprob is None and d_entropy is None:
        return out
    d = scoring.backward(*on, out["stats"], *(None if t is None else t.to(dev)
                                              for t in (d_logprob, d_entropy)))
    assert d.shape == logits.shape and d.dtype == logits.dtype and d.is_contiguous()
    want = R.score_backward(logits, tokens, d_logprob, d_entropy)
    size = torch.zeros(n, 1, dtype=torch.float64)
    for t in (d_logprob, d_entropy):
        if t is not None:
            size = size + t.double().abs()[:, None]
    # p <= 1 off by 2^-16 of itself where it is smallest and by 80 u of itself where it is 1; times
    # h (log p + H), at most 64 + H < 80 of h, on top of errors of 200 u in log p + H
    p = torch.softmax(logits.double(), dim=1).nan_to_num(0.0)
    x = (logits.double() - logits.double().amax(dim=1, keepdim=True)).nan_to_num(0.0).clamp(min=-64).abs()
    factor = 1.0 if d_entropy is None else 1 + x + entropy.nan_to_num(0.0)[:, None]
    bar = size * p * ((3 * x + 80) * factor + (0 if d_entropy is None else 200)) * U + 2 * size * U * p
    bar = bar + want.abs().nan_to_num(0.0) * 2 * U + 1e-37
    if logits.dtype != torch.float32:
        bar = bar + want.abs().nan_to_num(0.0) * torch.finfo(logits.dtype).eps / 2
        bar = bar + (2.0 ** -25 if logits.dtype == torch.float16 else 0.0)  # half of the smallest step
    _near(d, want, bar)
    return out


SIZES = [(1, 1), (3, 2), (2, 7), (5, 64), (4, 500), (3, 1021), (2, 4096), (7, 4099), (2, 16385), (1, 40000)]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V", SIZES)
def test_values_and_gradient(cuda_device, n, V, io):
    logits, tokens = _problem(n, V, io, n + V)
    g = torch.Generator().manual_seed(1)
    d_logprob, d_entropy = torch.randn(n, generator=g), torch.randn(n, generator=g)
    _check(logits, tokens, cuda_device, min(V, 5), d_logprob, d_entropy)
    _check(logits, tokens, cuda_device, 0, d_logprob, None)
    _check(logits, tokens, cuda_device, 0, None, d_entropy)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 2, 20, 31, 32])
@pytest.mark.parametrize("n,V", [(3, 40), (2, 700), (2, 9001), (1, 50001), (40, 3000)])
def test_alternatives(cuda_device, n, V, top, io):
    logits, tokens = _problem(n, V, io, top + V)
    _check(logits, tokens, cuda_device, top)


@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "two values", "few finite"])
@pytest.mark.parametrize("V", [300, 5000, 33333])
def test_alternatives_in_awkward_rows(cuda_device, order, V):
    """Equal logits go to the lowest token; rows whose every next logit is a new largest one."""
    g = torch.Generator().manual_seed(V)
    if order == "equal":
        logits = torch.full((2, V), 1.5)
    elif order in ("ascending", "descending"):
        logits = torch.arange(V).float()[None].expand(2, V) * (64 / V)
        logits = logits.flip(1) if order == "descending" else logits
    elif order == "two values":
        logits = (torch.rand(2, V, generator=g) < 0.5).float()
    else:
        logits = torch.full((2, V), -math.inf)
        logits[0, torch.randint(0, V, (7,), generator=g)] = torch.randn(7, generator=g)
        logits[1, V - 1] = 3.0
    for io in ("f32", "f16"):
        _check(logits.to(IO[io]), torch.tensor([0, V - 1]), cuda_device, 32, torch.ones(2))


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [5, 600, 20000])
def test_masks_infinities_and_nan(cuda_device, V, io):
    logits, _ = _problem(9, V, io, V, masked=0.0)
    logits[1] = -math.inf  # nothing is left
    logits[2, 0], logits[3, V - 1] = math.nan, math.inf
    logits[4, :V - 1] = torch.finfo(logits.dtype).min  # a mask of the lowest value
    logits[5] = torch.finfo(logits.dtype).min  # of every value
    logits[6, 1:] = -math.inf  # one logit
    logits[7] = math.nan
    logits[8, : V // 2], logits[8, V - 1] = -math.inf, math.nan
    tokens = torch.tensor([V, 0, 0, 1, V - 1, 2, 0, 3, -1])
    d = torch.linspace(-1, 1, 9)
    _check(logits, tokens, cuda_device, 3, d, d.flip(0))


def test_the_largest_numbers(cuda_device):
    """Differences that leave fp32's range."""
    logits = torch.tensor([[3e38, -3e38, 0.0, 3e38], [-3e38, -3.4e38, -3e38, 0.0]])
    _check(logits, torch.tensor([0, 3]), cuda_device, 2, torch.ones(2))


@pytest.mark.parametrize("tokens", [torch.int64, torch.int32])
def test_strides(cuda_device, tokens):
    """Rows inside a wider product, at odd addresses, tokens and cotangents with strides of their own."""
    from hsn_amd import scoring

    for io in ("f32", "bf16"):
        wide, _ = _problem(6, 2100, io, 5)
        target = torch.randint(0, 999, (6, 3), generator=torch.Generator().manual_seed(0)).to(tokens)
        d = torch.randn(6, 2, generator=torch.Generator().manual_seed(1))
        wide, target, d = wide.to(cuda_device), target.to(cuda_device), d.to(cuda_device)
        for start in (0, 1, 3, 1101):
            view, t = wide[:, start:start + 999], target[:, 1]
            out, ref = scoring.forward(view, t, top=4), scoring.forward(view.contiguous(), t.contiguous(), top=4)
            # the sums' order goes by the rows' addresses, so either is within its bar of the formula's value
            assert torch.equal(out["top_tokens"], ref["top_tokens"])
            for name in ("logprob", "top_logprobs"):
                _near(out[name], ref[name].cpu(), 2 * (60 + 2 * (ref[name].cpu().abs().double() + 1)) * U)
            _near(out["entropy"], ref["entropy"].cpu(), 2 * 130 * U * ref["entropy"].cpu().double().clamp(min=1.0))
            ref = out
            back = scoring.backward(view, t, out["stats"], d[:, 0], d[:1, 1].expand(6))
            same = scoring.backward(view.contiguous(), t.contiguous(), ref["stats"],
                                    d[:, 0].contiguous(), d[:1, 1].expand(6).contiguous())
            assert torch.equal(back, same)
        turned = wide[::2, :999]
        got, want = (scoring.forward(x, target[::2, 0])["logprob"].cpu() for x in (turned, turned.contiguous()))
        _near(got, want, 2 * (60 + 2 * (want.abs().double() + 1)) * U)


def test_the_gradient_against_differences(cuda_device):
    from hsn_amd import scoring

    logits, tokens = _problem(3, 37, "f32", 11, masked=0.0)
    logits, tokens = logits.to(cuda_device).requires_grad_(), tokens.to(cuda_device)
    w, v = torch.tensor([[1.0, -2.0, 0.5], [0.3, 0.7, -1.0]], device=cuda_device)

    def loss(l):
        logprob, entropy = scoring.token_logprobs(l, tokens)
        return (logprob * w).sum() + (entropy * v).sum()

    grad, = torch.autograd.grad(loss(logits), logits)
    for i in range(3):
        for j in range(0, 37, 5):
            step = torch.zeros_like(logits)
            step[i, j] = 2.0 ** -6
            with torch.no_grad():
                slope = (loss(logits + step) - loss(logits - step)) / 2.0 ** -5
            # the third derivative is below 8 here (2^-12 / 6 of it), a loss off by 2^-20 each side
            assert abs(float(slope - grad[i, j])) <= 8 * 2.0 ** -12 / 6 + 2.0 ** -20 * 2 ** 5


def test_the_autograd_node(cuda_device):
    """Any leading shape, a cotangent that is expanded or absent, no second derivative, no gradient kept
    where none is wanted."""
    from hsn_amd import scoring

    logits, tokens = _problem(12, 250, "bf16", 3)
    logits, tokens = logits.to(cuda_device), tokens.to(cuda_device)
    leaf = logits.view(3, 4, 250).clone().requires_grad_()
    logprob, entropy = scoring.token_logprobs(leaf, tokens.view(3, 4))
    assert logprob.shape == entropy.shape == (3, 4) and logprob.dtype == torch.float32
    grad, = torch.autograd.grad(logprob.sum(), leaf, create_graph=True)
    out = scoring.forward(logits, tokens)
    assert torch.equal(grad.detach().view(12, 250), scoring.backward(logits, tokens, out["stats"],
                                                                    torch.ones(12, device=cuda_device)))
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    (scoring.token_logprobs(leaf, tokens.view(3, 4))[1].mean()).backward()
    assert torch.equal(leaf.grad.view(12, 250), scoring.backward(
        logits, tokens, out["stats"], None, torch.full((12,), 1 / 12, device=cuda_device)))
    turned = logits.view(3, 4, 250).transpose(0, 1)  # (made contiguous by either)
    assert torch.equal(scoring.token_logprobs(turned, tokens.view(3, 4).t())[0],
                       scoring.token_logprobs(turned.contiguous(), tokens.view(3, 4).t())[0])
    one = scoring.token_logprobs(logits[0], tokens[0])[0]
    assert one.shape == () and torch.equal(one, out["logprob"][0])
    with pytest.raises(ValueError, match="tokens must be"):
        scoring.token_logprobs(leaf, tokens)


def test_empty_and_one(cuda_device):
    from hsn_amd import scoring

    none = torch.zeros(0, 50, device=cuda_device)
    tokens = torch.zeros(0, dtype=torch.int64, device=cuda_device)
    out = scoring.forward(none, tokens, top=3)
    assert out["logprob"].shape == (0,) and out["top_tokens"].shape == (0, 3) and out["stats"].shape == (0, 4)
    assert scoring.backward(none, tokens, out["stats"], None).shape == (0, 50)


def test_the_same_bits_in_every_batch_and_from_graphs(cuda_device):
    """The same call gives the same bits, eager or replayed, with its own work between the replays."""
    from hsn_amd import scoring

    source = [_problem(3, 70001, "bf16", seed) for seed in range(3)]
    logits, tokens = (t.to(cuda_device) for t in source[0])
    d = torch.randn(3, generator=torch.Generator().manual_seed(0)).to(cuda_device)

    def both():
        out = scoring.forward(logits, tokens, top=9)
        return [*(out[k] for k in sorted(out)), scoring.backward(logits, tokens, out["stats"], d, d)]

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
        logits.copy_(source[i % 3][0])
        tokens.copy_(source[i % 3][1])
        for graph in graphs:
            graph.replay()
        eager = both()
        torch.cuda.synchronize()
        for results in held:
            for a, b in zip(results, eager):
                assert torch.equal(a, b)


@pytest.mark.parametrize("helper", [True, False])
def test_refusals(cuda_device, monkeypatch, helper):
    from hsn_amd import scoring

    if not helper:
        monkeypatch.setattr(scoring, "native_calls", lambda *names: None)
    logits, tokens = torch.zeros(4, 10, device=cuda_device), torch.zeros(4, dtype=torch.int64, device=cuda_device)
    stats = torch.zeros(4, 4, device=cuda_device)
    for bad in (logits.double(), logits[0], logits[None]):
        with pytest.raises(ValueError, match="logits must be"):
            scoring.forward(bad, tokens)
    with pytest.raises(ValueError, match="cpu"):
        scoring.forward(logits.cpu(), tokens)
    with pytest.raises(ValueError, match="V must be"):
        scoring.forward(logits[:, :0], tokens)
    with pytest.raises(ValueError, match="V must be"):
        scoring.forward(logits[:, :1].expand(4, 2 ** 24 + 1), tokens)
    with pytest.raises(ValueError, match="contiguous"):
        scoring.forward(logits.t(), tokens.new_zeros(10))
    for bad in (tokens[:3], tokens.float(), tokens.cpu(), tokens[None]):
        with pytest.raises(ValueError, match="tokens must be"):
            scoring.forward(logits, bad)
    for bad in (-1, 33):
        with pytest.raises(ValueError, match="top must be"):
            scoring.forward(logits, tokens, top=bad)
    for bad in (stats[:3], stats.double(), torch.zeros(4, 8, device=cuda_device)[:, ::2]):
        with pytest.raises(ValueError, match="stats must be"):
            scoring.backward(logits, tokens, bad, None)
    for bad in (stats[0, :3], tokens, stats):
        with pytest.raises(ValueError, match="d_logprob must be"):
            scoring.backward(logits, tokens, stats, bad)
        with pytest.raises(ValueError, match="d_entropy must be"):
            scoring.backward(logits, tokens, stats, None, bad)


def test_both_ways_of_calling_give_the_same(cuda_device, monkeypatch):
    from hsn_amd import scoring

    logits, tokens = (t.to(cuda_device) for t in _problem(5, 30001, "f32", 8))
    d = torch.randn(5, device=cuda_device)

    def everything():
        out = scoring.forward(logits, tokens, top=6)
        bare = scoring.forward(logits.half(), tokens.int(), save=False)
        return [out[k] for k in sorted(out)] + [bare["logprob"], bare["entropy"],
                                                scoring.backward(logits, tokens, out["stats"], d, d)]

    with_it = everything()
    monkeypatch.setattr(scoring, "native_calls", lambda *names: None)
    for a, b in zip(with_it, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype
