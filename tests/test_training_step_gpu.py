"""The training step's operators together, as a language model runs them: one step's loss and gradients
against the same step in float64, the clip on top, devices, streams and graphs.

The float64 step takes the fp32 operators' choice of units, so that no tie decides. Everything else is smooth:
with u = 2^-24, the products over up to 64 terms of order 1 are off by 64 u, and what follows by some tens of u
more each, so that a gradient is within 4000 u of the largest of its tensor (2.4e-4); 10^-3 is the bar."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


class Small:
    """``embed -> router -> units -> logits`` with a balance loss."""

    def __init__(self, dev, V=53, D=24, M=6, k=2, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weight(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g) * scale).to(dev).requires_grad_()

        self.V, self.D, self.M, self.k = V, D, M, k
        self.embed, self.router = weight(V, D), weight(M, D, scale=D ** -0.5)
        self.W, self.out = weight(M, D, D, scale=D ** -0.5), weight(V, D, scale=D ** -0.5)
        self.weights = [self.embed, self.router, self.W, self.out]

    def loss(self, tokens, target, valid):
        from hsn_amd import embedding, scoring, unit_router

        x = embedding.embed(tokens, self.embed, scale=2.0).flatten(0, 1)
        units, share, balance, counts = unit_router.choose_units(x @ self.router.t(), self.k, valid=valid.flatten())
        W = self.W[units.clamp(min=0)]
        o = ((x[:, None, None, :] @ W)[:, :, 0] * share[..., None]).sum(1)
        logprob, entropy = scoring.token_logprobs((o @ self.out.t()).view(*tokens.shape, self.V), target)
        live = valid.float().sum()
        return (-(logprob * valid).sum() / live + 0.1 * balance
                - 0.05 * (entropy * valid).sum() / live), units

    def loss64(self, weights, tokens, target, valid, units):
        embed, router, W, out = weights
        inside = ((tokens >= 0) & (tokens < self.V)).flatten()
        x = torch.where(inside[:, None], embed[tokens.flatten().clamp(0, self.V - 1)] * 2.0, 0.0)
        logits, keep = x @ router.t(), valid.flatten()
        at = units.clamp(min=0)
        share = torch.softmax(logits.gather(1, at), dim=1) * keep[:, None]
        load = torch.bincount(units[keep].flatten(), minlength=self.M).double()
        balance = self.M * (load / load.sum() * torch.softmax(logits[keep], dim=1).mean(0)).sum()
        o = ((x[:, None, None, :] @ W[at])[:, :, 0] * share[..., None]).sum(1)
        logp = torch.log_softmax(o @ out.t(), dim=1)
        entropy = -(logp.exp() * logp).sum(1)
        goal = target.flatten()
        given = (goal >= 0) & (goal < self.V)
        logprob = torch.where(given, logp.gather(1, goal.clamp(0, self.V - 1)[:, None])[:, 0], 0.0)
        live = keep.double().sum()
        return -(logprob * keep).sum() / live + 0.1 * balance - 0.05 * (entropy * keep).sum() / live


def _batch(dev, B=5, T=37, V=53, seed=1):
    g = torch.Generator().manual_seed(seed)
    text = torch.randint(0, V, (B, T + 1), generator=g)
    length = torch.randint(1, T + 1, (B, 1), generator=g)
    valid = torch.arange(T) < length
    tokens, target = torch.where(valid, text[:, :-1], -1), torch.where(valid, text[:, 1:], -1)
    return tokens.to(dev), target.to(dev), valid.to(dev)


def test_a_step_against_float64(cuda_device):
    from hsn_amd import grad_clip

    model, batch = Small(cuda_device), _batch(cuda_device)
    loss, units = model.loss(*batch)
    loss.backward()
    wide = [w.detach().cpu().double().requires_grad_() for w in model.weights]
    tokens, target, valid = (t.cpu() for t in batch)
    want = model.loss64(wide, tokens, target, valid, units.cpu())
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    for got, w in zip(model.weights, wide):
        off = (got.grad.cpu().double() - w.grad).abs().max()
        assert float(off) <= 1e-3 * float(w.grad.abs().max()), got.shape
    grads = [w.grad for w in model.weights]
    before = [g.clone() for g in grads]
    norm, coefficient = grad_clip.clip(grads, 0.1)
    norm64 = math.sqrt(sum(float((w.grad ** 2).sum()) for w in wide))
    assert abs(float(norm) - norm64) <= 1e-3 * norm64
    assert abs(float(coefficient) - 0.1 / (float(norm) + 1e-6)) <= 1e-12
    for g, b in zip(grads, before):
        assert torch.equal(g, (b.double() * coefficient).float())
    # padding has no gradient
    used = torch.zeros(model.V, dtype=torch.bool)
    used[tokens[valid]] = True
    assert not model.embed.grad.cpu()[~used].any()


def test_the_same_bits_and_a_captured_step(cuda_device):
    """The forward and the backward in one graph, replayed with other batches between eager steps."""
    from hsn_amd import embedding, grad_clip, scoring, unit_router

    model = Small(cuda_device, seed=3)
    batches = [_batch(cuda_device, seed=s) for s in range(3)]
    held = [t.clone() for t in batches[0]]
    weights = [w.detach() for w in model.weights]
    embed, router, _, out_w = weights

    @torch.no_grad()
    def step(tokens, target, valid):
        x = embedding.forward(tokens, embed)
        flat = x.flatten(0, 1)
        routed = unit_router.forward(flat @ router.t(), 2, valid=valid.flatten())
        scored = scoring.forward(flat @ out_w.t(), target.flatten(), top=4)
        d = scoring.backward(flat @ out_w.t(), target.flatten(), scored["stats"],
                             torch.full((flat.shape[0],), -0.01, device=cuda_device))
        d_x = d @ out_w + unit_router.backward(flat @ router.t(), routed["units"], routed["tally"],
                                               torch.ones_like(routed["shares"]), routed["balance"],
                                               valid=valid.flatten()) @ router
        d_embed = embedding.backward(tokens, d_x.view(*tokens.shape, -1), model.V)
        norm, coefficient = grad_clip.clip([d_embed], 0.01)
        return [scored["logprob"], scored["top_tokens"], routed["shares"], routed["balance"], d_embed, norm]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*held)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*held)
    for i in range(5):
        for h, b in zip(held, batches[i % 3]):
            h.copy_(b)
        graph.replay()
        eager = step(*batches[i % 3])
        torch.cuda.synchronize()
        for a, b in zip(results, eager):
            assert torch.equal(a, b)


def test_on_another_stream(cuda_device):
    """Each call runs on its tensors' device's current stream: two streams' steps side by side give what
    one gives."""
    model, batch = Small(cuda_device, seed=5), _batch(cuda_device, B=16, T=200, seed=4)

    def grads():
        loss, _ = model.loss(*batch)
        return [loss, *torch.autograd.grad(loss, model.weights)]

    want = grads()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(2):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(grads())
    torch.cuda.synchronize()
    for results in got:
        assert torch.equal(results[0], want[0])
        for a, b in zip(results[1:2], want[1:2]):  # the embedding's, by this package's kernels throughout
            torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-6)


MODULES = ("embedding", "scoring", "unit_router", "grad_clip")


def _everything(device):
    from hsn_amd import embedding, grad_clip, scoring, unit_router

    g = torch.Generator().manual_seed(3)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(device)

    tokens = torch.randint(0, 30, (9000,), generator=g).to(device)
    out = embedding.forward(tokens, rnd(30, 16))
    d_table = embedding.backward(tokens, out, 30)
    scored = scoring.forward(rnd(2, 300000), tokens[:2], top=3)
    d = scoring.backward(rnd(2, 40), tokens[:2], scored["stats"], scored["logprob"])
    routed = unit_router.forward(rnd(50, 8), 2)
    d_r = unit_router.backward(rnd(50, 8), routed["units"], routed["tally"], routed["shares"])
    norm, coefficient = grad_clip.clip([d_table, d], 1.0)
    return [out, d_table, scored["logprob"], scored["top_tokens"], d, routed["balance"], d_r, norm, coefficient,
            grad_clip.norm([d])]


def test_the_python_calls_make_the_tensors_device_current(cuda_device, monkeypatch):
    """The calls without the host helper, with a record of what is current at each launch."""
    import hsn_amd
    from hsn_amd import _lib

    modules = [__import__(f"hsn_amd.{name}", fromlist=["x"]) for name in MODULES]
    current, launched, call = [], [], _lib.call

    class Device(torch.cuda.device):
        def __enter__(self):
            current.append(self.idx)
            super().__enter__()

        def __exit__(self, *args):
            current.pop()
            return super().__exit__(*args)

    def recorded(name, *args):
        if not name.endswith("workspace"):
            launched.append((name, list(current)))
        call(name, *args)

    want = _everything(cuda_device)
    monkeypatch.setattr(torch.cuda, "device", Device)
    for module in modules:
        monkeypatch.setattr(module, "native_calls", lambda *names: None)
        monkeypatch.setattr(module, "call", recorded)
    monkeypatch.setattr(_lib, "call", recorded)
    for a, b in zip(_everything(cuda_device), want):
        assert torch.equal(a, b)
    assert launched == [(name, [0]) for name in (
        "hsn_embed_forward", "hsn_embed_backward", "hsn_score_forward", "hsn_score_backward",
        "hsn_unit_router_forward", "hsn_unit_router_backward", "hsn_clip", "hsn_clip")]
    assert hsn_amd.__version__


@pytest.mark.parametrize("helper", [True, False])
def test_on_a_second_device(cuda_device, monkeypatch, helper):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    if not helper:
        for name in MODULES:
            module = __import__(f"hsn_amd.{name}", fromlist=["x"])
            monkeypatch.setattr(module, "native_calls", lambda *names: None)
    want = _everything(cuda_device)
    got = _everything(torch.device("cuda", 1))
    assert torch.cuda.current_device() == 0
    for a, b in zip(got, want):
        assert a.device.index == 1 and torch.equal(a.cpu(), b.cpu())


def test_inference_tensors_and_mode(cuda_device):
    """Under inference mode, where tensors have no version."""
    from hsn_amd import grad_clip

    with torch.inference_mode():
        results = _everything(cuda_device)
        g = torch.ones(5, device=cuda_device)
        grad_clip.clip([g], 1.0)
    assert all(r.is_inference() for r in results)
