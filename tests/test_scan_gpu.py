"""The gated linear recurrence on the GPU against the float64 oracle: forward, backward, the
autograd node, the single position, and what they refuse.

Tolerances. A gate's share is right to a few ulps (3e-7), and an error made at one position stays in
the state for about 1/b positions, so fp32 states are within 3e-7 / b of the exact ones, relative
to the largest |h| and |c| on the way; with the gates below (b above 0.005 but for a few positions)
that is 6e-5. The cotangents run through the same shares. A 16-bit output adds half a unit in its
last place."""

from __future__ import annotations

import pytest
import torch

from oracle import language as L

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STATE = 6e-5


def _close(got, want, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    got, want = got.nan_to_num(), want.nan_to_num()
    scale = max(1.0, float(want.abs().max())) if want.numel() else 1.0
    return got, want, scale


def _check(got, want, io=torch.float32, what=""):
    a, b, scale = _close(got, want, what)
    # 2^-24: the half unit of an fp16 value below its normal range
    room = STATE * scale + HALF_ULP[io] * b.abs() * (1 + 1e-3) + (2.0 ** -24 if io == torch.float16 else 0)
    off = (a - b).abs()
    assert bool((off <= room).all()), f"{what}: off by {float((off - room).max()):.3g} over the bound"


def _problem(B, T, D, io, dev, reset_p=0.05, h0=True, seed=0, layout="dense"):
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape, mean=0.0, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g) * scale + mean).to(dtype)

    if layout == "dense":
        y, gate = rnd(B, T, D, dtype=io).to(dev), rnd(B, T, D, mean=-1.0, dtype=io).to(dev)
    elif layout == "fused":  # both in one product's rows
        z = torch.cat([rnd(B, T, D), rnd(B, T, D, mean=-1.0)], 2).to(io).to(dev)
        y, gate = z[..., :D], z[..., D:]
    elif layout == "positions_first":
        y = rnd(T, B, D, dtype=io).to(dev).transpose(0, 1)
        gate = rnd(T, B, D, mean=-1.0, dtype=io).to(dev).transpose(0, 1)
    else:  # one element past an aligned start: no wide loads
        y = rnd(B * T * D + 1, dtype=io).to(dev)[1:].view(B, T, D)
        gate = rnd(B * T * D + 1, mean=-1.0, dtype=io).to(dev)[1:].view(B, T, D)
    reset = (torch.rand(B, T, generator=g) < reset_p).to(dev) if reset_p else None
    start = rnd(B, D).to(dev) if h0 else None
    d_h, d_h_T = rnd(B, T, D, dtype=io).to(dev), rnd(B, D).to(dev)
    return y, gate, reset, start, d_h, d_h_T


def _cpu(*ts):
    return [None if t is None else t.cpu() for t in ts]


def _both_ways(p, candidate="tanh"):
    from hsn_amd import scan

    y, gate, reset, h0, d_h, d_h_T = p
    io = y.dtype
    out = scan.forward(y, gate, reset, h0, candidate=candidate)
    d_y, d_gate, d_h0 = scan.backward(y, gate, out["marks"], reset, d_h, d_h_T,
                                      candidate=candidate)
    bare = scan.forward(y, gate, reset, h0, candidate=candidate, save=False)
    assert bare["marks"] is None and torch.equal(bare["h"], out["h"])
    c = _cpu(*p)
    h, h_T = L.scan_forward(*c[:4], candidate)
    want = L.scan_backward(*c, candidate)
    assert out["h"].dtype == d_y.dtype == d_gate.dtype == io
    _check(out["h"], h, io, "h")
    _check(out["h_T"], h_T, what="h_T")
    _check(d_y, want[0], io, "d_y")
    _check(d_gate, want[1], io, "d_gate")
    _check(d_h0, want[2], what="d_h0")
    return out, (d_y, d_gate, d_h0)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 7, 64), (3, 130, 100), (1, 257, 72), (2, 129, 8),
                                   (5, 16, 33), (1, 1000, 130), (4, 256, 512), (1, 2049, 20)])
def test_sizes(cuda_device, io, B, T, D):
    _both_ways(_problem(B, T, D, IO[io], cuda_device, seed=T + D))


@pytest.mark.parametrize("layout", ["fused", "positions_first", "odd_start"])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 104, 37])
def test_layouts(cuda_device, io, layout, D):
    _both_ways(_problem(3, 300, D, IO[io], cuda_device, layout=layout, seed=D), "linear")


@pytest.mark.parametrize("candidate", ["tanh", "linear"])
@pytest.mark.parametrize("reset_p", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("h0", [False, True])
def test_resets_and_start(cuda_device, candidate, reset_p, h0):
    _both_ways(_problem(2, 300, 96, torch.float32, cuda_device, reset_p, h0, seed=4), candidate)


@pytest.mark.parametrize("B,T,D", [(1, 5000, 64), (2, 9001, 24), (1, 4097, 200)])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_long_axis_in_few_rows(cuda_device, B, T, D, io):
    """Time is split over workgroups; the same bits come back every time."""
    p = _problem(B, T, D, IO[io], cuda_device, 1 / 700, seed=T)
    first = _both_ways(p)
    for _ in range(3):
        again = _both_ways(p)
        for a, b in zip((first[0]["h"], first[0]["h_T"], *first[1]),
                        (again[0]["h"], again[0]["h_T"], *again[1])):
            assert torch.equal(a, b)


def test_saturated_and_infinite_gates(cuda_device):
    """A gate of +inf writes the candidate, of -inf keeps the state; a share of 1e-30 is itself."""
    y, gate, reset, h0, d_h, d_h_T = _problem(1, 300, 64, torch.float32, cuda_device, 0.0, seed=9)
    gate[:, 10:40] = float("inf")
    gate[:, 100:200] = float("-inf")
    gate[:, 200:220] = -69.0
    gate[:, 230:240] = 200.0
    out, _ = _both_ways((y, gate, reset, h0, d_h, d_h_T))
    _check(out["h"][:, 199], out["h"][:, 100].double().cpu())  # joined apart: not the same bits


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T", [40, 3000])
def test_what_a_reset_drops_does_not_come_back(cuda_device, bad, T):
    """A state that is not finite stays in its own row and channel, and ends at the next reset,
    whatever lies between the two; without a reset a NaN stays to the end."""
    y, gate, _, h0, d_h, d_h_T = _problem(2, T, 64, torch.float32, cuda_device, 0.0, seed=2)
    reset = torch.zeros(2, T, dtype=torch.bool, device=cuda_device)
    reset[0, T - 7] = True
    h0[:, 5] = bad
    from hsn_amd import scan

    out = scan.forward(y, gate, reset, h0)
    finite = torch.isfinite(out["h"])
    assert bool(finite[0, T - 7:].all()) and not bool(finite[1, 0, 5])
    assert bool(torch.isfinite(out["h_T"][0]).all())
    rest = [c for c in range(64) if c != 5]
    assert bool(finite[:, :, rest].all())
    if bad != bad:
        assert not bool(finite[0, :T - 7, 5].any()) and not bool(finite[1, :, 5].any())
    want, _ = L.scan_forward(*_cpu(y, gate, reset, h0))
    _check(out["h"][0, T - 7:], want[0, T - 7:])
    # backward: the cotangent that the reset drops is exactly absent before it
    d_h[0, T - 7:, 9] = bad
    d_y, d_gate, _ = scan.backward(y, gate, out["marks"], reset, d_h, None)
    assert bool(torch.isfinite(d_y[0, :T - 7, 9]).all())
    assert not bool(torch.isfinite(d_y[0, T - 7, 9]))


def test_a_nan_candidate_reaches_later_positions_until_the_reset(cuda_device):
    y, gate, _, h0, _, _ = _problem(1, 600, 16, torch.float32, cuda_device, 0.0, seed=3)
    y[0, 100, 3] = float("nan")
    gate[0, 150, 7] = float("nan")
    reset = torch.zeros(1, 600, dtype=torch.bool, device=cuda_device)
    reset[0, 500] = True
    from hsn_amd import scan

    got = scan.forward(y, gate, reset, h0)["h"]
    nan = torch.isnan(got[0]).cpu()
    want = torch.zeros(600, 16, dtype=torch.bool)
    want[100:500, 3] = True
    want[150:500, 7] = True
    assert torch.equal(nan, want)


def test_empty(cuda_device):
    from hsn_amd import scan

    h0 = torch.randn(3, 10, device=cuda_device)
    y = torch.empty(3, 0, 10, device=cuda_device)
    out = scan.forward(y, y, None, h0)
    assert out["h"].shape == (3, 0, 10) and torch.equal(out["h_T"], h0)
    assert torch.equal(scan.forward(y, y)["h_T"], torch.zeros_like(h0))
    d_y, d_gate, d_h0 = scan.backward(y, y, out["marks"], None, None, h0)
    assert d_y.numel() == d_gate.numel() == 0 and torch.equal(d_h0, h0)
    none = torch.empty(0, 5, 10, device=cuda_device)
    out = scan.forward(none, none)
    assert out["h"].shape == (0, 5, 10) and out["h_T"].shape == (0, 10)
    assert scan.backward(none, none, out["marks"], None, none)[2].shape == (0, 10)
    assert scan.step(none[:, 0], none[:, 0], h0).shape == (0, 10)


def test_absent_cotangents(cuda_device):
    from hsn_amd import scan

    y, gate, reset, h0, d_h, d_h_T = _problem(2, 150, 48, torch.float32, cuda_device, seed=6)
    marks = scan.forward(y, gate, reset, h0)["marks"]
    for a, b in ((None, d_h_T), (d_h, None), (None, None)):
        got = scan.backward(y, gate, marks, reset, a, b)
        want = L.scan_backward(*_cpu(y, gate, reset, h0, a, b))
        for g, w in zip(got, want):
            _check(g, w)


@pytest.mark.parametrize("candidate", ["tanh", "linear"])
def test_autograd(cuda_device, candidate):
    """The node's gradients against float64 autograd, with an expanded cotangent (a sum's), a
    broadcast gate, and a second window that carries the state."""
    from hsn_amd import scan

    y, gate, reset, h0, _, _ = _problem(2, 200, 24, torch.float32, cuda_device, seed=8)
    gate = gate[:, :, :1].clone()  # one gate for all channels: its gradient is the channels' sum

    def loss(y, gate, h0, run):
        gates = gate.expand(-1, -1, y.shape[2])
        gates = gates if run is None else gates.contiguous()
        cut = 120
        parts = []
        for lo, hi in ((0, cut), (cut, 200)):
            r = reset[:, lo:hi].contiguous()
            if run is None:
                h, now = [], h0
                c = torch.tanh(y) if candidate == "tanh" else y
                b = torch.sigmoid(gates)
                for t in range(lo, hi):
                    now = torch.where(reset[:, t, None].to(y.device), torch.zeros_like(now), now)
                    now = now + b[:, t] * (c[:, t] - now)
                    h.append(now)
                h = torch.stack(h, 1)
            else:
                h, now = run(y[:, lo:hi], gates[:, lo:hi], r, h0, candidate=candidate)
            h0 = now
            parts.append(h.sum())
        return parts[0] + 2 * parts[1] + (now * now).sum()

    got_in = [t.clone().requires_grad_() for t in (y, gate, h0)]
    got = torch.autograd.grad(loss(*got_in, scan.gated_scan), got_in)
    want_in = [t.double().cpu().requires_grad_() for t in (y, gate, h0)]
    reset = reset.cpu()
    want = torch.autograd.grad(loss(*want_in, None), want_in)
    for g, w in zip(got, want):
        _check(g, w)


def test_the_state_alone_carries_a_gradient(cuda_device):
    from hsn_amd import scan

    y, gate, reset, h0, _, d = _problem(2, 30, 12, torch.float32, cuda_device, seed=5)
    h0.requires_grad_()
    _, h_T = scan.gated_scan(y, gate, reset, h0)
    (got,) = torch.autograd.grad((h_T * d).sum(), [h0])
    want = L.scan_backward(*_cpu(y, gate, reset, h0.detach(), None, d))[2]
    _check(got, want)


def test_offsets_past_31_bits(cuda_device):
    """Rows and positions whose offsets in elements and bytes pass 2^31."""
    from hsn_amd import scan

    B, T, D = 2, 3, 64
    far = 2 ** 31 + 64
    room = torch.empty(far + 2 * 2 ** 20 + T * D, dtype=torch.bfloat16, device=cuda_device)
    y = room.as_strided((B, T, D), (far, D, 1))
    src, gate, reset, h0, d_h, d_h_T = _problem(B, T, D, torch.bfloat16, cuda_device, seed=1)
    y.copy_(src)
    a, b = scan.forward(y, gate, reset, h0), scan.forward(src, gate, reset, h0)
    assert torch.equal(a["h"], b["h"])
    wide = room.as_strided((1, 3, D), (0, 2 ** 30 + 64, 1))  # the last position past 2^31
    wide.copy_(src[:1])
    a = scan.forward(wide, gate[:1], None, h0[:1].contiguous())
    b = scan.forward(src[:1], gate[:1], None, h0[:1].contiguous())
    assert torch.equal(a["h"], b["h"])
    ga = scan.backward(wide, gate[:1], a["marks"], None, wide)
    gb = scan.backward(src[:1], gate[:1], b["marks"], None, src[:1])
    assert all(torch.equal(x, z) for x, z in zip(ga, gb))


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,S,D", [(1, 1, 1), (5, 9, 33), (32, 256, 512), (3, 3, 100), (17, 40, 72)])
@pytest.mark.parametrize("candidate", ["tanh", "linear"])
def test_step(cuda_device, io, n, S, D, candidate):
    from hsn_amd import scan

    g = torch.Generator().manual_seed(n + D)
    z = torch.randn(n, 2 * D, generator=g).to(IO[io]).to(cuda_device)
    y, gate = z[:, :D], z[:, D:]
    state = torch.randn(S, D, generator=g)
    rows = torch.randperm(S, generator=g)[:n].to(torch.int32)
    rows[n // 2] = [-1, S, -7][n % 3] if n > 1 else rows[0]
    reset = torch.rand(n, generator=g) < 0.3
    for r, f in ((rows, reset), (None, None)):
        pool = state.to(cuda_device)
        h = scan.step(y, gate, pool, rows=None if r is None else r.to(cuda_device),
                      reset=None if f is None else f.to(cuda_device), candidate=candidate)
        want, after = L.scan_step(*_cpu(y, gate), state, r, f, candidate)
        _check(h, want, IO[io], "h")
        _check(pool, after, what="state")
        touched = set(range(n)) if r is None else set(r.tolist())
        for row in set(range(S)) - touched:
            assert torch.equal(pool[row].cpu(), state[row])


def test_step_of_many_sequences(cuda_device):
    """More sequences than one dimension of a grid holds workgroups."""
    from hsn_amd import scan

    n, D = 70001, 3
    g = torch.Generator().manual_seed(1)
    y, gate = torch.randn(n, D, generator=g), torch.randn(n, D, generator=g)
    state = torch.randn(n, D, generator=g)
    pool = state.to(cuda_device)
    h = scan.step(y.to(cuda_device), gate.to(cuda_device), pool)
    b = torch.sigmoid(gate.double())
    want = state.double() + b * (torch.tanh(y.double()) - state.double())
    _check(h, want)
    _check(pool, want)


def test_a_second_derivative_is_refused(cuda_device):
    from hsn_amd import scan

    y, gate, _, _, _, _ = _problem(1, 20, 4, torch.float32, cuda_device, 0.0)
    y.requires_grad_()
    h, _ = scan.gated_scan(y, gate)
    (d,) = torch.autograd.grad((h * h).sum(), [y], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_step_by_step_is_the_scan(cuda_device):
    """Decoding position by position gives the window's states (the same arithmetic; the scan joins
    spans, so the last bits may differ)."""
    from hsn_amd import scan

    y, gate, reset, h0, _, _ = _problem(3, 40, 64, torch.float32, cuda_device, seed=12)
    want = scan.forward(y, gate, reset, h0)
    state = h0.clone()
    for t in range(40):
        h = scan.step(y[:, t], gate[:, t], state, reset=reset[:, t].contiguous())
        _check(h, want["h"][:, t].double().cpu())
    _check(state, want["h_T"].double().cpu())


def test_on_another_stream_and_in_a_graph(cuda_device):
    """The calls run on the current stream and may be captured; every replay equals the eager
    result."""
    from hsn_amd import scan

    p = _problem(1, 3000, 64, torch.float32, cuda_device, seed=21)
    y, gate, reset, h0, d_h, d_h_T = p

    def both():
        out = scan.forward(y, gate, reset, h0)
        return out["h"], out["h_T"], *scan.backward(y, gate, out["marks"], reset, d_h, d_h_T)

    want = [t.clone() for t in both()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(3):
        y.copy_(torch.randn(y.shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        now = both()
        assert all(torch.equal(a, b) for a, b in zip(held, now))


def test_refusals(cuda_device):
    from hsn_amd import scan

    y, gate, reset, h0, d_h, d_h_T = _problem(2, 20, 8, torch.float32, cuda_device)
    marks = scan.forward(y, gate, reset, h0)["marks"]
    state = torch.zeros(4, 8, device=cuda_device)
    bad = [
        lambda: scan.forward(y, gate[:, :-1]),
        lambda: scan.forward(y, gate.bfloat16()),
        lambda: scan.forward(y.double(), gate.double()),
        lambda: scan.forward(y.transpose(1, 2), gate.transpose(1, 2)),
        lambda: scan.forward(y[0], gate[0]),
        lambda: scan.forward(y.cpu(), gate.cpu()),
        lambda: scan.forward(y, gate.cpu()),
        lambda: scan.forward(y, gate, reset.int()),
        lambda: scan.forward(y, gate, reset[:, :-1]),
        lambda: scan.forward(y, gate, reset, h0.bfloat16()),
        lambda: scan.forward(y, gate, reset, h0[:1]),
        lambda: scan.forward(y, gate, reset, h0, candidate="relu"),
        lambda: scan.forward(y[..., :0], gate[..., :0]),
        lambda: scan.backward(y, gate, marks[:, :, :4], reset, d_h),
        lambda: scan.backward(y, gate, marks, reset, d_h.bfloat16()),
        lambda: scan.backward(y, gate, marks, reset, d_h, d_h_T.double()),
        lambda: scan.step(y[:, 0], gate[:, 0], state.bfloat16()),
        lambda: scan.step(y[:, 0], gate[:, 0], state, rows=torch.zeros(2, dtype=torch.int64,
                                                                       device=cuda_device)),
        lambda: scan.step(y[:, 0], gate[:, 0], state[:, :4]),
        lambda: scan.step(y[:, 0], gate[:, 0], state, reset=reset[:, :1].expand(2, 2)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):  # more sequences than states, and no rows
        scan.step(y[:, 0], gate[:, 0], state[:1])


@pytest.fixture(params=["helper", "python"])
def either_way(request, monkeypatch):
    """With the host helper, and with the Python checks alone."""
    if request.param == "python":
        from hsn_amd import scan

        monkeypatch.setattr(scan, "native_calls", lambda *names: None)


def test_step_counts_as_an_update_in_place(cuda_device, either_way):
    """A pool that an operation has saved for its gradient and that the step then updates is refused by
    that operation's backward, as after any update in place; a step of no sequences updates nothing."""
    from hsn_amd import scan

    y = torch.randn(2, 8, device=cuda_device)
    w = torch.ones(3, 8, device=cuda_device, requires_grad=True)
    state = torch.randn(3, 8, device=cuda_device)
    out = (w * state).sum()
    scan.step(y[:0], y[:0], state)
    torch.autograd.grad(out, [w], retain_graph=True)
    version = state._version
    scan.step(y, y, state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, [w])
    with torch.inference_mode():  # such a pool keeps no version, and no operation saves it
        pool = torch.zeros(2, 8, device=cuda_device)
        scan.step(y, y, pool)
    scan.step(y, y, pool)
    assert bool((pool != 0).any())


def test_step_refuses_what_needs_a_gradient(cuda_device, either_way):
    from hsn_amd import scan

    y, state = torch.randn(2, 8, device=cuda_device), torch.zeros(2, 8, device=cuda_device)
    for which in range(3):
        args = [y.clone(), y.clone(), state.clone()]
        args[which].requires_grad_()
        with pytest.raises(ValueError, match="no gradient"):
            scan.step(*args)
        assert bool((args[2] == 0).all())
        with torch.no_grad():
            assert not scan.step(*args).requires_grad


@pytest.mark.parametrize("T", [40, 3000])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_a_nan_gate_after_a_reset_stays_behind_it(cuda_device, T, io):
    """Backward, a NaN gate makes the cotangents before it NaN only down to the next reset: the
    positions before that reset belong to another document. The gate follows the reset in one
    thread's segment, in one wave, in one workgroup, and in another tile."""
    from hsn_amd import scan

    y, gate, _, h0, d_h, d_h_T = _problem(1, T, 64, IO[io], cuda_device, 0.0, seed=14)
    resets = [20] if T == 40 else [20, 700, 1400, 2000]
    after = [2, 9, 17] if T == 40 else [2, 9, 17, 90, 250, 500]
    reset = torch.zeros(1, T, dtype=torch.bool, device=cuda_device)
    reset[0, resets] = True
    for channel, far in enumerate(after):
        for at in resets:
            gate[0, at + far, channel] = float("nan")
    gate[0, resets[-1], 40] = -float("nan")  # the reset's own position
    d_h[0, -1, 41] = float("inf")
    p = (y, gate, reset, h0, d_h, None)
    marks = scan.forward(y, gate, reset, h0)["marks"]
    got = scan.backward(y, gate, marks, reset, d_h, None)
    want = L.scan_backward(*_cpu(*p))
    for g, w, what in zip(got, want, ("d_y", "d_gate", "d_h0")):
        assert torch.equal(torch.isfinite(g).cpu(), torch.isfinite(w)), what
        finite = torch.isfinite(w)
        _check(g.cpu()[finite], w[finite], g.dtype, what)
    assert bool(torch.isfinite(got[2]).all())
    assert bool(torch.isfinite(got[0][0, :resets[0]]).all())


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 300])
def test_positions_masked_by_the_lowest_value_keep_the_state(cuda_device, io, T):
    """Masked positions hold the type's lowest value in the gate and in the linear candidate alike
    (a mask laid over both halves of one product): their share is 0, so that candidate counts for
    nothing, in the state as in the gradients. The definition's product is 0 there, exactly."""
    from hsn_amd import scan

    y, gate, _, h0, d_h, d_h_T = _problem(2, T, 64, IO[io], cuda_device, 0.0, seed=T)
    masked = torch.zeros(T, dtype=torch.bool)
    masked[::3] = True
    low = torch.finfo(IO[io]).min
    y[:, masked], gate[:, masked] = low, low
    y[0, masked] = -low
    gate[0, masked] = -float("inf")
    out, grads = _both_ways((y, gate, None, h0, d_h, d_h_T), "linear")
    assert float(grads[0][:, masked].abs().max()) == 0.0
    assert float(grads[1][:, masked].abs().max()) == 0.0
    assert torch.equal(out["h"][:, 0], h0.to(IO[io]))
    pool = h0.clone()
    h = scan.step(y[:, 0], gate[:, 0], pool, candidate="linear")
    assert torch.equal(pool, h0) and torch.equal(h, h0.to(IO[io]))


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
def test_an_infinite_linear_candidate_has_a_finite_gradient(cuda_device, io):
    """The linear candidate's derivative is 1 whatever its value: d_y of an infinite candidate is the
    share of its cotangent."""
    from hsn_amd import scan

    y, gate, _, h0, d_h, d_h_T = _problem(1, 50, 64, IO[io], cuda_device, 0.0, seed=15)
    y[0, 20, 3], y[0, 30, 5] = float("inf"), -float("inf")
    marks = scan.forward(y, gate, None, h0, candidate="linear")["marks"]
    got = scan.backward(y, gate, marks, None, d_h, d_h_T, candidate="linear")[0]
    want = L.scan_backward(*_cpu(y, gate, None, h0, d_h, d_h_T), "linear")[0]
    assert bool(torch.isfinite(want).all())
    _check(got, want, IO[io])


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("candidate", ["tanh", "linear"])
@pytest.mark.parametrize("B,T,D,reset_p,layout", [
    (256, 300, 40, 0.05, "fused"), (64, 129, 250, 0.0, "dense"), (128, 1000, 99, 1 / 300, "dense"),
    (300, 257, 7, 0.05, "fused"), (260, 512, 64, 1 / 100, "positions_first"), (256, 1024, 33, 0.0, "odd_start")])
def test_a_walk_over_several_tiles(cuda_device, io, candidate, B, T, D, reset_p, layout):
    """Rows and channels enough for the GPU and a few tiles: a workgroup walks them one after the other,
    with the next one's loads in flight. Two to eight tiles, the last one whole, ragged or of a
    single position, one and two channels a thread."""
    import ctypes

    from hsn_amd import _lib

    size = ctypes.c_int64(-1)
    for backward in (0, 1):  # no exchange between workgroups, and more than a tile backward and in fp32
        _lib.call("hsn_scan_workspace", B, T, D, {"f32": 0, "f16": 1, "bf16": 2}[io], backward, ctypes.byref(size))
        assert size.value == 0
    assert 128 < T <= 1024
    _both_ways(_problem(B, T, D, IO[io], cuda_device, reset_p, seed=B + D, layout=layout), candidate)


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_what_a_reset_drops_in_a_walk(cuda_device, io):
    """The walk's carry over tiles: a start state of infinity or NaN ends at the reset, forward, and a
    cotangent of either backward."""
    from hsn_amd import scan

    B, T, D = 256, 700, 20
    y, gate, _, h0, d_h, d_h_T = _problem(B, T, D, IO[io], cuda_device, 0.0, seed=31)
    reset = torch.zeros(B, T, dtype=torch.bool, device=cuda_device)
    at = torch.arange(B) * 2 + 100  # in every tile but the first and the last
    reset[torch.arange(B), at] = True
    before = (torch.arange(T)[None, :] < at[:, None]).to(cuda_device)
    h0[:, 5], h0[:, 6] = float("inf"), float("nan")
    d_h_T[:, 8], d_h_T[:, 9] = float("nan"), float("inf")
    out = scan.forward(y, gate, reset, h0)
    clean = scan.forward(y, gate, reset, torch.where(torch.isfinite(h0), h0, 0.0))
    after = ~before[..., None].expand(-1, -1, D)
    assert torch.equal(out["h"][after], clean["h"][after]) and torch.equal(out["h_T"], clean["h_T"])
    assert bool(torch.isnan(out["h"][..., 6][before]).all())
    got = scan.backward(y, gate, clean["marks"], reset, d_h, d_h_T)
    want = scan.backward(y, gate, clean["marks"], reset, d_h, torch.where(torch.isfinite(d_h_T), d_h_T, 0.0))
    rows = before[..., None].expand(-1, -1, D)
    assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows])
    assert torch.equal(got[2], want[2])
    assert bool(torch.isnan(got[0][..., 8][~before]).all())


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_small_shares_are_right_to_parts_of_themselves(cuda_device, io):
    """One position from a zero state: h = b y, so h_T / y is the share itself, d_y = b d_h_T, and its
    complement shows in d_h0 = a d_h_T where a is small (large gates). The exponent's rounding is
    2^-24 |g| log2(e) in base 2, that is |g| 2^-24 of the share, log2(e)'s own |g| 1.4e-8; a few
    ulps for the rest."""
    from hsn_amd import scan

    g = torch.tensor([-0.25, -1.0, -12.0, -30.0, -69.0, -80.0]).repeat(8)
    g = torch.cat([g, -g]).to(IO[io])
    y = torch.linspace(0.5, 2.0, g.numel()).to(IO[io])
    one = torch.ones(1, g.numel())
    args = [t.reshape(1, 1, -1).to(cuda_device) for t in (y, g)]
    out = scan.forward(*args, candidate="linear")
    _, _, d_h0 = scan.backward(*args, out["marks"], None, None, one.to(cuda_device), candidate="linear")
    g, y = g.double(), y.double()
    room = g.abs() * (2.0 ** -24 + 1.4e-8) + 8 * 2.0 ** -24
    b, a = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    assert bool(((out["h_T"][0].double().cpu() / (b * y) - 1).abs() <= room).all())
    assert bool(((d_h0[0].double().cpu() / a - 1).abs() <= room).all())


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
def test_small_candidates_are_right_to_parts_of_themselves(cuda_device, io):
    """tanh(y) itself, from a gate of +inf: h_T = tanh(y). From the limit on it is 1 - 2 / (1 + e): the
    exponential, the sum and the reciprocal are off by 2.5 ulps of 1/2 together, twice that and the
    last rounding 2.7e-7 of 1. Below the limit the series' next term (17 y^7 / 315 in fp32, y^3 / 3 in
    16 bits) and four roundings."""
    from hsn_amd import scan

    y = torch.cat([torch.logspace(-6, 0.5, 256), torch.tensor([0.125, 0.1249, 0.0078125, 0.0078])])
    y = torch.cat([y, -y]).to(IO[io])
    gate = torch.full_like(y, float("inf"))
    args = [t.reshape(1, 1, -1).to(cuda_device) for t in (y, gate)]
    got = scan.forward(*args, save=False)["h_T"][0].double().cpu()
    want = torch.tanh(y.double())
    off = (got / want - 1).abs()
    if io == "f32":
        room = torch.where(y.abs() < 0.125, 17 / 315 * y.double() ** 6 + 4 * 2.0 ** -24, 2.7e-7 / want.abs())
    else:
        room = torch.where(y.abs() < 0.0078125, y.double() ** 2 / 3 + 2.0 ** -24, 2.7e-7 / want.abs())
    assert bool((off <= room).all()), float(off.max())
