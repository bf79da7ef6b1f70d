"""The choice of a token on the GPU against the float64 oracle. Every weight is within 2e-6 of
itself and 2^-40 of the largest, so a token is the oracle's wherever ``u`` and the filters' edges
are more than 1e-5 of the mass away from a place where the answer changes; the oracle gives the
distance for ``u``, and the problems below keep the edges away from it."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import language as L

pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
AWAY = 1e-5


def _rows(n, V, io, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, V, generator=g) * spread).to(IO[io]), torch.rand(n, generator=g)


def _away(logits, t, k, p, m):
    """Whether the filters' edges are away from where their answer changes."""
    if not t > 0:
        return True
    kept = L.kept_tokens(logits, t, k, 1.0, 0.0)
    total, run, ok = sum(w for _, w in kept), 0.0, True
    for _, w in kept:
        if p < 1:
            ok &= abs(run / total - p) > AWAY or run == 0
        if m > 0 and w < 1:
            ok &= abs(w - m) > AWAY * m
        run += w
    return ok


def _check(logits, u, settings, dev):
    """``settings``: one ``(t, k, p, m)`` a row; every row that is away from an edge has to agree,
    and most rows have to be."""
    from hsn_amd import sampling

    t, k, p, m = (torch.tensor(c, dtype=d) for c, d in zip(
        zip(*settings), (torch.float32, torch.int32, torch.float32, torch.float32)))
    got = sampling.sample(logits.to(dev), u.to(dev), temperature=t.to(dev), top_k=k.to(dev),
                          top_p=p.to(dev), min_p=m.to(dev))
    assert got.dtype == torch.int64 and got.shape == (logits.shape[0],)
    checked = 0
    for i, token in enumerate(got.tolist()):
        row = logits[i].float()
        s = tuple(float(c[i]) for c in (t, k, p, m))
        s = (s[0], int(s[1]), s[2], s[3])
        want, margin = L.sample(row, float(u[i]), *s)
        if margin > AWAY and _away(row, *s):
            assert token == want, (i, s, float(u[i]), margin)
            checked += 1
    assert checked >= 0.8 * len(got)
    return got


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.7, 0.0), (0.9, 0, 1.0, 0.05),
           (0.8, 40, 0.9, 0.02), (0.0, 3, 0.5, 0.1), (1.0, 1, 1.0, 0.0), (2.0, 100000, 0.95, 0.0),
           (0.6, 0, 0.0, 0.0), (0.05, 7, 0.99, 0.0)]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 1000, 1025, 4099, 9001])
def test_filters(cuda_device, io, V):
    logits, u = _rows(2 * len(FILTERS), V, io, V)
    _check(logits, u, FILTERS * 2, cuda_device)


def _check_share(row, u, token, t, k, p, m):
    """The tokens of one row for many ``u``: each is kept, and ``u`` lies in its part of the kept
    share, but for rounding and for one token more or less at the filters' edge."""
    l = row.double()
    w = torch.exp((l - l.max()) / t)
    order = torch.sort(l, descending=True, stable=True).indices
    ws = w[order]
    if k:
        ws[k:] = 0
    if p < 1:
        ws[(ws.cumsum(0) - ws) >= torch.tensor(p).double() * ws.sum()] = 0
    ws[ws < torch.tensor(m).double() * ws[0]] = 0
    last = ws[ws > 0].min() / ws.sum()
    share = torch.zeros_like(w)
    share[order] = ws / ws.sum()
    run = share.cumsum(0)
    room = AWAY + (float(last) if p < 1 or m > 0 else 0.0)
    assert bool((w[token] / ws.sum() >= float(last) * (1 - 1e-4)).all())
    assert bool((run[token] > u - room).all())
    assert bool((run[token] - share[token] < u + room).all())


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("settings", [(1.0, 3000, 1.0, 0.0), (1.0, 0, 0.97, 0.0),
                                      (1.5, 2500, 0.9, 0.0), (1.0, 0, 0.9, 0.001)])
def test_cuts_that_keep_many_tokens(cuda_device, io, settings):
    """Flat rows: the cut keeps more tokens than are sorted in one place."""
    from hsn_amd import sampling

    logits, _ = _rows(1, 20011, io, 5, spread=0.7)
    u = (torch.arange(40) + 0.5) / 40
    t, k, p, m = settings
    got = sampling.sample(logits.expand(40, -1).to(cuda_device), u.to(cuda_device), temperature=t,
                          top_k=k, top_p=p, min_p=m)
    _check_share(logits[0], u, got.cpu(), *settings)


@pytest.mark.parametrize("V", [5, 700, 5003])
def test_equal_logits_go_to_the_lowest_tokens(cuda_device, V):
    """All equal, and two levels whose cut lies among equals: the cut keeps the lowest tokens."""
    from hsn_amd import sampling

    u = torch.tensor([0.0, 0.31, 0.5, 0.999], device=cuda_device)
    flat = torch.full((4, V), 2.5, device=cuda_device)
    for k in (1, 3, V // 2 + 1, V):
        got = sampling.sample(flat, u, top_k=k)
        assert got.tolist() == [int(float(v) * k) for v in u], k
    for p in (0.25, 0.5, 0.9):  # the shortest prefix with p V of V equal masses
        keep = math.ceil(torch.tensor(p).item() * V)
        assert sampling.sample(flat, u, top_p=p).tolist() == [int(float(v) * keep) for v in u]
    two = flat.clone()
    two[:, ::2] -= 1.0  # the odd tokens are larger
    odd = V // 2
    got = sampling.sample(two, u, top_k=odd + 2)
    want = [L.sample(two[0].cpu(), float(v), 1.0, odd + 2)[0] for v in u]
    assert got.tolist() == want


def test_masked_and_odd_values(cuda_device):
    from hsn_amd import sampling

    inf, nan = math.inf, math.nan
    logits = torch.zeros(9, 300)
    logits[0] = -inf
    logits[1] = nan
    logits[2, :] = -inf
    logits[2, 77] = -3e38
    logits[3, 5:] = -inf
    logits[3, 2] = nan
    logits[4, 30] = inf
    logits[4, 90] = inf
    logits[5] = torch.finfo(torch.float32).min
    logits[6, 0] = -0.0
    logits[7] = 3e38
    logits[7, ::3] = -3e38
    logits[8, 100] = 60.0
    u = torch.full((9,), 0.6, device=cuda_device)
    on = logits.to(cuda_device)
    for settings in (dict(), dict(top_k=400), dict(top_p=0.999), dict(top_k=200, top_p=0.9999),
                     dict(min_p=1e-3)):
        got = sampling.sample(on, u, **settings).tolist()
        assert got[0] == got[1] == -1
        assert got[2] == 77
        assert got[3] == 3  # 0, 1, 3, 4 with a quarter each
        assert got[4] == 90
        assert 0 <= got[5] < 300 and got[7] % 3 != 0
        assert got[8] == 100
    assert sampling.sample(on, u, temperature=0.0).tolist() == [-1, -1, 77, 0, 30, 0, 0, 1, 100]
    # the lowest value of a 16-bit type as a mask
    for io in (torch.bfloat16, torch.float16):
        masked = torch.full((1, 900), torch.finfo(io).min, dtype=io, device=cuda_device)
        masked[0, 500] = 1.0
        for settings in (dict(), dict(top_k=10), dict(top_p=0.9), dict(temperature=0.0)):
            assert sampling.sample(masked, u[:1], **settings).tolist() == [500]


def test_ends_of_the_random_number(cuda_device):
    from hsn_amd import sampling

    logits = torch.randn(1, 5000, device=cuda_device)
    logits[0, 0] = logits[0, 4999] = 0.0
    below_one = torch.tensor([1 - 2.0 ** -24], device=cuda_device)
    assert sampling.sample(logits, torch.zeros(1, device=cuda_device)).tolist() == [0]
    assert sampling.sample(logits, below_one).tolist() == [4999]


@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_rows_at_any_address(cuda_device, io):
    """Rows that start anywhere, further apart than their length."""
    from hsn_amd import sampling

    logits, u = _rows(8, 2050, io, 1)
    dense, u = logits.to(cuda_device), u.to(cuda_device)
    want = sampling.sample(dense, u, top_k=50, top_p=0.9)
    for pad, start in ((1, 0), (3, 1), (7, 5)):
        room = torch.zeros(8 * (2050 + pad) + start, dtype=IO[io], device=cuda_device)
        view = room[start:].view(8, 2050 + pad)[:, :2050]
        view.copy_(dense)
        assert torch.equal(sampling.sample(view, u, top_k=50, top_p=0.9), want)
        assert torch.equal(sampling.sample(view, u), sampling.sample(dense, u))


def test_rows_past_31_bits(cuda_device):
    from hsn_amd import sampling

    far = 2 ** 31 + 8
    room = torch.empty(far + 2000, dtype=torch.bfloat16, device=cuda_device)
    view = room.as_strided((2, 1500), (far, 1))
    logits, u = _rows(2, 1500, "bf16", 3)
    view.copy_(logits)
    u = u.to(cuda_device)
    assert torch.equal(sampling.sample(view, u), sampling.sample(logits.to(cuda_device), u))


@pytest.mark.parametrize("V", [32000, 131072, 262144])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_large_vocabularies_follow_the_share(cuda_device, V, io):
    """One row for each of many random numbers: the tokens are the quantiles of the kept share."""
    from hsn_amd import sampling

    logits, _ = _rows(1, V, io, V)
    u = (torch.arange(64) + 0.5) / 64
    rows = logits.expand(64, V).to(cuda_device)  # one row in memory
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 64, 1.0, 0.0), (0.8, 0, 0.8, 0.01)):
        got = sampling.sample(rows, u.to(cuda_device), temperature=t, top_k=k, top_p=p, min_p=m)
        _check_share(logits[0], u, got.cpu(), t, k, p, m)


@pytest.mark.parametrize("io,V", [("f32", 100003), ("bf16", 150001)])
def test_a_rows_token_does_not_depend_on_the_batch(cuda_device, io, V):
    """A row alone, in a batch of 30 and in one of 120: how the rows are spread over the GPU differs,
    the sums are of whole numbers and may not."""
    from hsn_amd import sampling

    n = 120
    logits, u = _rows(n, V, io, 17)
    logits[7] = -math.inf  # a row without a token, and one with a single token
    logits[8, 1:] = -math.inf
    t, k, p, m = (torch.tensor(c, dtype=d).to(cuda_device) for c, d in zip(
        zip(*[FILTERS[i % len(FILTERS)] for i in range(n)]),
        (torch.float32, torch.int32, torch.float32, torch.float32)))
    logits, u = logits.to(cuda_device), u.to(cuda_device)

    def run(size):
        return [x for i in range(0, n, size) for x in sampling.sample(
            logits[i:i + size], u[i:i + size], temperature=t[i:i + size], top_k=k[i:i + size],
            top_p=p[i:i + size], min_p=m[i:i + size]).tolist()]

    alone = run(1)
    assert run(30) == alone and run(n) == alone
    assert alone[7] == -1 and alone[8] == 0
    plain = [i for i in range(n) if i % len(FILTERS) == 3 and i > 8]  # a temperature and min_p
    for i in plain[:4]:
        _check_share(logits[i].float().cpu(), u[i:i + 1].cpu(), torch.tensor(alone[i:i + 1]), *FILTERS[3])


def test_settings_as_numbers_and_as_rows(cuda_device):
    from hsn_amd import sampling

    logits, u = (t.to(cuda_device) for t in _rows(6, 3000, "f32", 9))
    one = dict(temperature=0.9, top_k=30, top_p=0.8, min_p=0.01)
    rows = {k: torch.full((6,), v, device=cuda_device,
                          dtype=torch.int32 if k == "top_k" else torch.float32)
            for k, v in one.items()}
    want = sampling.sample(logits, u, **one)
    assert torch.equal(sampling.sample(logits, u, **rows), want)
    assert torch.equal(sampling.sample(logits, u, **{**one, "top_k": rows["top_k"]}), want)
    assert torch.equal(torch.cat([sampling.sample(logits[i:i + 1], u[i:i + 1], **one)
                                  for i in range(6)]), want)
    assert sampling.sample(logits[:0], u[:0]).shape == (0,)


def test_in_a_graph(cuda_device):
    from hsn_amd import sampling

    logits, u = (t.to(cuda_device) for t in _rows(4, 40000, "bf16", 2))
    sampling.sample(logits, u, top_k=50)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = sampling.sample(logits, u, top_k=50)
        free = sampling.sample(logits, u)
    for k in range(3):
        u.copy_(torch.rand(4, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, sampling.sample(logits, u, top_k=50))
        assert torch.equal(free, sampling.sample(logits, u))


def test_refusals(cuda_device):
    from hsn_amd import sampling

    logits, u = torch.zeros(3, 10, device=cuda_device), torch.zeros(3, device=cuda_device)
    bad = [
        lambda: sampling.sample(logits.cpu(), u.cpu()),
        lambda: sampling.sample(logits.double(), u),
        lambda: sampling.sample(logits[0], u),
        lambda: sampling.sample(logits.t(), torch.zeros(10, device=cuda_device)),
        lambda: sampling.sample(logits, u[:2]),
        lambda: sampling.sample(logits, u.double()),
        lambda: sampling.sample(logits, u.cpu()),
        lambda: sampling.sample(logits, u, top_k=-1),
        lambda: sampling.sample(logits, u, top_k=torch.zeros(3, device=cuda_device)),
        lambda: sampling.sample(logits, u, temperature=torch.zeros(2, device=cuda_device)),
        lambda: sampling.sample(logits, u, top_p=torch.zeros(3)),
        lambda: sampling.sample(logits[:, :0], u),
        lambda: sampling.sample(torch.zeros(1, 1, device=cuda_device).expand(1, 2 ** 18 + 1), u[:1]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("V", [32000, 131072, 262144])
def test_large_vocabularies_in_fp16(cuda_device, V):
    from hsn_amd import sampling

    logits, _ = _rows(1, V, "f16", V + 1)
    u = (torch.arange(64) + 0.5) / 64
    for n in (64, 3):  # whole rows or few slices, and many slices
        rows = logits.expand(n, V).to(cuda_device)
        for settings in ((1.0, 0, 1.0, 0.0), (1.0, 64, 1.0, 0.0), (0.8, 0, 0.8, 0.01), (1.0, 0, 1.0, 0.001)):
            t, k, p, m = settings
            got = sampling.sample(rows, u[:n].to(cuda_device), temperature=t, top_k=k, top_p=p, min_p=m)
            _check_share(logits[0], u[:n], got.cpu(), *settings)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [9500, 140000])
@pytest.mark.parametrize("k,level", [(5700, 1.0), (5700, 2.0), (2000, 2.0), (0, 1.0), (5700, None), (0, None)])
def test_cuts_among_thousands_of_equal_logits(cuda_device, io, V, k, level):
    """200 tokens of 3, 3000 of 2 and 6000 of 1, anywhere in the row: top_k (above what a list holds) and
    top_p each cut among more equal tokens than are sorted in one place. top_p lies half a token's
    mass from its edges and u in the middle of a token's share, so fp32 decides nothing."""
    from hsn_amd import sampling

    g = torch.Generator().manual_seed(k + V)
    row = torch.full((V,), -math.inf)
    row[torch.randperm(V, generator=g)[:9200]] = torch.tensor([3.0] * 200 + [2.0] * 3000 + [1.0] * 6000)
    row = row.to(IO[io])
    p = 1.0
    if level is not None:
        all_kept = L.kept_tokens(row.float(), 1.0, k, 1.0, 0.0)
        total = sum(w for _, w in all_kept)
        inside = [i for i, (j, _) in enumerate(all_kept) if float(row[j]) == level]
        cut = inside[len(inside) * 2 // 3]
        p = (sum(w for _, w in all_kept[:cut]) + 0.5 * all_kept[cut][1]) / total
    p = float(torch.tensor(p, dtype=torch.float32))
    kept = sorted(L.kept_tokens(row.float(), 1.0, k, p, 0.0))
    total, run, at = sum(w for _, w in kept), 0.0, []
    for j, w in kept:
        at.append((j, (run + 0.5 * w) / total))
        run += w
    picks = [at[i] for i in (0, 1, len(at) // 3, len(at) // 2, len(at) - 2, len(at) - 1)]
    u = torch.tensor([v for _, v in picks], dtype=torch.float32)
    rows = row.expand(len(picks), V).to(cuda_device)
    got = sampling.sample(rows, u.to(cuda_device), top_k=k, top_p=p)
    assert got.tolist() == [j for j, _ in picks]
