"""The training step's operators where offsets pass 2^31 elements and 2^32 bytes: what is far behind is computed
as what is in front."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free(cuda_device):
    if torch.cuda.get_device_properties(cuda_device).total_memory < 100 << 30:
        pytest.skip("needs 100 GiB of device memory")
    yield
    torch.cuda.empty_cache()


def test_logits_past_32_bits(cuda_device):
    """36000 rows of 131073 in bf16, 9.4 GB: the last rows repeat the first ones."""
    from hsn_amd import scoring

    n, V = 36000, 131073
    logits = torch.zeros(n, V, dtype=torch.bfloat16, device=cuda_device)
    few = torch.randn(8, V, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(cuda_device)
    logits[:8], logits[-8:] = few, few  # (the distance of rows is odd and n - 8 is even: the same addresses mod 16)
    tokens = torch.zeros(n, dtype=torch.int64, device=cuda_device)
    tokens[-8:] = tokens[:8] = torch.arange(8, device=cuda_device) * 16001
    out = scoring.forward(logits, tokens, top=2)
    for name in out:
        assert torch.equal(out[name][:8], out[name][-8:]), name
    assert abs(float(out["logprob"][n // 2]) + math.log(V)) <= 1e-5
    d = scoring.backward(logits, tokens, out["stats"], torch.ones(n, device=cuda_device))
    assert torch.equal(d[:8], d[-8:]) and bool(d[-1].any())
    # the row between: 1 - 1 / V at the token, -1 / V elsewhere
    assert float(d[n // 2, 0]) == 1.0
    assert bool((d[n // 2, 1:] == torch.tensor(-1 / V).to(torch.bfloat16).to(cuda_device)).all())


def test_tables_past_32_bits(cuda_device):
    """2^21 rows of 4096 in bf16, 17 GB: the first and the last rows, 30000 tokens of them."""
    from hsn_amd import embedding

    V, D, n = 1 << 21, 4096, 30000
    table = torch.empty(V, D, dtype=torch.bfloat16, device=cuda_device)
    table[:4] = torch.randn(4, D, device=cuda_device)
    table[-4:] = table[:4]
    low = torch.randint(0, 4, (n,), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    got = embedding.forward(low + V - 4, table)
    assert torch.equal(got, embedding.forward(low, table)) and torch.equal(got, table[low])
    d = torch.randn(n, D, dtype=torch.bfloat16, device=cuda_device)
    back = embedding.backward(low + V - 4, d, V)
    assert torch.equal(back[-4:], embedding.backward(low, d, 4))
    assert not back[:-4].any()


def test_rows_past_32_bits(cuda_device):
    """1.2 M positions of 2048 in bf16, 4.9 GB, both ways."""
    from hsn_amd import embedding

    n, D = 1200007, 2048
    table = torch.randn(7, D, device=cuda_device).to(torch.bfloat16)
    tokens = torch.arange(n, device=cuda_device) % 7
    out = embedding.forward(tokens, table)
    assert torch.equal(out[-7:], table[tokens[-7:]]) and torch.equal(out[n // 2], table[tokens[n // 2]])
    del out
    d = torch.zeros(n, D, dtype=torch.bfloat16, device=cuda_device)
    d[0], d[n // 2], d[-1] = 1.0, 2.0, 4.0
    want = torch.zeros(7, D, device=cuda_device)
    for i, v in ((0, 1.0), (n // 2, 2.0), (n - 1, 4.0)):
        want[int(tokens[i])] += v
    assert torch.equal(embedding.backward(tokens, d, 7, dtype=torch.float32), want)


def test_slots_past_32_bits(cuda_device):
    """2^28 + 5 tokens of 8 units, 8 chosen: 2^31 slots, 17 GB of them."""
    from hsn_amd import unit_router

    n, M = (1 << 28) + 5, 8
    logits = torch.zeros(n, M, dtype=torch.bfloat16, device=cuda_device)
    logits[-3:] = logits[:3] = torch.randn(3, M, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    out = unit_router.forward(logits, 8)
    assert torch.equal(out["units"][:3], out["units"][-3:]) and torch.equal(out["shares"][:3], out["shares"][-3:])
    assert torch.equal(out["units"][n // 2], torch.arange(8, device=cuda_device))
    assert out["counts"].tolist() == [n] * M and int(out["tally"][M]) == n
    torch.testing.assert_close(out["probs"], torch.full((M,), 0.125, device=cuda_device), rtol=1e-6, atol=0)
    g = torch.zeros(1, 8, device=cuda_device).expand(n, 8)
    d = unit_router.backward(logits, out["units"], out["tally"], g, torch.full((), 1e8, device=cuda_device))
    assert torch.equal(d[:3], d[-3:])


def test_a_gradient_past_32_bits(cuda_device):
    """One tensor of 2^32 + 9 elements in bf16, 8.6 GB."""
    from hsn_amd import grad_clip

    n = (1 << 32) + 9
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda_device)
    g[0], g[n // 2], g[-1] = 3.0, 12.0, 4.0
    norm, coefficient = grad_clip.clip([g], 6.5)
    assert abs(float(norm) - 13.0) <= 1e-14 * 13
    assert abs(float(coefficient) - 0.5) <= 1e-7
    assert [float(v) for v in (g[0], g[n // 2], g[-1])] == [1.5, 6.0, 2.0] and not g[1:1000].any()
