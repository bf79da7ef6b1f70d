"""The training step's operators' host side on the CPU: what the entry points refuse before any launch,
their workspace sizes, the Python mirrors' checks and the native calls' refusals. No kernel runs here."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from hsn_amd import build


@pytest.fixture(scope="module")
def lib():
    if build.stale() is not None:
        pytest.skip("library not built here")
    from hsn_amd import _lib

    return _lib.library()


@pytest.fixture()
def message(lib):
    return lambda: lib.hsn_win_last_error().decode()


def _embed(lib, **change):
    a = dict(tokens=64, tb=8, tt=1, bytes=8, table=64, row=16, code=0, scale=1.0, out=64, out_code=0,
             B=1, T=8, V=10, D=16, stream=None)
    a.update(change)
    return lib.hsn_embed_forward(*a.values())


def _embed_back(lib, **change):
    a = dict(tokens=64, tb=8, tt=1, bytes=8, d_out=64, db=128, dt=16, code=0, scale=1.0, d_table=64,
             table_code=0, B=1, T=8, V=10, D=16, ws=64, n=1 << 40, stream=None)
    a.update(change)
    return lib.hsn_embed_backward(*a.values())


def test_embedding_refusals(lib, message):
    for call in (_embed, _embed_back):
        assert call(lib, code=3) == 2 and call(lib, code=-1) == 2
        assert call(lib, V=0) == 1 and call(lib, D=0) == 1 and call(lib, B=-1) == 1
        assert call(lib, V=(1 << 24) + 1) == 5 and call(lib, D=65537) == 5
        assert call(lib, B=1 << 13, T=1 << 13) == 5 and "tokens" in message()
        assert call(lib, tokens=None) == 1 and call(lib, bytes=2) == 1
    assert _embed(lib, out_code=5) == 2 and _embed_back(lib, table_code=5) == 2
    assert _embed(lib, table=None) == 1 and _embed(lib, table=66) == 1 and "aligned" in message()
    assert _embed(lib, out=65, out_code=2) == 1
    assert _embed(lib, B=0) == 0 and _embed(lib, T=0) == 0
    assert _embed_back(lib, d_out=None) == 1 and _embed_back(lib, d_table=None) == 1
    assert _embed_back(lib, d_out=65, code=1) == 1
    assert _embed_back(lib, ws=None) == 1 and _embed_back(lib, ws=72) == 1 and "16" in message()
    assert _embed_back(lib, n=48) == 1 and "small" in message()


def test_embedding_workspace(lib):
    size = ctypes.c_int64(-1)

    def bytes_of(n, V=1000, D=64, code=0):
        assert lib.hsn_embed_workspace(1, n, V, D, code, ctypes.byref(size)) == 0
        return size.value

    assert bytes_of(0) == 16 and bytes_of(1) == 16
    assert bytes_of(8192) == 8 * 8192  # the entries alone
    assert bytes_of(8192, D=4096) == 8 * 8192 + 8192 // 64 * 2 * 4096 * 4  # two sums of each chunk of 64
    # two lists of entries, the tiles' counts, two sums of each chunk of eight
    assert bytes_of(65536) == 2 * 8 * 65536 + 64 * 4096 + 65536 // 8 * 2 * 64 * 4
    assert lib.hsn_embed_workspace(1, 8, 8, 8, 0, None) == 1


def _score(lib, **change):
    a = dict(logits=64, row=100, code=0, tokens=64, stride=1, bytes=8, logprob=64, entropy=64, top_tokens=64,
             top_logprobs=64, stats=64, n=2, V=100, top=3, ws=None, size=0, stream=None)
    a.update(change)
    return lib.hsn_score_forward(*a.values())


def _score_back(lib, **change):
    a = dict(logits=64, row=100, code=0, tokens=64, stride=1, bytes=8, stats=64, g=64, gs=1, h=64, hs=1, d=64,
             n=2, V=100, stream=None)
    a.update(change)
    return lib.hsn_score_backward(*a.values())


def test_scoring_refusals(lib, message):
    for call in (_score, _score_back):
        assert call(lib, code=3) == 2
        assert call(lib, V=0) == 1 and call(lib, n=-1) == 1
        assert call(lib, V=(1 << 24) + 1) == 5 and call(lib, n=1 << 24) == 5
        assert call(lib, n=1 << 23, V=1 << 17) == 5 and "logits" in message()
        assert call(lib, logits=None) == 1 and call(lib, tokens=None) == 1 and call(lib, bytes=1) == 1
        assert call(lib, logits=65, code=2) == 1 and "aligned" in message()
        assert call(lib, stats=72) == 1
        assert call(lib, n=0) == 0
    assert _score(lib, top=-1) == 1 and _score(lib, top=33) == 1
    assert _score(lib, logprob=None) == 1 and _score(lib, top_tokens=None) == 1
    assert _score(lib, V=262144, row=262144) == 1 and "workspace" in message()
    assert _score(lib, V=262144, row=262144, ws=72, size=1 << 40) == 1 and "aligned" in message()
    assert _score_back(lib, stats=None) == 1 and _score_back(lib, d=None) == 1
    assert _score_back(lib, d=65, code=1) == 1


def test_scoring_workspace(lib):
    size = ctypes.c_int64(-1)
    for n, V, code in ((1, 500, 0), (1, 32000, 2), (300, 32000, 2), (1000, 131071, 2), (8192, 32000, 0)):
        assert lib.hsn_score_workspace(n, V, code, 20, ctypes.byref(size)) == 0 and size.value == 0
    # 32 parts of four waves' batch each: three sums, and twenty candidates
    assert lib.hsn_score_workspace(1, 262144, 2, 20, ctypes.byref(size)) == 0
    assert size.value == 32 * (16 + 20 * 8)
    assert lib.hsn_score_workspace(1, 8, 0, 0, None) == 1


def _route(lib, **change):
    a = dict(logits=64, row=8, code=0, valid=None, units=64, shares=64, tally=64, probs=64, balance=64, n=4, M=8,
             k=2, ws=64, size=1 << 40, stream=None)
    a.update(change)
    return lib.hsn_unit_router_forward(*a.values())


def _route_back(lib, **change):
    a = dict(logits=64, row=8, code=0, valid=None, units=64, tally=64, g=64, g_row=2, b=64, d=64, n=4, M=8, k=2,
             stream=None)
    a.update(change)
    return lib.hsn_unit_router_backward(*a.values())


def test_unit_router_refusals(lib, message):
    for call in (_route, _route_back):
        assert call(lib, code=3) == 2
        assert call(lib, M=0) == 1 and call(lib, n=-1) == 1
        assert call(lib, M=257) == 5 and call(lib, n=1 << 30) == 5
        assert call(lib, k=0) == 1 and call(lib, k=9) == 1 and call(lib, M=64, k=17) == 1
        assert call(lib, logits=None) == 1 and call(lib, units=None) == 1 and call(lib, tally=None) == 1
        assert call(lib, logits=65, code=2) == 1 and "aligned" in message()
    assert _route(lib, ws=None) == 1 and _route(lib, ws=72) == 1 and _route(lib, size=8) == 1
    assert _route(lib, balance=None) == 1 and _route(lib, probs=None) == 1
    assert _route_back(lib, n=0) == 0 and _route_back(lib, d=None) == 1
    size = ctypes.c_int64(-1)
    assert lib.hsn_unit_router_workspace(4, 8, 0, ctypes.byref(size)) == 0
    assert size.value == 64 + 32 + 16  # one workgroup's eight sums and counts, its live tokens
    assert lib.hsn_unit_router_workspace(4, 8, 0, None) == 1


def _clip(lib, grads=(256,), outs="in place", numels=(8,), codes=(0,), max_norm=1.0, result=64, ws=64,
          size=1 << 40):
    n = len(grads)
    pointers = ctypes.c_void_p * n
    given = None if outs is None else pointers(*(grads if outs == "in place" else outs))
    return lib.hsn_clip(pointers(*grads), given, (ctypes.c_int64 * n)(*numels), (ctypes.c_int * n)(*codes), n,
                        max_norm, result, ws, size, None)


def test_clip_refusals(lib, message):
    assert _clip(lib, codes=(3,)) == 2
    assert _clip(lib, numels=(-1,)) == 1 and "negative" in message()
    assert _clip(lib, max_norm=-1.0) == 1 and _clip(lib, max_norm=math.nan) == 1
    assert _clip(lib, result=None) == 1 and _clip(lib, ws=None) == 1 and _clip(lib, ws=68) == 1
    assert _clip(lib, size=8) == 1 and "small" in message()
    assert _clip(lib, grads=(None,)) == 1 and _clip(lib, grads=(258,)) == 1 and "aligned" in message()
    assert _clip(lib, grads=(1 << 50,)) == 1
    assert _clip(lib, grads=(4096,) * 2, numels=(1 << 44, 8), codes=(0, 0), outs=None) == 5
    # what is written overlaps: itself, a neighbour, another one's gradient
    assert _clip(lib, grads=(256, 256), numels=(8, 8), codes=(0, 0)) == 1 and "overlap" in message()
    assert _clip(lib, grads=(256, 284), numels=(8, 8), codes=(0, 0)) == 1
    assert _clip(lib, grads=(284, 256), numels=(8, 8), codes=(0, 0)) == 1
    assert _clip(lib, grads=(256, 512), outs=(512, 1024), numels=(8, 8), codes=(0, 0)) == 1
    assert "gradient 1" in message()
    assert _clip(lib, grads=(256,), outs=(260,)) == 1 and "gradient 0" in message()
    assert _clip(lib, grads=(256,), outs=(252,)) == 1
    assert _clip(lib, grads=(256, 320), outs=(256, 310), numels=(8, 8), codes=(2, 2)) == 1
    size = ctypes.c_int64(-1)
    assert lib.hsn_clip_workspace((ctypes.c_int64 * 1)(8), 1, ctypes.byref(size)) == 0
    assert size.value == 8 * 2048
    assert lib.hsn_clip_workspace(None, 1, ctypes.byref(size)) == 1
    assert lib.hsn_clip_workspace(None, 0, None) == 1


def test_the_python_mirrors_take_no_host_tensors(lib):
    from hsn_amd import embedding, grad_clip, scoring, unit_router

    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: embedding.forward(t, x), lambda: embedding.backward(t, x, 5),
                 lambda: embedding.embed(t, x.requires_grad_()), lambda: scoring.forward(x, t),
                 lambda: scoring.backward(x, t, torch.zeros(3, 4), None),
                 lambda: scoring.token_logprobs(x, t), lambda: unit_router.forward(x, 2),
                 lambda: unit_router.backward(x, t[:, None], t, None), lambda: unit_router.choose_units(x, 2),
                 lambda: grad_clip.norm([x.detach()]), lambda: grad_clip.clip([x.detach()], 1.0)):
        with pytest.raises(ValueError, match="ROCm device tensors"):
            call()


def test_the_native_calls_decline_host_tensors_and_other_things(lib):
    if build.host_stale("_calls") is not None:
        pytest.skip("host helper not built here")
    from hsn_amd import _lib

    calls, at = _lib.native_calls("hsn_score_forward")
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    assert calls.embed_forward(at, 0, t, x, 1.0, 0) is None
    assert calls.embed_backward(at, at, 0, t, x, 5, 1.0, 0) is None
    assert calls.score_forward(at, at, 0, x, t, 0, 1) is None
    assert calls.score_backward(at, 0, x, t, x, None, None) is None
    assert calls.unit_router_forward(at, at, 0, x, 2, None) is None
    assert calls.unit_router_backward(at, 0, x, x, x, None, None, None) is None
    assert calls.grad_clip(at, at, 0, [x], [x], 1.0) is None
    for bad in ((), (at, at, 0, None, None, 1.0), (at, at, 0, [], [], 1.0), (at, at, 0, [None], [x], 1.0),
                (at, at, 0, x, x, 1.0), (at, at, 0, [x], [], 1.0)):
        assert calls.grad_clip(*bad) is None
    for name in ("embed_forward", "embed_backward", "score_forward", "score_backward", "unit_router_forward",
                 "unit_router_backward"):
        assert getattr(calls, name)() is None and getattr(calls, name)(at, at, 0, "x", "y") is None


def test_no_call_writes_a_gradient_for_a_double_backward(lib):
    """The autograd nodes keep nothing that a second derivative could go through."""
    from hsn_amd import embedding, scoring, unit_router

    for node in (embedding.Embed, scoring.TokenLogprobs, unit_router.ChooseUnits):
        assert "once_differentiable" in repr(node.backward) or node.backward.__wrapped__ is not None
