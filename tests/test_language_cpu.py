"""The language-model operators' host side on the CPU: what the entry points refuse before any
launch, their workspace sizes, and the Python mirror's checks. No kernel runs here."""

from __future__ import annotations

import ctypes

import pytest
import torch

from hsn_amd import build


@pytest.fixture(scope="module")
def lib():
    if build.stale() is not None:
        pytest.skip("library not built here")
    from hsn_amd import _lib

    return _lib.library()


def _scan_forward(lib, **change):
    a = dict(y=64, ys=64, yp=64, g=64, gs=64, gp=64, dtype=0, candidate=0, reset=None, h0=None, h=64,
             h_T=64, marks=None, B=1, T=8, D=64, ws=None, n=0)
    a.update(change)
    return lib.hsn_scan_forward(*a.values(), None)


def test_scan_refusals(lib):
    def message():
        return lib.hsn_win_last_error().decode()

    assert _scan_forward(lib, dtype=3) == 2
    assert _scan_forward(lib, candidate=2) == 1 and "candidate" in message()
    assert _scan_forward(lib, D=0) == 1
    assert _scan_forward(lib, B=-1) == 1
    assert _scan_forward(lib, y=None) == 1 and "NULL" in message()
    assert _scan_forward(lib, h_T=None) == 1
    assert _scan_forward(lib, T=4000) == 1 and "workspace" in message()
    assert _scan_forward(lib, T=4000, ws=8, n=1 << 30) == 1 and "aligned" in message()
    assert _scan_forward(lib, B=0) == 0
    assert _scan_forward(lib, T=(1 << 30) + 1) == 5 and _scan_forward(lib, D=(1 << 30) + 1) == 5
    assert lib.hsn_scan_backward(64, 64, 64, 64, 64, 64, 0, 0, None, None, 64, 64, 64, None, 64, 64, 64,
                                 1, 8, 64, None, 0, None) == 1  # no marks
    assert lib.hsn_scan_step(64, 64, 64, 64, 0, 0, None, None, 64, 64, 5, 4, 64, None) == 1
    assert lib.hsn_scan_step(64, 64, 64, 64, 0, 0, 64, None, None, 64, 5, 4, 64, None) == 1
    assert lib.hsn_scan_step(64, 64, 64, 64, 0, 0, None, None, 64, 64, 0, 4, 64, None) == 0


def test_scan_workspace(lib):
    size = ctypes.c_int64(-1)
    for backward in (0, 1):
        assert lib.hsn_scan_workspace(4, 128, 512, 0, backward, ctypes.byref(size)) == 0
        assert size.value == 0  # one tile
        assert lib.hsn_scan_workspace(1, 32768, 1024, 2, backward, ctypes.byref(size)) == 0
        tiles = 32768 // (128 if backward else 256)
        assert size.value == 8 * (64 + (tiles + tiles // 32) * 16 * 64)
    assert lib.hsn_scan_workspace(1, 8, 8, 0, 0, None) == 1
    # more tiles than one grid holds
    assert lib.hsn_scan_workspace(1 << 20, 1 << 20, 64, 0, 0, ctypes.byref(size)) == 5


def test_sizes_past_one_grid(lib):
    """A dimension of a grid holds fewer than 2^32 threads: what needs more is refused by name."""
    size = ctypes.c_int64(-1)

    def message():
        return lib.hsn_win_last_error().decode()

    # 1024 tiles of 256 positions, 512 threads each
    assert lib.hsn_scan_workspace((1 << 13) - 1, 1 << 18, 64, 2, 0, ctypes.byref(size)) == 0
    assert lib.hsn_scan_workspace(1 << 13, 1 << 18, 64, 2, 0, ctypes.byref(size)) == 5
    assert _scan_forward(lib, B=1 << 23) == 5 and "one grid" in message()
    assert _scan_forward(lib, B=1 << 30, T=0) == 5 and "one grid" in message()
    assert lib.hsn_scan_step(64, 64, 64, 64, 0, 0, None, None, 64, 64, 1 << 24, 1 << 24, 1, None) == 5
    assert "one grid" in message()
    assert _sample(lib, n=1 << 22) == 5 and "rows" in message()
    assert lib.hsn_sample_workspace(1 << 22, 8, 0, ctypes.byref(size)) == 5


def _units(lib, **change):
    a = dict(x=64, x_row=16, router=64, W1=64, b1=None, W2=64, b2=None, y=64, n=2, M=4, K=2, d_in=16,
             H=8, d_out=16, dtype=0, activation=0, ws=256, bytes=1 << 20)
    a.update(change)
    return lib.hsn_units_layer(*a.values(), None)


def test_unit_layer_refusals(lib):
    def message():
        return lib.hsn_win_last_error().decode()

    assert _units(lib, dtype=7) == 2
    assert _units(lib, activation=2) == 1
    assert _units(lib, K=5) == 1 and "K <= M" in message()
    assert _units(lib, K=0) == 1
    assert _units(lib, n=65) == 5 and "64 tokens" in message()
    assert _units(lib, M=257) == 5
    assert _units(lib, M=32, K=17) == 5
    assert _units(lib, H=0) == 1
    assert _units(lib, W2=None) == 1 and "NULL" in message()
    assert _units(lib, ws=None) == 1
    assert _units(lib, ws=264) == 1 and "aligned" in message()
    assert _units(lib, bytes=64) == 1 and "small" in message()
    assert _units(lib, n=0) == 0


def _sample(lib, **change):
    settings = (ctypes.c_int32 * 4)(0, 0, 0, 0)
    a = dict(logits=64, row=100, dtype=0, u=64, t=64, k=64, p=64, m=64, settings=ctypes.byref(settings),
             tokens=64, n=2, V=100, ws=None, bytes=0)
    a.update(change)
    return lib.hsn_sample(*a.values(), None)


def test_sample_refusals(lib):
    def message():
        return lib.hsn_win_last_error().decode()

    assert _sample(lib, dtype=4) == 2
    assert _sample(lib, V=0) == 1
    assert _sample(lib, V=(1 << 18) + 1) == 5
    assert _sample(lib, u=None) == 1
    assert _sample(lib, settings=None, p=None) == 1 and "settings" in message()
    assert _sample(lib, n=1, V=1 << 18) == 1 and "workspace" in message()
    assert _sample(lib, n=0) == 0
    size = ctypes.c_int64(-1)
    assert lib.hsn_sample_workspace(300, 32000, 2, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.hsn_sample_workspace(1, 262144, 0, ctypes.byref(size)) == 0 and size.value > 0
    assert lib.hsn_sample_workspace(1, 8, 0, None) == 1


def test_python_refuses_host_tensors():
    from hsn_amd import sampling, scan
    from hsn_amd.unit_layer import unit_layer

    y = torch.zeros(2, 3, 4)
    for call in (lambda: scan.forward(y, y), lambda: scan.gated_scan(y, y),
                 lambda: scan.backward(y, y, y, None, y),
                 lambda: scan.step(y[0], y[0], torch.zeros(3, 4)),
                 lambda: unit_layer(y[0], y[0], y, None, y, None, 1),
                 lambda: sampling.sample(y[0], torch.zeros(3))):
        with pytest.raises(ValueError, match="device"):
            call()
