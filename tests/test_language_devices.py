"""The language-model operators on tensors whose device is not the current one: they launch there, on
that device's current stream, and leave the current device as it was."""

from __future__ import annotations

import subprocess

import pytest
import torch

from hsn_amd import build


def test_the_host_helper_makes_the_tensors_device_current():
    """One device cannot show it: the module takes its device guard from PyTorch's registry of them."""
    if build.host_stale("_calls") is not None:
        pytest.skip("host helper not built here")
    symbols = subprocess.run(["nm", "-D", "--undefined-only", str(build.PKG / "_calls.so")],
                             check=True, capture_output=True, text=True).stdout
    assert "device_guard_impl_registry" in symbols


def _everything(device):
    from hsn_amd import sampling, scan
    from hsn_amd.unit_layer import unit_layer

    g = torch.Generator().manual_seed(3)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(device)

    y, gate, state = rnd(2, 700, 8), rnd(2, 700, 8), rnd(4, 8)
    out = scan.forward(y, gate)
    grads = scan.backward(y, gate, out["marks"], None, y)
    h = scan.step(y[:, 0], gate[:, 0], state)
    o = unit_layer(rnd(3, 8), rnd(4, 8), rnd(4, 8, 8), None, rnd(4, 8, 8), None, 2)
    token = sampling.sample(rnd(3, 70000), torch.rand(3, generator=g).to(device), top_p=0.9)
    return [out["h"], out["h_T"], *grads, h, state, o, token]


@pytest.mark.gpu
def test_the_python_calls_make_the_tensors_device_current(cuda_device, monkeypatch):
    """The calls without the host helper, with a record of what is current at each launch."""
    from hsn_amd import _lib, sampling, scan, unit_layer

    for module in (scan, unit_layer, sampling):
        monkeypatch.setattr(module, "native_calls", lambda *names: None)
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

    monkeypatch.setattr(torch.cuda, "device", Device)
    for module in (_lib, scan, unit_layer, sampling):
        monkeypatch.setattr(module, "call", recorded)
    _everything(cuda_device)
    assert launched == [(name, [0]) for name in ("hsn_scan_forward", "hsn_scan_backward", "hsn_scan_step",
                                                 "hsn_units_layer", "hsn_sample")]


@pytest.mark.gpu
@pytest.mark.parametrize("helper", [True, False])
def test_on_a_second_device(cuda_device, monkeypatch, helper):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    from hsn_amd import sampling, scan, unit_layer

    if not helper:
        for module in (scan, unit_layer, sampling):
            monkeypatch.setattr(module, "native_calls", lambda *names: None)
    want = _everything(cuda_device)
    got = _everything(torch.device("cuda", 1))
    assert torch.cuda.current_device() == 0
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, got))
