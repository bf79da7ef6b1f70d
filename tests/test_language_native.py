"""The host helper that makes the language-model operators' calls in one step (``hsn_amd/_calls.so``):
it is built from the current source, declines what the Python checks refuse, and gives the same
outputs as the calls without it."""

from __future__ import annotations

import pytest
import torch

from hsn_amd import build


def test_it_is_current_and_declines_host_tensors():
    assert build.host_stale("_calls") is None
    if build.stale() is not None:
        pytest.skip("library not built here")
    from hsn_amd import _lib

    calls, size_at, call_at = _lib.native_calls("hsn_scan_workspace", "hsn_scan_forward")
    y = torch.zeros(2, 3, 4)
    assert calls.scan_forward(size_at, call_at, 0, y, y, None, None, 0, 1, 128) is None
    assert calls.scan_backward(size_at, call_at, 0, y, y, y, None, y, None, 0, 128) is None
    assert calls.scan_step(call_at, 0, y[0], y[0], y[0], None, None, 0) is None
    assert calls.unit_layer(size_at, call_at, 0, y[0], y[0], y, None, y, None, 1, 0, 0) is None
    assert calls.sample(size_at, call_at, 0, y[0], y[0, 0], 1.0, 0, 1.0, 0.0) is None
    # too few arguments, and things that are no tensors
    assert calls.scan_step(call_at, 0, y[0]) is None
    assert calls.scan_step(call_at, 0, "y", y[0], y[0], None, None, 0) is None
    assert calls.sample() is None


@pytest.mark.gpu
def test_the_calls_without_it_give_the_same(cuda_device, monkeypatch):
    from hsn_amd import sampling, scan, unit_layer

    g = torch.Generator().manual_seed(0)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(cuda_device)

    y, gate, d_h, h0, d_h_T = rnd(2, 900, 24), rnd(2, 900, 24), rnd(2, 900, 24), rnd(2, 24), rnd(2, 24)
    reset = torch.rand(2, 900, generator=g).to(cuda_device) < 0.01
    state, rows = rnd(6, 24), torch.tensor([4, -1], dtype=torch.int32, device=cuda_device)
    x, router, W1, b1, W2, b2 = (rnd(3, 16), rnd(5, 16), rnd(5, 16, 16), rnd(5, 16), rnd(5, 8, 12),
                                 rnd(5, 12))
    logits, u = rnd(3, 70000), torch.rand(3, generator=g).to(cuda_device)
    k = torch.tensor([5, 0, 40], dtype=torch.int32, device=cuda_device)

    def everything():
        out = scan.forward(y, gate, reset, h0)
        bare = scan.forward(y, gate, candidate="linear", save=False)
        back = scan.backward(y, gate, out["marks"], reset, d_h, d_h_T)
        pool = state.clone()
        step = scan.step(y[:, 0], gate[:, 0], pool, rows=rows, reset=reset[:, 0].contiguous())
        layer = unit_layer.unit_layer(x, router, W1, b1, W2, b2, 2, activation="swiglu")
        tokens = sampling.sample(logits, u, temperature=0.8, top_k=k, top_p=0.9)
        return [out["h"], out["h_T"], out["marks"], bare["h"], *back, pool, step, layer, tokens]

    with_it = everything()
    assert bare_is_none(scan, y, gate)
    for module in (scan, unit_layer, sampling):
        monkeypatch.setattr(module, "native_calls", lambda *names: None)
    for a, b in zip(with_it, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype
    assert bare_is_none(scan, y, gate)


def bare_is_none(scan, y, gate) -> bool:
    return scan.forward(y, gate, save=False)["marks"] is None


@pytest.mark.gpu
def test_a_status_raises(cuda_device):
    """A refusal that only the entry point knows comes back with its message."""
    from hsn_amd import scan

    y = torch.zeros(5, 8, device=cuda_device)
    with pytest.raises(RuntimeError, match="every sequence"):
        scan.step(y, y, torch.zeros(3, 8, device=cuda_device))


def test_a_rows_sums_are_out_before_they_are_counted(tmp_path):
    """The workgroups that share a row's sums count themselves by an atomic, and the last one reads
    them all. The wave that counts waits for its own stores alone, so any other wave's have to be
    complete at the barrier before. In the code as built (the sampling's own, from this source), no
    store lies between the last wait for all of a wave's memory operations and that barrier, nor
    between the last such wait and the atomic."""
    import shutil
    import subprocess

    if build.stale() is not None:
        pytest.skip("library not built here")
    objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    if shutil.which(objdump) is None:
        pytest.skip("no llvm-objdump")
    shutil.copy(build.LIBRARY, tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found = 0
    for part in sorted(tmp_path.glob("lib.so.*gfx950*")):
        if b"sample_parts" not in part.read_bytes():
            continue
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", str(part)], check=True,
                              capture_output=True, text=True).stdout
        for kernel in text.split("\n\n"):
            if "sample_parts" not in kernel.strip().split("\n")[0]:
                continue
            lines = [line.split("//")[0].strip() for line in kernel.split("\n")]
            count = next(i for i, line in enumerate(lines) if line.startswith("global_atomic_add"))
            barrier = max(i for i in range(count) if lines[i].startswith("s_barrier"))
            for end in (barrier, count):
                waited = max(i for i in range(end) if "s_waitcnt" in lines[i] and "vmcnt(0)" in lines[i])
                stores = [line for line in lines[waited:end] if "global_store" in line]
                assert not stores, stores
            found += 1
    assert found == 3  # fp32, fp16, bf16
