"""Build the HIP library ``hsn_amd/libhsn_amd.so`` for gfx950 (MI355X), in-tree.

``python -m hsn_amd.build`` (or ``__graft_entry__.build()``) compiles every source under
``hsn_amd/csrc`` with ``hipcc --offload-arch=gfx950`` in parallel and links one shared library
exporting the C ABI of the headers under ``include/``. A manifest (``hsn_amd/libhsn_amd.json``)
records the SHA-256 of every source and of the library, so the loader can refuse a library built
from other sources. The host modules (``hsn_amd/host``: the trainer's pointer tables, the calls of the
language-model operators) are built beside it, each with a manifest of its own.
"""

from __future__ import annotations

import concurrent.futures
import hashlib
import json
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = ROOT / "_build"
LIBRARY = PKG / "libhsn_amd.so"
MANIFEST = PKG / "libhsn_amd.json"
ARCH = "gfx950"

#: hipcc flags. Packed fp32 arithmetic is switched off (the compiler would otherwise form
#: v_pk_* fp32 ops from scalar code); a*b+c may fuse where written apart, except where a file
#: says `#pragma clang fp contract(off)` (the router: the CPU path rounds every operation).
HIP_FLAGS = [
    "-O3",
    "-std=c++17",
    f"--offload-arch={ARCH}",
    "-fPIC",
    "-ffp-contract=fast-honor-pragmas",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.hip")) + list(CSRC.glob("*.cpp")))


def headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) +
                  list((ROOT / "include").glob("*.h")))


def _sha(path: Path) -> str:
    return hashlib.sha256(path.read_bytes()).hexdigest()


def hipcc() -> str:
    found = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(found).exists():
        raise RuntimeError("hipcc not found: the HIP library cannot be built")
    return found


def _stamp(src: Path) -> str:
    """Digest of what an object depends on: the source, every header and the flags."""
    h = hashlib.sha256(" ".join(HIP_FLAGS).encode())
    for path in [src, *headers()]:
        h.update(path.read_bytes())
    return h.hexdigest()


def _compile(src: Path, incremental: bool = False) -> Path:
    obj = BUILD / (src.name + ".o")
    stamp = BUILD / (src.name + ".stamp")
    digest = _stamp(src)
    if incremental and obj.is_file() and stamp.is_file() and stamp.read_text() == digest:
        return obj
    cmd = [hipcc(), *HIP_FLAGS, "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd[1:1] = ["-x", "hip"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{proc.stderr[-6000:]}")
    stamp.write_text(digest)
    return obj


def build(verbose: bool = False, incremental: bool = False) -> Path:
    """Compile and link the library; returns its path. ``incremental`` reuses an object whose
    source, headers and flags are unchanged since it was compiled (the default compiles all)."""
    BUILD.mkdir(exist_ok=True)
    srcs = sources()
    jobs = min(len(srcs), int(os.environ.get("MAX_JOBS", os.cpu_count() or 4)), 16)
    with concurrent.futures.ThreadPoolExecutor(max_workers=max(jobs, 1)) as pool:
        objs = list(pool.map(lambda src: _compile(src, incremental), srcs))
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr[-6000:]}")
    os.replace(tmp, LIBRARY)
    manifest = {
        "arch": ARCH,
        "library_sha256": _sha(LIBRARY),
        "sources": {str(p.relative_to(ROOT)): _sha(p) for p in srcs + headers()},
        "flags": HIP_FLAGS,
    }
    MANIFEST.write_text(json.dumps(manifest, indent=1, sort_keys=True) + "\n")
    if verbose:
        print(f"built {LIBRARY} ({LIBRARY.stat().st_size} bytes) from {len(srcs)} sources")
    return LIBRARY


#: The host helper modules, built with the host compiler against the installed PyTorch's headers and
#: libraries: the trainer's pointer tables (``hsn_amd/host/tables.cpp`` -> ``hsn_amd/_tables.so``) and
#: the language-model operators' calls (``hsn_amd/host/calls.cpp`` -> ``hsn_amd/_calls.so``).
HOST_MODULES = ("_tables", "_calls")


def _host_paths(name: str) -> tuple[Path, Path, Path]:
    """``(source, module, manifest)`` of a host helper module."""
    return PKG / "host" / f"{name[1:]}.cpp", PKG / f"{name}.so", PKG / f"{name}.json"


def _host_digest(source: Path) -> str:
    """Digest of what a host helper module depends on here: its source and the C ABI's headers."""
    h = hashlib.sha256(source.read_bytes())
    for path in sorted((ROOT / "include").glob("*.h")):
        h.update(path.read_bytes())
    return h.hexdigest()


def _build_host(name: str) -> Path:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    source, module, manifest = _host_paths(name)
    torch_lib = str(Path(torch.__file__).resolve().parent / "lib")
    tmp = module.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{p}" for p in cpp_extension.include_paths()],
           f"-isystem{sysconfig.get_paths()['include']}",
           str(source), "-o", str(tmp),
           f"-L{torch_lib}", "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python",
           f"-Wl,-rpath,{torch_lib}"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"host helper build failed on {source.name}:\n{proc.stderr[-6000:]}")
    os.replace(tmp, module)
    manifest.write_text(json.dumps({"source_sha256": _host_digest(source),
                                    "module_sha256": _sha(module)}, indent=1) + "\n")
    return module


def build_host(verbose: bool = False) -> list[Path]:
    """Compile the host helper modules (CPython extensions, host code only); returns their paths."""
    import torch  # noqa: F401  (imported once, before the threads)

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(HOST_MODULES)) as pool:
        modules = list(pool.map(_build_host, HOST_MODULES))
    if verbose:
        for module in modules:
            print(f"built {module} ({module.stat().st_size} bytes)")
    return modules


def host_stale(name: str = "_tables") -> str | None:
    """Why a host helper module is not the build of its current source, or None."""
    source, module, manifest_path = _host_paths(name)
    if not module.is_file() or not manifest_path.is_file():
        return f"hsn_amd/{module.name} is not built"
    manifest = json.loads(manifest_path.read_text())
    if manifest.get("module_sha256") != _sha(module):
        return f"hsn_amd/{module.name} differs from its build manifest"
    if manifest.get("source_sha256") != _host_digest(source):
        return f"hsn_amd/host/{source.name} or a header changed since hsn_amd/{module.name} was built"
    return None


def stale() -> str | None:
    """Why the built library does not match the sources (None: it matches)."""
    if not LIBRARY.is_file() or not MANIFEST.is_file():
        return "the HIP library is not built (python -m hsn_amd.build)"
    manifest = json.loads(MANIFEST.read_text())
    if manifest.get("library_sha256") != _sha(LIBRARY):
        return "libhsn_amd.so differs from its build manifest"
    for name, digest in manifest.get("sources", {}).items():
        path = ROOT / name
        if not path.is_file() or _sha(path) != digest:
            return f"source changed since the build: {name}"
    for path in sources() + headers():
        if str(path.relative_to(ROOT)) not in manifest.get("sources", {}):
            return f"source added since the build: {path.relative_to(ROOT)}"
    return None


if __name__ == "__main__":
    build(verbose=True, incremental="--incremental" in sys.argv[1:])
    build_host(verbose=True)
    sys.exit(0)
