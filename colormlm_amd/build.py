"""Build libs14hip.so in-tree for gfx950.

    python -m colormlm_amd.build

Each source is compiled to an object of its own (in parallel), then linked
into colormlm_amd/lib/libs14hip.so:

- the gfx950 kernel files (*.hip) with -ffp-contract=off (the exact kernels'
  multiply-then-add must stay unfused) and with packed FP32 instructions
  disabled (-Xclang -target-feature -Xclang -packed-fp32-ops).  Clang has no
  driver spelling that forwards an -Xclang pair to the device pass alone, so
  the host pass of these files prints a one-line notice that it does not
  know the feature; the device code objects are what the flag is for;
- the host-only translation units (*.cpp: the C ABI, the pool and loader
  contracts) without that flag.

Beside it lib/_s14attn.so, the attention calls' Python side (s14_attn_py.cpp, a
CPython extension over torch's headers and libraries, which are loaded before it;
left out where there is no torch).
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT = PKG / "lib" / "libs14hip.so"
PY_OUT = PKG / "lib" / "_s14attn.so"
OBJ = PKG / "lib" / "obj"
DEVICE_SOURCES = ["s14_device.hip", "s14_block.hip", "s14_prefill.hip", "s14_static.hip", "s14_linear.hip",
                  "s14_norm.hip", "s14_attn_rows.hip", "s14_attn_paged.hip", "s14_attn_append4.hip", "s14_attn_paged4.hip",
                  "s14_attn_prompt.hip"]
HOST_SOURCES = ["s14_api.cpp", "s14_attn_api.cpp", "s14_pool.cpp", "s14_loader.cpp"]
SOURCES = DEVICE_SOURCES + HOST_SOURCES
ARCH = os.environ.get("S14_OFFLOAD_ARCH", "gfx950")
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required)")


def common_flags() -> list:
    return [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall",
            f"-I{ROOT / 'include'}", f"-I{CSRC}"]


def compile_command(src: str) -> list:
    extra = NO_PACKED_FP32 if src.endswith(".hip") else []
    return [hipcc(), *common_flags(), *extra, "-c", str(CSRC / src), "-o", str(OBJ / (src + ".o"))]


def link_command(out: Path) -> list:
    return [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *[str(OBJ / (s + ".o")) for s in SOURCES],
            "-o", str(out)]


def command(out: Path = OUT) -> list:
    """The single-invocation form of the build (kept for reference): every
    source on one hipcc line."""
    return [hipcc(), *common_flags(), *NO_PACKED_FP32, "-shared",
            *[str(CSRC / s) for s in SOURCES], "-o", str(out)]


def python_command(out: Path = PY_OUT) -> list:
    import torch

    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++") or str(Path(hipcc()).parent / "amdclang++")
    home = Path(torch.__file__).resolve().parent
    inc = home / "include"
    return [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f"-I{sysconfig.get_paths()['include']}", f"-I{ROOT / 'include'}", "-isystem", str(inc), "-isystem",
            str(inc / "torch/csrc/api/include"), str(CSRC / "s14_attn_py.cpp"), f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-o", str(out)]


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"{Path(cmd[0]).name} failed with status {proc.returncode}: {' '.join(cmd[-3:])}")
    notes = [ln for ln in (proc.stdout + proc.stderr).splitlines()
             if ln.strip() and "packed-fp32-ops' is not a recognized feature" not in ln]
    if notes:
        sys.stderr.write("\n".join(notes) + "\n")


def build(verbose: bool = False) -> Path:
    OUT.parent.mkdir(parents=True, exist_ok=True)
    OBJ.mkdir(parents=True, exist_ok=True)
    jobs = min(len(SOURCES), int(os.environ.get("MAX_JOBS", "8")))
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        for f in [ex.submit(_run, compile_command(s), verbose) for s in SOURCES]:
            f.result()
    tmp = OUT.with_suffix(".so.tmp")
    _run(link_command(tmp), verbose)
    os.replace(tmp, OUT)
    if importlib.util.find_spec("torch") is None:
        print(f"{PY_OUT.name} is not built: there is no torch (colormlm_amd.attention needs both)", file=sys.stderr)
        return OUT
    tmp = PY_OUT.with_suffix(".so.tmp")
    _run(python_command(tmp), verbose)
    os.replace(tmp, PY_OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose=True))
