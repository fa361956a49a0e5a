"""Build recipe for the gfx950 library.

    python 5_amd/csrc/build.py [-v]

compiles SRCS (the kernels and the C ABI declared in include/hcg_*.h) with
hipcc for gfx950, each to an object of its own, in parallel, and links them
into 5_amd/hc/gfx950/libhcg_gfx950.so, next to the Python code that loads it;
STAMPED_SRCS again with -DHCG_STAMPS into libhcg_gfx950_stamps.so, whose GEMM
kernels record per-workgroup timestamps for bench.py --stamps; hcg_probe.hip
(the hardware ceiling probes of include/hcg_probe.h, used by bench.py) into
libhcg_probe.so; and hcg_torch.cpp (host code: the device-tensor binding of
hcg_gemm_algo as a Python extension, linked against libhcg_gfx950.so) with
g++ against the installed PyTorch into _hcg_torch<EXT_SUFFIX>.
hipcc cross-compiles, so this runs on a machine without a GPU.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from collections.abc import Callable
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
STAMPED_SRCS = [os.path.join(HERE, f) for f in ("hcg_gemm.hip", "hcg_tile.hip", "hcg_mfma.hip")]
SRCS = STAMPED_SRCS + [os.path.join(HERE, f) for f in ("hcg_embed.hip", "hcg_norm.hip", "hcg_loss.hip")]
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(PKG, "hc", "gfx950", "libhcg_gfx950.so")
# The products' sources with -DHCG_STAMPS: the tiled and streaming kernels record
# per-workgroup timestamps (bench.py --stamps); never loaded by the package.
STAMPS_OUT = os.path.join(PKG, "hc", "gfx950", "libhcg_gfx950_stamps.so")
PROBE_SRCS = [os.path.join(HERE, "hcg_probe.hip")]
PROBE_OUT = os.path.join(PKG, "hc", "gfx950", "libhcg_probe.so")
TORCH_SRC = os.path.join(HERE, "hcg_torch.cpp")
TORCH_OUT = os.path.join(PKG, "hc", "gfx950", "_hcg_torch" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
ARCH = "gfx950"


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def flags() -> list[str]:
    return [
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++20",
        "-fPIC",
        # Packed fp32 VALU forms stay disabled for all device code.
        "-Xclang",
        "-target-feature",
        "-Xclang",
        "-packed-fp32-ops",
        f"-I{INCLUDE}",
        "-Wall",
    ]


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # The host pass does not know the device-only target feature; that
    # warning is expected and harmless.  Anything else is shown.
    noise = "'-packed-fp32-ops' is not a recognized feature for this target"
    err = "\n".join(line for line in proc.stderr.splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {what} ({proc.returncode}):\n{err}")
    if verbose and err.strip():
        print(err)


def _build_library(pool: ThreadPoolExecutor, srcs: list[str], out: str, extra: list[str], scratch: str,
                   verbose: bool) -> Callable[[], str]:
    """Starts compiling srcs; the result waits for that and links them into out."""
    os.makedirs(os.path.dirname(out), exist_ok=True)
    objs = [os.path.join(scratch, f"{os.path.basename(out)}.{os.path.basename(s)}.o") for s in srcs]
    jobs = [pool.submit(_run, [hipcc(), *flags(), *extra, "-c", s, "-o", o], os.path.basename(s), verbose)
            for s, o in zip(srcs, objs)]

    def link() -> str:
        for job in jobs:
            job.result()
        _run([hipcc(), *flags(), "-shared", *objs, "-o", out + ".tmp"], os.path.basename(out), verbose)
        os.replace(out + ".tmp", out)
        return out

    return link


def _compile_torch_binding(verbose: bool) -> str:
    """g++ on hcg_torch.cpp: PyTorch's headers and libraries, the HIP headers
    (host code only), and libhcg_gfx950.so found next to the module."""
    import torch.utils.cpp_extension as cpp

    import torch

    tmp = TORCH_OUT + ".tmp"
    # The C++ ABI the installed torch was built with (its headers' std::string
    # layout must match ours).
    abi = int(bool(torch._C._GLIBCXX_USE_CXX11_ABI))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
           "-DTORCH_EXTENSION_NAME=_hcg_torch", "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           *(f"-I{p}" for p in cpp.include_paths()), f"-I{sysconfig.get_paths()['include']}",
           "-I/opt/rocm/include", f"-I{INCLUDE}", TORCH_SRC, "-o", tmp,
           *(f"-L{p}" for p in cpp.library_paths()), "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu",
           "-ltorch_python", f"-L{os.path.dirname(OUT)}", "-l:libhcg_gfx950.so", "-Wl,-rpath,$ORIGIN",
           *(f"-Wl,-rpath,{p}" for p in cpp.library_paths())]
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stderr}")
    os.replace(tmp, TORCH_OUT)
    return TORCH_OUT


def build(verbose: bool = False) -> str:
    """Builds the library, the products' timestamped variant, the probe
    library and the device-tensor binding; returns the first."""
    with tempfile.TemporaryDirectory() as scratch, ThreadPoolExecutor(os.cpu_count() or 4) as pool:
        links = [_build_library(pool, srcs, out, extra, scratch, verbose)
                 for srcs, out, extra in ((SRCS, OUT, []), (STAMPED_SRCS, STAMPS_OUT, ["-DHCG_STAMPS"]),
                                          (PROBE_SRCS, PROBE_OUT, []))]
        outs = [link() for link in links]
    _compile_torch_binding(verbose)
    return outs[0]


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
