"""Builds libngpt_fp8.so (all HIP kernels + the C ABI) for gfx950 with hipcc, in-tree, and the host-side torch binding beside it.

    python -m modded_nanogpt_amd.build          # from the repository root
    python modded-nanogpt_amd/build.py          # where there is no torch: the library alone, for programs that use its C ABI

hipcc cross-compiles without a GPU.  The library lands in modded-nanogpt_amd/lib/ so it travels
with the source tree; nothing is installed into site-packages.
"""
from __future__ import annotations

import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB_PATH = LIB_DIR / "libngpt_fp8.so"
BINDING_PATH = LIB_DIR / "_ngpt_torch.so"             # torch_binding.cpp: host code that calls the library for torch tensors
BENCH_LIB_PATH = LIB_DIR / "libngpt_fp8_bench.so"     # + the timing aids behind NGPT_BENCH_BUILD, for measurements only
SOURCES = ["gemm_api.hip", "quant.hip", "ce.hip", "mlp_aux.hip", "linear.hip", "linear_small.hip", "qk_rope.hip", "distill.hip", "bench_kernels.hip"]   # the last one is empty without NGPT_BENCH_BUILD

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    # keep the compiler from forming packed-fp32 VALU ops out of scalar float code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc_path() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or add /opt/rocm/bin to PATH)")


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print("+", " ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    # the host pass does not know the device-only feature flag and says so once per file
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in proc.stderr.splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"{pathlib.Path(cmd[0]).name} failed ({proc.returncode}):\n{err}")
    if verbose and err.strip():
        print(err, file=sys.stderr)


def _binding_commands(obj: str, lib_dir: str) -> tuple[list[str], list[str]]:
    """Commands that compile and link the torch binding (host code only)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        raise RuntimeError("no C++ compiler for the torch binding")
    rocm = pathlib.Path(hipcc_path()).resolve().parent.parent
    compile_ = [cxx, "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                *[f"-isystem{p}" for p in include_paths()], f"-isystem{rocm / 'include'}", "-isystem/opt/rocm/include",
                f"-I{sysconfig.get_paths()['include']}", "-c", "-o", obj, str(CSRC / "torch_binding.cpp")]
    link = [cxx, "-shared", "-o", str(BINDING_PATH) + ".tmp", obj, f"-L{lib_dir}", "-l:libngpt_fp8.so", *[f"-L{p}" for p in library_paths()],
            "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def build(verbose: bool = True, bench: bool = False) -> pathlib.Path:
    """Compile every HIP source into one shared library; always recompiles.  `bench`: the measurement build.
    The torch binding needs torch and is left out where there is none; where it fails, the library is in place all the same."""
    LIB_DIR.mkdir(exist_ok=True)
    srcs = [str(CSRC / s) for s in SOURCES if (CSRC / s).exists()]
    out = BENCH_LIB_PATH if bench else LIB_PATH
    tmp = out.with_suffix(".so.tmp")
    flags = [*[f for f in HIPCC_FLAGS if f != "-shared"], *(["-DNGPT_BENCH_BUILD"] if bench else []), "-I", str(PKG.parent / "include")]
    with tempfile.TemporaryDirectory() as objdir:
        # one object a source, compiled side by side, then one link
        def compile_binding() -> list[str]:
            compile_, link = _binding_commands(str(pathlib.Path(objdir) / "torch_binding.o"), str(LIB_DIR))
            _run(compile_, verbose)
            return link

        objs = [str(pathlib.Path(objdir) / (pathlib.Path(s).stem + ".o")) for s in srcs]
        jobs = [[hipcc_path(), *flags, "-c", "-o", o, c] for c, o in zip(srcs, objs)]
        with_torch = not bench and importlib.util.find_spec("torch") is not None
        with ThreadPoolExecutor(max_workers=min(len(jobs) + 1, os.cpu_count() or 1, 8)) as pool:
            binding = pool.submit(compile_binding) if with_torch else None
            list(pool.map(lambda job: _run(job, verbose), jobs))
            _run([hipcc_path(), *HIPCC_FLAGS, "-o", str(tmp), *objs], verbose)
            os.replace(tmp, out)
            if binding:
                _run(binding.result(), verbose)
                os.replace(str(BINDING_PATH) + ".tmp", BINDING_PATH)
        if verbose and not bench and not with_torch:
            print("no torch: the library without its torch binding", flush=True)
    return out


if __name__ == "__main__":
    print(build())
    try:
        print(build(bench=True))
    except RuntimeError as e:      # only `bench.py --workload ceiling` needs it
        print("warning: the measurement build failed:", str(e)[:500], file=sys.stderr)
