"""Build libmlpk.so (the C-ABI CUDA library) in-tree for sm_100a.

Usage: ``python -m mlp_megakernel_b200.build`` (or ``__graft_entry__.build()``).
The library is written next to this file as ``lib/libmlpk.so`` so it travels
with the source tree; nothing is installed into site-packages.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libmlpk.so")
BINDING = os.path.join(LIBDIR, "mlpk_torch.so")
BINDING_SRC = "torch_binding.cpp"

# Each translation unit with the headers it is built from.
SOURCES = {
    "mlpk_api.cu": ["host.cuh", "pdl.cuh", "ptx.cuh", "layout.cuh", "softplus.cuh", "fwd_kernel.cuh", "bwd_kernel.cuh",
                    "wn_kernel.cuh", "stream_kernel.cuh", "wgrad_kernel.cuh", "peer_kernel.cuh", "cast_kernel.cuh"],
    **{f"norm_{part}.cu": ["host.cuh", "pdl.cuh", "vec.cuh", "norm_kernel.cuh", "norm_launch.cuh"]
       for part in ("api", "f16", "bf16", "f32")},
    "expert_api.cu": ["host.cuh", "pdl.cuh", "vec.cuh", "expert_plan.cuh", "expert_kernel.cuh"],
    **{f"product_{part}.cu": ["host.cuh", "pdl.cuh", "ptx.cuh", "pair.cuh", "layout.cuh", "softplus.cuh", "vec.cuh",
                              "act.cuh", "product_epi.cuh", "product_kernel.cuh", "product_launch.cuh",
                              "product_plan.cuh", "tail_kernel.cuh", "few_rows_plan.cuh", "few_rows_kernel.cuh", "product_type.cuh"] for part in ("f16", "bf16")},
    "ff_api.cu": ["host.cuh", "pdl.cuh", "ptx.cuh", "softplus.cuh", "vec.cuh", "act.cuh", "product_epi.cuh",
                  "product_launch.cuh", "ff_kernel.cuh"],
    "adamw_api.cu": ["host.cuh", "pdl.cuh", "vec.cuh", "adamw_kernel.cuh"],
}

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-diag-suppress", "20013",
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the CUDA library cannot be built")


def _inputs(source: str) -> list:
    return [os.path.join(CSRC, f) for f in [source, *SOURCES[source]]] + \
        [os.path.join(ROOT, "include", "mlpk.h"), os.path.abspath(__file__)]


def _object(source: str) -> str:
    return os.path.join(LIBDIR, source[:-3] + ".o")


def _newer(files, target: str) -> bool:
    """Whether the target is missing or older than one of the files."""
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(f) > t for f in files if os.path.exists(f))


def _stale() -> bool:
    return any(_newer(_inputs(s), LIB) for s in SOURCES)


DEVTEST_SRC = os.path.join(ROOT, "tests", "device_api", "devtest.cu")
DEVTEST_LIB = os.path.join(ROOT, "tests", "device_api", "libmlpk_devtest.so")


def build_devtest(force: bool = False, verbose: bool = False) -> str:
    """Compile the device-API test kernels (tests/device_api/devtest.cu, a
    user kernel calling include/mlpk_device.cuh) if missing or stale."""
    deps = [DEVTEST_SRC, os.path.join(ROOT, "include", "mlpk_device.cuh")] + \
        [os.path.join(CSRC, f) for f in SOURCES["mlpk_api.cu"] + ["device_mlp.cuh"]]
    if not force and os.path.exists(DEVTEST_LIB) and \
            all(os.path.getmtime(f) <= os.path.getmtime(DEVTEST_LIB) for f in deps if os.path.exists(f)):
        return DEVTEST_LIB
    tmp = DEVTEST_LIB + ".tmp"
    cmd = [nvcc_path(), *NVCC_FLAGS, "-shared", "-o", tmp, DEVTEST_SRC]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, DEVTEST_LIB)
    return DEVTEST_LIB


def _run(cmd, verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    return res.stdout + res.stderr


def _compile(source: str, verbose: bool, ptxas_info: bool) -> str:
    obj = _object(source)
    cmd = [nvcc_path(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if ptxas_info else []), "-c",
           "-o", obj + ".tmp", os.path.join(CSRC, source)]
    said = _run(cmd, verbose)
    os.replace(obj + ".tmp", obj)
    return said


def _torch_flags() -> list:
    """What the binding's compiler needs to find torch, Python and the library."""
    from torch.utils import cpp_extension

    flags = [f"-I{p}" for p in cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]]
    flags += [f"-L{p}" for p in cpp_extension.library_paths("cuda") + [LIBDIR]]
    return flags + ["-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10", "-l:libmlpk.so",
                    "-Wl,-rpath,$ORIGIN"]


def built_for() -> str:
    """What the binding is compiled against: another torch or Python may have other
    layouts under the same names."""
    import torch

    return f"mlpk_torch for torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"


def _binding_stale() -> bool:
    if _newer([os.path.join(CSRC, BINDING_SRC), os.path.join(ROOT, "include", "mlpk.h"), os.path.abspath(__file__)],
              BINDING):
        return True
    with open(BINDING, "rb") as f:
        return built_for().encode() + b"\0" not in f.read()


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile the torch binding of the block operators (host code only) if it is
    missing, older than its source or of another torch; return its path."""
    if force or _binding_stale():
        _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
              f'-DMLPK_BUILT_FOR="{built_for()}"', "-o", BINDING + ".tmp", os.path.join(CSRC, BINDING_SRC),
              *_torch_flags()], verbose)
        os.replace(BINDING + ".tmp", BINDING)
    return BINDING


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    """Compile the translation units of libmlpk.so that are older than their
    sources, side by side, link the library if any was, and see to the torch
    binding; return the library's path."""
    if not force and not _stale():
        build_binding(verbose=verbose)
        return LIB
    os.makedirs(LIBDIR, exist_ok=True)
    todo = [s for s in SOURCES if force or _newer(_inputs(s), _object(s))]
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        said = "".join(pool.map(lambda s: _compile(s, verbose, ptxas_info), todo))
    said += _run([nvcc_path(), *NVCC_FLAGS, "-shared", "-o", LIB + ".tmp"] + [_object(s) for s in SOURCES], verbose)
    if verbose or ptxas_info:
        sys.stderr.write(said)
    os.replace(LIB + ".tmp", LIB)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, ptxas_info="-v" in sys.argv))
