"""Builds libvitb200.so (the sm_100a kernels + C ABI) in-tree with nvcc, and
_serving.so (csrc/bindings.cpp: the serving operators' Python entry points,
compiled against the installed PyTorch, and left out where there is none) with g++.

    python vit-engine-cuda_b200/build.py [--force] [--jobs N]

The library lands next to the Python package (vit_cuda/libvitb200.so) so that it
travels with the source tree; it links the CUDA runtime statically and resolves
the driver's tensor-map encoder at run time, so it loads on a machine without a
GPU (the kernels themselves need an sm_100a device).
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
OUT_DIR = os.path.join(HERE, "vit_cuda")
LIB = os.path.join(OUT_DIR, "libvitb200.so")
OBJ_DIR = os.path.join(HERE, "_build")
BINDINGS = os.path.join(CSRC, "bindings.cpp")
BINDINGS_LIB = os.path.join(OUT_DIR, "_serving.so")
BINDINGS_STAMP = os.path.join(OBJ_DIR, "_serving.built_for")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-Xptxas", "-v",
    # No -use_fast_math: the parity kernels rely on IEEE division, sqrt, expf, erff.
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found")
    return path


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def headers() -> list[str]:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs.append(os.path.join(INCLUDE, "vitb200.h"))
    return hs


def newer_than(lib: str, inputs: list[str]) -> bool:
    if not os.path.exists(lib):
        return False
    t = os.path.getmtime(lib)
    return all(os.path.getmtime(f) <= t for f in inputs)


def up_to_date() -> bool:
    return newer_than(LIB, sources() + headers() + [__file__])


def torch_package() -> str | None:
    """PyTorch's directory, found without importing it; None where it is not installed."""
    spec = importlib.util.find_spec("torch")
    return spec.submodule_search_locations[0] if spec else None


def built_for(torch_dir: str) -> str:
    """The PyTorch that _serving.so is compiled against (its ABI differs by version)."""
    with open(os.path.join(torch_dir, "version.py")) as f:
        return re.search(r"__version__ = ['\"](.*?)['\"]", f.read()).group(1)


def build_bindings(force: bool = False) -> str | None:
    torch_dir = torch_package()
    if torch_dir is None:
        print("PyTorch is not installed: libvitb200.so (the C ABI) is built without vit_cuda/"
              "_serving.so, the serving operators' Python entry points", file=sys.stderr)
        return None
    header = os.path.join(INCLUDE, "vitb200.h")
    version = built_for(torch_dir)
    # File times say nothing about the PyTorch and the interpreter they were built for.
    stamp, wanted = BINDINGS_STAMP, f"{version}\n{sysconfig.get_config_var('EXT_SUFFIX')}\n"
    if not force and newer_than(BINDINGS_LIB, [BINDINGS, header, __file__]):
        if os.path.exists(stamp) and open(stamp).read() == wanted:
            return BINDINGS_LIB
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    includes = [os.path.join(torch_dir, "include"),
                os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"], INCLUDE]
    tmp = BINDINGS_LIB + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++20", "-fPIC", "-shared",
           "-fvisibility=hidden", f'-DVITB200_BUILT_FOR="{version}"',
           *(f"-I{d}" for d in includes), BINDINGS, "-o", tmp,
           f"-L{os.path.join(torch_dir, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDINGS}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDINGS_LIB)
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(wanted)
    return BINDINGS_LIB


def compile_one(src: str) -> tuple[str, str]:
    obj = os.path.join(OBJ_DIR, os.path.basename(src).replace(".cu", ".o"))
    cmd = [nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr


# Kernels that move registers between warpgroups with setmaxnreg, and the
# per-thread register count their split assumes. csrc/attention_f16.cu and
# csrc/attention_f16_tile.cu: 384 threads launched at 168, as csrc/gemm_fp8.cu's
# CTA-pair kernel and csrc/cross_attention.cu's tile kernel. csrc/gemm_tcgen05.cu: the last template argument
# (EPI, the number of epilogue warpgroups) sets it: 2 -> 384 threads at 168,
# 3 -> 512 threads at 128, 4 -> 640 threads at 96 (EpiCfg there). A kernel compiled to any other count
# could make setmaxnreg.inc wait forever.
def expected_registers(mangled: str) -> int | None:
    if any(k in mangled for k in ("attention_f16_kernel", "attention_f16_tile_kernel",
                                  "gemm_fp8_pair_kernel", "cross_attention_kernel")):
        return 168
    m = re.search(r"gemm_tf32x3_kernelI(.*?)EEv", mangled)
    if m:
        epi = int(re.findall(r"Li(\d+)E", m.group(1) + "E")[-1])
        return {2: 168, 3: 128, 4: 96}[epi]
    return None


def check_register_split(ptxas_log: str) -> None:
    current, expected = None, None
    for line in ptxas_log.splitlines():
        if "Compiling entry function" in line:
            current = line.split("'")[1] if "'" in line else line
            expected = expected_registers(current)
        elif expected is not None and "Used" in line and "registers" in line:
            used = int(line.split("Used")[1].split("registers")[0])
            if used != expected:
                raise RuntimeError(
                    f"{current} compiled to {used} registers per thread; its setmaxnreg split "
                    f"requires exactly {expected}")
            current, expected = None, None


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> str:
    with ThreadPoolExecutor(max_workers=1) as ex:
        bindings = ex.submit(build_bindings, force)
        lib = build_library(force, jobs, verbose)
        bindings.result()
    return lib


def build_library(force: bool = False, jobs: int | None = None, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        results = list(ex.map(compile_one, srcs))
    for _, log in results:
        check_register_split(log)
        if verbose:
            sys.stderr.write(log)
    objs = [o for o, _ in results]
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/smem usage")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.jobs, verbose=a.verbose))


if __name__ == "__main__":
    main()
