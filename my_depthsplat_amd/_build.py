"""Build the HIP extension libdsplat_hip.so in-tree (gfx950 only) and the CPU oracle.

Plain hipcc, no torch JIT cache: the .so lands in my_depthsplat_amd/lib/ so it travels
with the repository snapshot to the GPU box (it is git-ignored, not gpurun-ignored).
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "lib" / "libdsplat_hip.so"
TORCH_LIB = PKG / "lib" / "dsplat_torch.so"
OBJ = PKG / "lib" / "obj"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# -ffp-contract=off: the preprocess arithmetic must match the oracle bit for bit (sort keys,
# radii, tile rects). -munsafe-fp-atomics: native global_atomic_add_f32 (no CAS loop).
CFLAGS = [
    "-O3", "-std=c++17", f"--offload-arch={ARCH}", "-fPIC", "-ffp-contract=off",
    "-munsafe-fp-atomics", "-Wall", "-Wno-unused-function", "-I", str(ROOT / "include"),
]


# No packed FP32 instructions: some of their forms give wrong results now and then on this hardware
# (hipcc's host pass warns that it does not know the feature).
CFLAGS += ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# Per-file extra flags. The rasterizer's per-lane pixel math is scalar by design (pairs of list
# entries are written out with explicit vector types, which compile to scalar FMAs as above);
# the SLP vectorizer packs the scalar parts with register shuffles (k_render_bwd 119 -> 109 us
# without it at config B while packed FP32 was on; without that 90.6 K views/s against 90.3 K
# with the vectorizer, 16 scenes of 2 views at 256 x 256).
FILE_FLAGS = {"dsr_raster.hip": ["-fno-slp-vectorize"],
              # nothing there has to match another kernel bit for bit (the fused norm matches the plain one)
              **{f: ["-ffp-contract=fast"] for f in ("dtk_rotary.hip", "dtk_attention.hip", "dtk_attention_f32.hip",
                                                   "dtk_attention_bf16.hip", "dtk_attention_f16.hip")}}


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def _needs(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_hip(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    headers = list(CSRC.glob("*.h")) + [ROOT / "include" / "dsplat_hip.h", Path(__file__)]
    srcs = _sources()
    jobs = []
    for s in srcs:
        o = OBJ / (s.stem + ".o")
        if force or _needs(o, [s] + headers):
            jobs.append((s, o))

    def compile_one(job):
        s, o = job
        cmd = [HIPCC, *CFLAGS, *FILE_FLAGS.get(s.name, []), "-c", str(s), "-o", str(o)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for {s.name}:\n{r.stderr}")
        return o

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(compile_one, jobs))
    objs = [OBJ / (s.stem + ".o") for s in srcs]
    if force or jobs or _needs(LIB, objs):
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(LIB), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc link failed:\n{r.stderr}")
    return LIB


def build_torch(force: bool = False) -> Path:
    """The operators' torch layer (csrc/dtk_torch.cpp): host code against this torch's headers. It needs no
    HIP library to link to (its functions are bound by address when it is loaded)."""
    src = CSRC / "dtk_torch.cpp"
    OBJ.mkdir(parents=True, exist_ok=True)
    if not force and not _needs(TORCH_LIB, [src, ROOT / "include" / "dsplat_hip.h", Path(__file__)]):
        return TORCH_LIB
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ext
    libdir = Path(torch.__file__).resolve().parent / "lib"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in (*ext.include_paths("cuda"), sysconfig.get_paths()["include"])),
           str(src), "-o", str(TORCH_LIB), f"-L{libdir}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{r.stderr}")
    return TORCH_LIB


def build_oracle() -> Path:
    r = subprocess.run(["make", "-s", "-C", str(ROOT / "oracle")], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"oracle build failed:\n{r.stdout}\n{r.stderr}")
    return ROOT / "oracle" / "build" / "libdsr_oracle.so"


if __name__ == "__main__":
    print(build_hip(force="--force" in sys.argv, verbose=True))
    print(build_torch(force="--force" in sys.argv))
    print(build_oracle())
