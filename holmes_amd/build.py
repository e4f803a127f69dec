"""Compile the HIP sources of holmes_amd into holmes_amd/_lib/libholmes_ckks.so (gfx950).

Run ``python -m holmes_amd.build`` (or ``__graft_entry__.build()``).  Each ``.hip`` file is
compiled to an object in parallel, then linked into one shared library exporting the C ABI of
``include/holmes_ckks.h``.  ``csrc/clear_bind.cpp`` and ``csrc/window_bind.cpp``, the Python sides of the cleartext
operators, become the extension modules holmes_amd/_lib/_clear.so and _window.so (host code only, against the installed
PyTorch).  They take g++ and PyTorch's and Python's headers; where these are missing the library is there all the same, and
only ``holmes_amd.clear`` is not.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_lib"
LIB = OUT_DIR / "libholmes_ckks.so"
CLEAR = OUT_DIR / "_clear.so"
BINDINGS = {"clear_bind.cpp": "_clear.so", "window_bind.cpp": "_window.so"}   # beside the library
ARCH = os.environ.get("HOLMES_AMD_ARCH", "gfx950")

SOURCES = ["context.hip", "ntt.hip", "poly.hip", "keyswitch.hip", "ksfused.hip", "bsgs.hip", "encode.hip",
           "mul.hip", "noalloc.hip", "wide.hip", "wide_fused.hip", "kv4.hip", "kv4_attend.hip", "kv4_prompt.hip",
           "scores.hip", "rotary.hip", "prompt.hip", "kv4_weigh.hip", "kv4_evict.hip"]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "-O3",
    "-std=c++17",
    f"--offload-arch={ARCH}",
    "-fPIC",
    # packed FP32 instructions are kept out of every kernel (some of their forms have given
    # wrong results on these boxes); FP64 code does not need them.
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-Wno-unused-result",
    f"-I{ROOT / 'include'}",
]


def _compile(src: str, build_dir: Path) -> Path:
    obj = build_dir / (Path(src).stem + ".o")
    cmd = [HIPCC, *FLAGS, "-c", str(CSRC / src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stderr}")
    return obj


def _compile_binding(build_dir: Path) -> dict:
    import torch
    from torch.utils import cpp_extension

    paths = [*cpp_extension.include_paths(), str(Path(HIPCC).resolve().parent.parent / "include"), "/opt/rocm/include",
             sysconfig.get_paths()["include"]]

    def one(src: str) -> Path:
        obj = build_dir / (Path(src).stem + ".o")
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__=1",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-isystem{p}" for p in paths), "-c", str(CSRC / src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"g++ failed for {src}:\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=len(BINDINGS)) as pool:
        return dict(zip(BINDINGS.values(), pool.map(one, BINDINGS)))


def _link_binding(objs: dict) -> None:
    import torch

    made = {}
    for name, obj in objs.items():
        made[name] = tmp = (OUT_DIR / name).with_suffix(f".so.tmp{os.getpid()}")
        cmd = ["g++", "-shared", "-o", str(tmp), str(obj), f"-L{OUT_DIR}", f"-l:{LIB.name}",
               f"-L{Path(torch.__file__).parent / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python",
               "-Wl,-rpath,$ORIGIN"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stderr}")
    for name, tmp in made.items():   # all or none
        os.replace(tmp, OUT_DIR / name)


def build(verbose: bool = False) -> Path:
    build_dir = OUT_DIR / "obj"
    build_dir.mkdir(parents=True, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(len(SOURCES) + 1, 8)) as pool:
        binding = pool.submit(_compile_binding, build_dir)
        objs = list(pool.map(lambda s: _compile(s, build_dir), SOURCES))
    tmp = LIB.with_suffix(f".so.tmp{os.getpid()}")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)
    try:
        _link_binding(binding.result())
    except (ImportError, OSError, RuntimeError) as e:  # no PyTorch, no g++, or one of them failed
        for name in BINDINGS.values():
            (OUT_DIR / name).unlink(missing_ok=True)   # none rather than an old one
        print(f"holmes_amd.clear is not available: its extension modules were not built: {e}", file=sys.stderr)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
