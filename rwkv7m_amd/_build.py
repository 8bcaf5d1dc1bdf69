"""Build librwkv7m_wkv.so in-tree with hipcc for gfx950, and the torch binding
of the language model head's operators and the gated delta rule beside it.

The library is plain ``extern "C"`` (include/*.h) with no torch or Python
types in its signatures; Python reaches it through ctypes, and for those
operators through ``_lm_head_torch.so`` (csrc/torch_*.cpp, host code).
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_NAME = "librwkv7m_wkv.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
TORCH_LIB_PATH = os.path.join(PKG_DIR, "_lm_head_torch.so")
ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    # Packed fp32 VALU forms are kept out of every code object.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found; cannot build librwkv7m_wkv.so")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC)
                  if f.endswith(".hip"))


def _torch_flags() -> tuple[list[str], list[str]]:
    """(compile, link) flags of the torch binding."""
    import torch
    from torch.utils import cpp_extension

    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]
    compile_ = ["-O2", "-std=c++17", "-fPIC", "-DTORCH_API_INCLUDE_EXTENSION_H",
                "-DTORCH_EXTENSION_NAME=_lm_head_torch",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                *(f for i in inc for f in ("-isystem", i))]
    dirs = cpp_extension.library_paths()
    link = [*(f for d in dirs for f in ("-L" + d, "-Wl,-rpath," + d)),
            "-Wl,-rpath,$ORIGIN", "-lc10", "-lc10_hip", "-ltorch_cpu",
            "-ltorch", "-ltorch_python"]
    return compile_, link


def build(verbose: bool = False, jobs: int = 8) -> str:
    """Compile every csrc/*.hip for gfx950 and link the shared library, then
    the torch binding against it."""
    hipcc = _hipcc()
    os.makedirs(BUILD_DIR, exist_ok=True)
    objs = []
    bindings = [os.path.join(CSRC, f)
                for f in ("torch_lm_head.cpp", "torch_gated_delta.cpp")]
    torch_compile, torch_link = _torch_flags()

    def compile_one(src: str) -> str:
        obj = os.path.join(BUILD_DIR,
                           os.path.splitext(os.path.basename(src))[0] + ".o")
        flags = torch_compile if src in bindings else HIPCC_FLAGS
        cmd = [hipcc, *flags, "-c", src, "-o", obj]
        res = subprocess.run(cmd, capture_output=True, text=True)
        msg = "\n".join(line for line in (res.stdout + res.stderr).splitlines()
                        if "packed-fp32-ops" not in line)
        if res.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{msg}")
        if verbose and msg.strip():
            print(msg)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        # (the bindings take longest: first)
        objs = list(pool.map(compile_one, [*bindings, *sources()]))
    binding_objs, objs = objs[:len(bindings)], objs[len(bindings):]
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs,
           "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}{res.stderr}")
    os.replace(tmp, LIB_PATH)
    tmp = TORCH_LIB_PATH + ".tmp"
    cmd = [hipcc, "-shared", "-fPIC", "-no-hip-rt", *binding_objs,
           "-L" + PKG_DIR, "-l:" + LIB_NAME, *torch_link, "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}{res.stderr}")
    os.replace(tmp, TORCH_LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
