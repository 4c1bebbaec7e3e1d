"""Build the orthossm_b200 C-ABI shared library in-tree with nvcc (sm_100a).

    python -m orthossm_b200.build            # -> orthossm_b200/_lib/liborthossm_b200.so

The library links the CUDA runtime dynamically (libcudart.so.12), so inside a
PyTorch process it shares torch's runtime and streams.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIBDIR = os.path.join(PKG, "_lib")
LIBNAME = "liborthossm_b200.so"
SOURCES = ["ossm_attn.cu", "ossm_attn_prompt.cu", "ossm_attn_token.cu", "ossm_capi.cu", "ossm_embed.cu",
           "ossm_forward.cu", "ossm_forward_3p.cu", "ossm_forward_grp.cu", "ossm_host.cu", "ossm_lce.cu",
           "ossm_lion.cu", "ossm_noalloc.cu", "ossm_norm.cu", "ossm_norm_bf16.cu", "ossm_norm_f16.cu", "ossm_norm_f32.cu",
           "ossm_norm_f32_bf16.cu", "ossm_norm_f32_f16.cu", "ossm_reverse.cu", "ossm_sample.cu", "ossm_ttt.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


def lib_path() -> str:
    return os.path.join(LIBDIR, LIBNAME)


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(LIBDIR, exist_ok=True)
    out = lib_path()
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    deps.append(os.path.join(INCLUDE, "orthossm_b200.h"))
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(d) for d in deps):
        return out
    stamps = {d: os.stat(d).st_mtime_ns for d in deps}
    cuda_lib = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "lib64")
    cc = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", f"-I{INCLUDE}", f"-I{CSRC}"]
    if verbose:
        cc.insert(1, "-Xptxas=-v")
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(os.cpu_count() or 1) as pool:
        objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in srcs]
        # a file a process (nvcc's own -split-compile made kernels up to half slower), the longest ones first
        order = sorted(zip(srcs, objs), key=lambda so: ("_norm_" not in so[0], -os.path.getsize(so[0])))
        cmds = [[*cc, "-c", "-o", o, s] for s, o in order]
        cmds_link = [nvcc(), *ARCH, "-shared", "-cudart", "shared", "-Xlinker", f"-rpath,{cuda_lib}", "-o", out + ".tmp",
                     *objs]
        if verbose:
            print("\n".join(" ".join(c) for c in [*cmds, cmds_link]), flush=True)
        list(pool.map(lambda c: subprocess.run(c, check=True), cmds))
        subprocess.run(cmds_link, check=True)
    # files compiled before and after an edit of a header do not agree on its structs
    changed = [os.path.basename(d) for d, t in stamps.items() if not os.path.exists(d) or os.stat(d).st_mtime_ns != t]
    if changed:
        os.unlink(out + ".tmp")
        raise RuntimeError(f"{', '.join(changed)} changed while the library was compiled: build again")
    os.replace(out + ".tmp", out)
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
