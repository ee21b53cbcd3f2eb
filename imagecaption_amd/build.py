"""Build libcapdec.so (hand-written gfx950 HIP kernels + C ABI) in-tree with hipcc.

    python -m imagecaption_amd.build [--force]

Each ``csrc/*.hip`` is compiled to an object under ``csrc/_build/`` (skipped when up to date), then
linked into ``imagecaption_amd/libcapdec.so``.  hipcc cross-compiles for gfx950 without a GPU.
"""
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "_build")
LIB = os.path.join(HERE, "libcapdec.so")
CALLS = os.path.join(HERE, "_calls.so")
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 -- some of their operand forms have given wrong results on this hardware now
# and then, and -O3 makes them from ordinary float code.  (The host pass does not know the feature and says so: harmless.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# Per-file extras.  -amdgpu-mfma-vgpr-form: MFMA accumulators live in ordinary VGPRs (gfx950 has one unified register
# file) instead of AGPRs -- kernels that touch their accumulators with vector instructions between products (softmax
# rescale, masking, bf16 packing, stores) otherwise pay a v_accvgpr_read / _write pair around every such touch.
FILE_FLAGS = {
    "attention_bf16.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "attention_f32_ring.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "attention_packed.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    "attention_paged.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form=1"],
    # no SLP vectorisation in the files that hold the vector epilogue (gemm_common.h, epilogue_store_vec)
    "gemm_bf16s_dma.hip": ["-fno-slp-vectorize"],
    "gemm_bf16s_p8.hip": ["-fno-slp-vectorize"],
    "gemm_bf16s.hip": ["-fno-slp-vectorize"],
    "gemm_bf16.hip": ["-fno-slp-vectorize"],
    "gemm_f32x3.hip": ["-fno-slp-vectorize"],
    "gemm_f32.hip": ["-fno-slp-vectorize"],
}


EXTRA = os.environ.get("CAPDEC_EXTRA_FLAGS", "").split()  # diagnostic builds (-DCAPDEC_...); never set by the package


def _hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    raise RuntimeError("hipcc not found")


def _deps_mtime():
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    hdrs.append(os.path.join(os.path.dirname(HERE), "include", "capdec.h"))
    return max(os.path.getmtime(h) for h in hdrs)


def build(force=False, verbose=True):
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    hmt = _deps_mtime()
    hipcc = _hipcc()
    jobs = []
    for s in srcs:
        src, obj = os.path.join(CSRC, s), os.path.join(OBJ, s[:-4] + ".o")
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hmt):
            jobs.append((src, obj))

    def run(job):
        src, obj = job
        cmd = [hipcc] + FLAGS + FILE_FLAGS.get(os.path.basename(src), []) + EXTRA + ["-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr[-4000:]}")
        if verbose and r.stderr.strip():
            print(r.stderr[-2000:], file=sys.stderr)
        return obj

    if jobs:
        if verbose:
            print(f"[capdec build] compiling {len(jobs)} file(s): {[os.path.basename(j[0]) for j in jobs]}")
        with ThreadPoolExecutor(max_workers=min(6, len(jobs))) as ex:
            list(ex.map(run, jobs))
    objs = [os.path.join(OBJ, s[:-4] + ".o") for s in srcs]
    if jobs or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
        if verbose:
            print(f"[capdec build] linked {LIB}")
    build_calls(force, verbose)
    return LIB


def calls_stamp():
    """What a build of csrc/calls.cpp was made for: it reads torch's objects by their layout, and no loader checks that."""
    import torch
    return f"capdec calls for torch {torch.__version__} {torch.version.git_version} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)} {sys.implementation.cache_tag};"


def calls_fit():
    """Whether _calls.so is there and was built for the running torch and Python (its stamp is read, nothing of it is run)."""
    if not os.path.exists(CALLS):
        return False
    with open(CALLS, "rb") as f:
        return calls_stamp().encode() in f.read()


def _calls_need():
    """What a build of csrc/calls.cpp needs and this machine lacks; None: nothing."""
    try:
        import torch
    except ImportError:
        return "torch"
    if shutil.which("g++") is None:
        return "g++"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python.h"
    if not os.path.exists(os.path.join(os.path.dirname(torch.__file__), "include", "torch", "csrc", "autograd", "python_variable.h")):
        return "torch's headers"
    return None


def build_calls(force=False, verbose=True):
    """csrc/calls.cpp -> _calls.so: host code only, built against the installed torch.  It saves host time; without it the
    same calls go through ctypes, so a machine that has hipcc alone gets the library without it."""
    src, missing = os.path.join(CSRC, "calls.cpp"), _calls_need()
    if missing != "torch" and not force and calls_fit() and os.path.getmtime(CALLS) >= max(os.path.getmtime(src), _deps_mtime()):
        return
    if missing is not None:
        if os.path.exists(CALLS):  # made for another torch, or from older sources than the library
            os.remove(CALLS)
        if verbose:
            print(f"[capdec build] no {missing}: the direct calls ({os.path.basename(CALLS)}) are not built")
        return
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DCAPDEC_CALLS_STAMP="{calls_stamp()}"']
    cmd += ["-isystem" + i for i in inc] + [src, "-o", CALLS, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stderr[-4000:]}")
    if verbose:
        if r.stderr.strip():
            print(r.stderr[-2000:], file=sys.stderr)
        print(f"[capdec build] linked {CALLS}")


if __name__ == "__main__":
    build(force="--force" in sys.argv)
