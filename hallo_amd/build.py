"""Build libhallo_amd.so (the gfx950 operator library) in-tree with hipcc.

hipcc cross-compiles for gfx950 without a GPU, so this runs in the authoring container as
well as on the MI355X box.  The library is placed next to this file so that it travels with
the repository snapshot (it is git-ignored, not gpurun-ignored).
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libhallo_amd.so")
SOURCES = ["gemm.hip", "gemm3.hip", "gemm4.hip", "gemm_rs.hip", "gemm_rs2.hip", "gemm_ff.hip", "attention.hip", "attention40.hip", "fp8.hip", "fused_xattn.hip", "norm_elementwise.hip", "wav2vec.hip",
           "norm_train.hip", "rope.hip", "window_attention.hip", "window_attention_bwd.hip"]
HEADERS = [os.path.join(CSRC, "common.h"), os.path.join(CSRC, "gemm_args.h"), os.path.join(CSRC, "attn_args.h"), os.path.join(CSRC, "window_args.h"), os.path.join(HERE, "..", "include", "hallo_amd.h")]

# No packed fp32 instructions (v_pk_add / mul / fma_f32): some of their forms give wrong results now and then on this hardware, and hipcc
# -O3 forms them from ordinary float code.  The host pass warns that it does not know the feature; that is harmless.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    return "hipcc"


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _flags(cmd):
    """Of a compile command, what decides about the object besides the sources."""
    return " ".join(cmd[1:cmd.index("-c")])


def _built_with(o):
    """The flags that an object was built with: other ones make it stale as a newer source does."""
    try:
        with open(o + ".flags") as f:
            return f.read()
    except OSError:
        return None


def build(force=False, verbose=False):
    """Compile every HIP source for gfx950 and link libhallo_amd.so.  Returns the library path."""
    hipcc = _hipcc()
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs, todo = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src.replace(".hip", ".o"))
        cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", *NO_PACKED_FP32, "-c", s, "-o", o]
        if os.environ.get("HALLO_ABLATIONS") == "1":      # timing-ablation switches of the row-stationary GEMMs (tools/cbench)
            cmd.insert(1, "-DHALLO_ABLATIONS")
        if force or _stale(o, [s] + HEADERS) or _built_with(o) != _flags(cmd):
            todo.append(cmd)
        objs.append(o)

    def compile_one(cmd):
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        with open(cmd[-1] + ".flags", "w") as f:
            f.write(_flags(cmd))

    with ThreadPoolExecutor(min(8, int(os.environ.get("MAX_JOBS") or 8), max(len(todo), 1))) as pool:
        list(pool.map(compile_one, todo))
    if force or _stale(LIB, objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
