"""Builds libt2s_hip.so in-tree with hipcc for gfx950 (cross-compiles without a GPU).

    python -m vitxt_gqa_amd.build [--force]
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libt2s_hip.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# -fno-slp-vectorize: under plain -O3 the SLP vectoriser packs adjacent scalar f32 multiplies / adds of the attention kernels
# into v_pk_mul_f32 / v_pk_fma_f32, which issue slower beside MFMAs than the scalar forms (MI355X_MICROARCH.md, per-instruction
# constants); measured on the attention backward: 6.10 -> 5.87 ms without dropout, 7.95 -> 7.76 ms with (B=8, same box)
# -packed-fp32-ops: no packed fp32 instructions at all, also where the code has pairs of floats: some of their forms have given wrong results on
# this card now and then, without an error.  The train step without them, on one box in turn: 659.1 / 659.6 -> 654.3 / 655.2 ms.
FLAGS = ["--offload-arch=gfx950", "-O3", "-fno-slp-vectorize", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
OBJ = os.path.join(HERE, "build")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")))


def _headers():
    h = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".inc"))]
    return h + [os.path.join(os.path.dirname(HERE), "include", "t2s_hip.h"), os.path.abspath(__file__)]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _object(src):
    return os.path.join(OBJ, os.path.basename(src) + ".o")


def _compile(src, verbose):
    cmd = [HIPCC] + FLAGS + ["-c", src, "-o", _object(src)]
    if verbose:
        print("[vitxt_gqa_amd.build]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def build(force=False, verbose=True):
    """One object per source file (only the stale ones, a few at a time), linked into OUT."""
    deps = sources() + _headers()
    if not force and not _stale(OUT, deps):
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    todo = [s for s in sources() if force or _stale(_object(s), [s] + _headers())]
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        list(pool.map(lambda s: _compile(s, verbose), todo))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT] + [_object(s) for s in sources()]
    if verbose:
        print("[vitxt_gqa_amd.build]", " ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
