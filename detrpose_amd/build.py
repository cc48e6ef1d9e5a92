"""Build libdetrpose_hip.so (gfx950) in-tree from detrpose_amd/csrc.

    python -m detrpose_amd.build            # incremental
    python -m detrpose_amd.build --force    # rebuild everything

Each translation unit is compiled by hipcc in parallel into build/*.o, then linked into
detrpose_amd/lib/libdetrpose_hip.so. The .so is git-ignored but travels to the GPU box
with the repo snapshot.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(REPO, "build", "csrc")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libdetrpose_hip.so")
ARCH = os.environ.get("DETRPOSE_OFFLOAD_ARCH", "gfx950")


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found (ROCm required to build libdetrpose_hip.so)")


def _flags() -> list[str]:
    extra = os.environ.get("DETRPOSE_EXTRA_FLAGS", "").split()
    return ["-O3", "-fPIC", "-std=c++17", f"--offload-arch={ARCH}", "-Wall", "-Wno-unused-function",
            # no packed f32 instructions: some forms of v_pk_add / mul / fma_f32 have given wrong results on MI355X
            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
            "-I", os.path.join(REPO, "include")] + extra


# translation units no inference plan launches from (the training step's kernels, the token-sequence
# operators): left out of source_hash, so a training-only change keeps the inference line's
# committed PMC profile valid
TRAINING_ONLY = {"backbone_train.hip", "criterion.hip", "encoder_train.hip", "gemm.hip", "msda_train.hip",
                 "train.hip", "train_attn.hip", "preprocess.hip", "rms_norm.hip", "grad_clip.hip", "packed_attn_fwd.hip",
                 "packed_attn_bwd.hip", "packed_attn.h"}


def source_hash() -> str:
    """Content hash of everything that decides which kernels a plan launches and how they
    touch memory (kernel sources, the C-ABI header, the planner). Profiles committed under
    profiles/ record it, so bench.py only quotes measured HBM traffic for the exact code it
    is timing (the box receives no .git, so this is not a commit id)."""
    import hashlib
    h = hashlib.sha256()
    files = sorted(f for f in glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")) +
                   glob.glob(os.path.join(CSRC, "*.cpp")) if os.path.basename(f) not in TRAINING_ONLY)
    files += [os.path.join(REPO, "include", "detrpose_hip.h"), os.path.join(PKG, "engine.py")]
    for f in files:
        h.update(os.path.relpath(f, REPO).encode())
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


def lib_sources() -> list[str]:
    """Every file the library is compiled from (kernel sources, their headers, the C ABI)."""
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h")) +
                  glob.glob(os.path.join(CSRC, "*.cpp"))) + [os.path.join(REPO, "include", "detrpose_hip.h")]


def lib_source_hash() -> str:
    """Content hash of the library's sources. The build bakes it into the .so
    (dp_source_hash()); detrpose_amd._lib.load() refuses a library whose hash differs from
    the sources shipped beside it, so a stale prebuilt .so is never tested or benched."""
    import hashlib
    h = hashlib.sha256()
    for f in lib_sources():
        h.update(os.path.relpath(f, REPO).encode())
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


def _hash_object(build_dir: str) -> tuple[str, bool]:
    """build/<dir>/dp_source_hash.o exporting dp_source_hash(); rebuilt when the hash changes."""
    src = os.path.join(build_dir, "dp_source_hash.cpp")
    obj = src + ".o"
    txt = ('// generated by detrpose_amd/build.py: content hash of the sources this library was built from\n'
           f'extern "C" const char* dp_source_hash(void) {{ return "{lib_source_hash()}"; }}\n')
    if os.path.exists(obj) and os.path.exists(src) and open(src).read() == txt:
        return obj, False
    with open(src, "w") as f:
        f.write(txt)
    r = subprocess.run(["g++", "-O2", "-fPIC", "-c", src, "-o", obj], capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError("dp_source_hash.cpp: " + r.stdout + r.stderr)
    return obj, True


def _stale(obj: str, src: str, deps: list[str]) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(p) > t for p in [src] + deps)


def build(force: bool = False, verbose: bool = False, variant: str = "") -> str:
    """variant != '': build into build/csrc-<variant> and lib/variants/<variant>/ (A/B experiments,
    with DETRPOSE_EXTRA_FLAGS) instead of the production library."""
    global BUILD, LIB
    if variant:
        BUILD = os.path.join(REPO, "build", "csrc-" + variant)
        LIB = os.path.join(LIBDIR, "variants", variant, "libdetrpose_hip.so")
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    hipcc = _hipcc()
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    deps = glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(REPO, "include", "detrpose_hip.h")]
    # objects compiled with other flags are stale whatever their age
    stamp, flags = os.path.join(BUILD, "flags.txt"), " ".join(_flags())
    if not os.path.exists(stamp) or open(stamp).read() != flags:
        force = True
        if os.path.exists(stamp):   # until all are compiled, the objects are of no one set of flags
            os.remove(stamp)
    jobs = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s) + ".o")
        objs.append(o)
        if force or _stale(o, s, deps):
            jobs.append([hipcc, *_flags(), "-c", s, "-o", o])
    if jobs:
        nproc = max(1, min(len(jobs), int(os.environ.get("MAX_JOBS", os.cpu_count() or 4)), 16))
        with cf.ThreadPoolExecutor(nproc) as ex:
            for cmd, r in zip(jobs, ex.map(lambda c: subprocess.run(c, capture_output=True, text=True), jobs)):
                if verbose or r.returncode:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode:
                    raise RuntimeError(f"hipcc failed on {cmd[-3]}")
    with open(stamp, "w") as f:
        f.write(flags)
    hobj, hnew = _hash_object(BUILD)
    objs.append(hobj)
    if jobs or hnew or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
        os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    ap.add_argument("--variant", default="")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, variant=a.variant))
