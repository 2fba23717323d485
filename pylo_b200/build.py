"""Compile the CUDA sources into the in-tree shared library (plain nvcc, sm_100a only)."""

import os
import shutil
import subprocess

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG_DIR), "include")
LIB_PATH = os.path.join(CSRC, "libpylo_b200.so")
LOCK_PATH = os.path.join(CSRC, ".build.lock")
SOURCES = [os.path.join(CSRC, name) for name in ("pylo_kernels.cu", "pylo_adamw.cu", "pylo_rows.cu", "pylo_ffn.cu")]
HEADERS = [os.path.join(CSRC, "pylo_common.cuh"), os.path.join(CSRC, "pylo_pipe.cuh"), os.path.join(CSRC, "pylo_small_front.cuh"), os.path.join(CSRC, "pylo_apply_tc.cuh"), os.path.join(CSRC, "pylo_ns_gemm.cuh"), os.path.join(CSRC, "pylo_ns_f16.cuh"), os.path.join(CSRC, "pylo_ns_cluster.cuh"), os.path.join(CSRC, "pylo_launch.cuh"), os.path.join(INCLUDE, "pylo_b200.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared",
]


def find_nvcc():
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand if os.path.exists(cand) else None


def is_stale():
    if not os.path.exists(LIB_PATH):
        return True
    built = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(f) > built for f in SOURCES + HEADERS if os.path.exists(f))


def build(force=False, verbose=False):
    """Build ``csrc/libpylo_b200.so``; returns its path.  Raises if nvcc is missing or fails.

    Safe to call from several processes at once (one rank per GPU importing the package): a file lock lets one of
    them compile, into a temporary file that is renamed over the library in one step, while the others wait and
    then find the library up to date."""
    if not force and not is_stale():
        return LIB_PATH
    nvcc = find_nvcc()
    if nvcc is None:
        raise RuntimeError("nvcc not found: cannot build pylo_b200/csrc/libpylo_b200.so")
    import fcntl

    with open(LOCK_PATH, "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if not force and not is_stale():   # another process built it while this one waited
                return LIB_PATH
            # PYLO_B200_NVCC_FLAGS: extra nvcc flags for a one-off build (e.g. -DTC_STAGE_CLOCKS for the stage
            # clocks of the tensor-core apply kernel)
            extra = os.environ.get("PYLO_B200_NVCC_FLAGS", "").split()
            tmp = f"{LIB_PATH}.tmp.{os.getpid()}"
            objects = [f"{tmp}.{os.path.basename(src)}.o" for src in SOURCES]
            command = [nvcc] + NVCC_FLAGS + extra + ["-I", INCLUDE, "-I", CSRC] + (["-Xptxas=-v"] if verbose else [])
            try:
                # the sources side by side, then the library
                runs = [subprocess.Popen(command + ["-c", "-o", obj, src], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
                        for src, obj in zip(SOURCES, objects)]
                said = [run.communicate()[0] for run in runs]
                if not any(run.returncode for run in runs):
                    link = subprocess.run([nvcc] + NVCC_FLAGS + ["-o", tmp] + objects, capture_output=True, text=True)
                    runs, said = runs + [link], said + [link.stdout + link.stderr]
                if any(run.returncode for run in runs):
                    raise RuntimeError("nvcc failed:\n" + "".join(said))
                os.replace(tmp, LIB_PATH)
            finally:
                for path in objects + [tmp]:
                    if os.path.exists(path):
                        os.remove(path)
            if verbose:
                print("".join(said))
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return LIB_PATH


if __name__ == "__main__":
    import sys

    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
