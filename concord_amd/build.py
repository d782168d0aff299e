"""Build libconcord_amd.so (the gfx950 HIP kernels + C ABI) in-tree.

    python -m concord_amd.build        # or concord_amd.build.build()

Every .hip file under concord_amd/csrc is compiled with hipcc for gfx950 and
linked into concord_amd/_lib/libconcord_amd.so.  Flags:
  -ffp-contract=off   the numerical contract forbids FMA contraction;
  -Xclang -target-feature -Xclang -packed-fp32-ops
                      no v_pk_*_f32 instructions in device code.
Per-file extras (FILE_FLAGS): gemm_fast.hip keeps MFMA accumulators in
ordinary VGPRs (-amdgpu-mfma-vgpr-form); its kernels are written to fit them,
and the accumulator-register form made the compiler copy accumulators
around the main loops.

torch_ops.cpp (host code: autograd nodes over the library's entries) becomes
concord_amd/_lib/concord_torch_ops.so, against the installed torch.  Where that
fails the build does, with the C library in place.
"""
import glob
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "libconcord_amd.so")
OPS = os.path.join(OUT_DIR, "concord_torch_ops.so")
ARCH = os.environ.get("CONCORD_OFFLOAD_ARCH", "gfx950")

CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
    "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
]

FILE_FLAGS = {"gemm_fast.hip": ["-mllvm", "--amdgpu-mfma-vgpr-form"]}


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass does not know the device-only feature flag: drop that line
    err = "\n".join(l for l in r.stderr.splitlines()
                    if "packed-fp32-ops" not in l and "is not a recognized feature" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"command failed: {' '.join(cmd)}\n{err}")
    return err


def _ops_flags():
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "/opt/rocm/include", sysconfig.get_paths()["include"], os.path.join(ROOT, "include")]
    cflags = ["-O2", "-std=c++17", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
              "-DTORCH_EXTENSION_NAME=concord_torch_ops"] + [a for i in inc for a in ("-isystem", i)]
    libs = ["-L" + os.path.join(root, "lib"), "-L" + OUT_DIR, "-lconcord_amd", "-ltorch", "-ltorch_cpu", "-lc10",
            "-lc10_hip", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    return cflags, libs


def build(verbose=False, jobs=8):
    os.makedirs(OUT_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    objs = [os.path.join(OUT_DIR, os.path.basename(s)[:-4] + ".o") for s in srcs]

    ops_src, ops_obj = os.path.join(CSRC, "torch_ops.cpp"), os.path.join(OUT_DIR, "torch_ops.o")

    def compile_one(s, o):
        return _run([HIPCC] + CFLAGS + FILE_FLAGS.get(os.path.basename(s), []) + ["-c", s, "-o", o])

    def compile_ops():
        cflags, libs = _ops_flags()
        return _run([CXX] + cflags + ["-c", ops_src, "-o", ops_obj]), libs

    def show(msg):
        if verbose and msg.strip():
            print(msg, file=sys.stderr)

    with ThreadPoolExecutor(max_workers=jobs) as ex:
        ops = ex.submit(compile_ops)
        for msg in ex.map(compile_one, srcs, objs):
            show(msg)
        # the C library first: a binding without torch needs neither g++ nor torch's headers
        tmp = LIB + ".tmp"
        _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp] + objs)
        os.replace(tmp, LIB)
        for o in objs:
            os.remove(o)
        msg, ops_libs = ops.result()
        show(msg)
    _run([CXX, "-shared", "-o", OPS + ".tmp", ops_obj] + ops_libs)
    os.replace(OPS + ".tmp", OPS)
    os.remove(ops_obj)
    if verbose:
        print(f"built {LIB} and {OPS}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
