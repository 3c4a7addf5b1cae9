"""Builds lightfm_amd/_lib/liblfm_hip.so and liblfm_ops.so with hipcc for gfx950 (in-tree).

    python -m lightfm_amd.build [--force]

hipcc cross-compiles without a GPU.  -ffp-contract=off keeps the reference's
separate float32 multiply/add roundings (no FMA contraction);
-munsafe-fp-atomics selects the hardware global_atomic_add_f32.
"""
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "liblfm_hip.so")
OPS_LIB = os.path.join(OUT_DIR, "liblfm_ops.so")
SOURCES = ["fit_kernels.hip", "fit_kernels_wide.hip", "warp_tile.hip", "warp_tile_lpr16.hip", "warp_tile_lpr32.hip",
           "warp_tile_lpr64.hip", "warp_tile_ahead.hip", "warp_tile_bpr.hip", "logistic_tile.hip", "feat_kernels.hip", "feat_kernels_wide.hip", "feat_kernels_hot.hip", "feat_kernels_ada.hip", "hot_slices.hip", "predict_kernels.hip", "csr_build.hip", "softmax_epoch.hip", "session.hip"]
# the device-memory operators: in liblfm_ops.so with their C ABI, in liblfm_hip.so for the softmax epochs
OPS_SOURCES = ["softmax_loss.hip", "embedding_ops.hip", "clip_norm.hip"]
OPS_API = ["lfm_ops.hip"]
TORCH_OPS = "torch_ops.cpp"  # their binding for torch tensors (host code)
HEADERS = ["ops_common.hpp", os.path.join("..", "..", "include", "lfm_ops.h"), "device.hpp", "kernels.hpp", "pool.hpp", "warp_tile_kernel.hpp", "warp_tile_ahead.hpp", "warp_tile_narrow.hpp", "feat_kernel.hpp", os.path.join("..", "..", "include", "lfm_hip.h")]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-munsafe-fp-atomics", "-Wall", "-Wno-unused-function",
         # no packed float32 instructions: some of their forms have given wrong results on MI355X
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
if os.environ.get("LFM_BUILD_DEBUG"):  # line tables + symbols for rocgdb (same code generation)
    FLAGS.append("-g")
# A/B builds: LFM_BUILD_DEFINES="-DX -DY" LFM_BUILD_DIR=<dir under lightfm_amd/> python -m lightfm_amd.build
FLAGS += os.environ.get("LFM_BUILD_DEFINES", "").split()
if os.environ.get("LFM_BUILD_DIR"):
    OUT_DIR = os.path.join(HERE, os.environ["LFM_BUILD_DIR"])
    LIB = os.path.join(OUT_DIR, "liblfm_hip.so")
    OPS_LIB = os.path.join(OUT_DIR, "liblfm_ops.so")


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    os.makedirs(OUT_DIR, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS]
    objs, jobs = {}, []
    for src in SOURCES + OPS_SOURCES + OPS_API:
        s = os.path.join(CSRC, src)
        o = os.path.join(OUT_DIR, src.replace(".hip", ".o"))
        objs[src] = o
        if force or _stale(o, [s] + hdrs):
            jobs.append([HIPCC] + FLAGS + ["-c", s, "-o", o])
    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    with ThreadPoolExecutor(max_workers=len(objs)) as ex:
        list(ex.map(run, jobs))
    mine = [objs[s] for s in SOURCES + OPS_SOURCES]
    if force or _stale(LIB, mine):
        run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", LIB] + mine + ["-ldl"])
    mine = [objs[s] for s in OPS_SOURCES + OPS_API]
    if force or _stale(OPS_LIB, mine):
        # liblfm_ops.so works on torch's memory and streams, so it has to bind to the HIP runtime torch has loaded --
        # which is torch's own copy, known to the loader as "libamdhip64.so" (liblfm_hip.so asks for the system's
        # versioned name).  An empty stand-in of that name gives the library the right dependency.
        stand_in = os.path.join(OUT_DIR, "link", "libamdhip64.so")
        os.makedirs(os.path.dirname(stand_in), exist_ok=True)
        run(["gcc", "-shared", "-fPIC", "-x", "c", os.devnull, "-Wl,-soname,libamdhip64.so", "-o", stand_in])
        run([HIPCC, "--offload-arch=gfx950", "-no-hip-rt", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", OPS_LIB] + mine
            + ["-Wl,--no-as-needed", stand_in])
        os.remove(stand_in)
    binding, src = os.path.join(OUT_DIR, "_torch_ops.so"), os.path.join(CSRC, TORCH_OPS)
    if importlib.util.find_spec("torch") and (force or _stale(binding, [src, OPS_LIB, hdrs[1]])):
        import torch
        if torch.version.hip is None:
            return LIB
        root = os.path.dirname(torch.__file__)
        run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), "-I" + os.path.join(root, "include"),
             "-I" + os.path.join(os.path.dirname(os.path.dirname(HIPCC)), "include"), "-I" + sysconfig.get_paths()["include"],
             src, "-o", binding, "-L" + OUT_DIR, "-l:liblfm_ops.so", "-L" + os.path.join(root, "lib"), "-ltorch_python",
             "-ltorch_cpu", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
