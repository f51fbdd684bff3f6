"""
Build libbgmm_hip.so, libbgmm_ops.so (hipcc, gfx950 only) and the operators' torch binding (g++) in-tree.

The shared objects are git-ignored and go with the tree where it is copied.
``build()`` is idempotent: it recompiles only sources newer than
their objects.
"""
import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbgmm_hip.so")
SOURCES = ["api_context.hip", "api_inputs.hip", "api_perm.hip", "api_sweep.hip", "api_group.hip", "api_comm.hip", "kernels_state.hip", "kernels_score.hip", "kernels_prune.hip", "kernels_choice.hip",
           "kernels_resolve.hip", "kernels_rng.hip", "kernels_seq.hip", "kernels_gram.hip", "kernels_home.hip", "kernels_safe.hip",
           "kernels_perm.hip", "kernels_resid.hip"]
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
# every header next to the sources + the public one: editing any of them rebuilds every object
HEADERS = sorted(h for h in glob.glob(os.path.join(CSRC, "*.h")) if not os.path.basename(h).startswith("ops_")) + [os.path.join(INCLUDE, "bgmm.h")]
# the operators on torch tensors (pybgmm_amd.ops): a library of its own, because it has to bind to the HIP runtime that
# torch brings, while libbgmm_hip.so links the system's (a process may hold both)
OPS_LIB = os.path.join(HERE, "libbgmm_ops.so")
OPS_SOURCES = ["ops_common.hip", "ops_groups.hip", "ops_products.hip", "ops_products_f64.hip", "ops_products_f32.hip",
               "ops_products_f16.hip", "ops_products_bf16.hip", "ops_route.hip", "ops_verify.hip"]
OPS_BINDING = os.path.join(HERE, "ops", "_binding.so")          # what pybgmm_amd.ops imports: libbgmm_ops.so on torch tensors
BOUND_TO = os.path.join(CSRC, "_obj", "binding_torch.txt")      # the torch that the binding was built for
OPS_HEADERS = sorted(glob.glob(os.path.join(CSRC, "ops_*.h"))) + [os.path.join(INCLUDE, "bgmm_ops.h")]
# -ffp-contract=off: the sufficient-statistics updates must round product and sum
# separately (bit-identical m / S to the reference); hot loops call fma() explicitly.
# -fvisibility=hidden: the shared object exports the BGMM_API entry points of include/bgmm.h and nothing else.
# -packed-fp32-ops: no packed single-precision arithmetic (some of its forms have given wrong results on this hardware);
# hipcc's host pass does not know the feature and says so, which is harmless.
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fvisibility=hidden",
         "-Wall", "-Wno-unused-result", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def hipcc():
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found: libbgmm_hip.so cannot be built")
    return exe


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False, extra_flags=()):
    """Both libraries and the binding; returns the path of libbgmm_hip.so."""
    path = build_sampler(force, verbose, extra_flags)
    build_ops(force, verbose, extra_flags)
    return path


def build_sampler(force=False, verbose=False, extra_flags=()):
    """libbgmm_hip.so alone: the samplers need neither g++ nor torch."""
    return _build_one(LIB, SOURCES, HEADERS, [], force, verbose, extra_flags)


def build_ops(force=False, verbose=False, extra_flags=()):
    """libbgmm_ops.so and, where there is a torch with HIP, the binding."""
    # -no-hip-rt: libbgmm_ops.so does not link a HIP runtime (include/bgmm_ops.h says which one it binds to)
    _build_one(OPS_LIB, OPS_SOURCES, OPS_HEADERS, ["-no-hip-rt", "-Wl,-soname," + os.path.basename(OPS_LIB)], force, verbose, extra_flags)
    _build_binding(force, verbose)


def bindable():
    """Whether there is a torch with HIP: without one there are no operators to bind, nor ``pybgmm_amd.ops``."""
    spec = importlib.util.find_spec("torch")
    return spec is not None and bool(spec.origin) and os.path.exists(os.path.join(os.path.dirname(spec.origin), "lib", "libc10_hip.so"))


def _build_binding(force, verbose):
    """Host code against torch's headers and libraries."""
    src = os.path.join(CSRC, "ops_torch.cpp")
    if not bindable() or not (force or _stale(OPS_BINDING, [src, OPS_HEADERS[-1]]) or _bound_to() != _torch_here()):
        return
    import torch
    from torch.utils.cpp_extension import include_paths
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    rocm = os.path.dirname(os.path.dirname(hipcc()))
    includes = include_paths() + [sysconfig.get_paths()["include"], os.path.join(rocm, "include"), "/opt/rocm/include"]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    for p in includes:
        cmd += ["-isystem", p]
    cmd += [src, "-o", OPS_BINDING, "-L" + lib, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip", "-L" + HERE, "-lbgmm_ops",
            "-Wl,-rpath,$ORIGIN/..", "-Wl,--allow-shlib-undefined"]
    _run(cmd, verbose)
    with open(BOUND_TO, "w") as f:
        f.write(_torch_here())


def _torch_here():
    """Which torch a binding built now is for: its C++ interface differs between versions."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:         # (a source tree on the path)
        version = "unknown"
    return "%s %s" % (version, importlib.util.find_spec("torch").origin)


def _bound_to():
    if not os.path.exists(BOUND_TO):
        return None
    with open(BOUND_TO) as f:
        return f.read()


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError("%s failed:\n%s\n%s" % (os.path.basename(cmd[0]), " ".join(cmd), r.stdout))
    return r.stdout


def _build_one(lib, sources, headers, link_flags, force, verbose, extra_flags):
    objdir = os.path.join(CSRC, "_obj")
    os.makedirs(objdir, exist_ok=True)
    cc = hipcc()
    jobs = []
    for src in sources:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src + ".o")
        if force or _stale(o, [s] + headers):
            jobs.append([cc] + FLAGS + list(extra_flags) + ["-c", s, "-o", o])

    if jobs:
        with ThreadPoolExecutor(max_workers=4) as ex:
            outs = list(ex.map(lambda cmd: _run(cmd, verbose), jobs))
        if verbose:
            for o in outs:
                if o.strip():
                    print(o)
    objs = [os.path.join(objdir, s + ".o") for s in sources]
    if force or jobs or _stale(lib, objs):
        _run([cc, "--offload-arch=gfx950", "-shared", "-fPIC"] + link_flags + ["-o", lib] + objs, verbose)
    return lib


if __name__ == "__main__":
    import sys
    print(build(force="--force" in sys.argv, verbose=True))
