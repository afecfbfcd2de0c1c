"""Builds ppo_amd/libppo_hip.so (gfx950) from csrc/*.hip with hipcc.  In-tree, no JIT cache.

Two libraries come out of one set of objects:
  libppo_hip.so      the product
  libppo_hip_sym.so  the same plus the symmetric-wave form of the fused update kernel (update_sym.hip,
                     never the default on any shape; selected with PPO_HIP_LIB=... PPO_FWDBWD=sym).  Kept
                     under test as the alternative form, kept out of the product binary.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libppo_hip.so")
LIB_SYM = os.path.join(HERE, "libppo_hip_sym.so")
FASTCALL = os.path.join(HERE, "_fastcall.so")          # CPython extension (csrc/fastcall.c), plain C
TOKEN_OPS = os.path.join(HERE, "_token_ops.so")        # torch extension (csrc/token_torch.cpp), host C++
SOURCES = ["scan.hip", "act.hip", "act_one.hip", "update.hip", "update_vjp.hip", "env.hip", "rollout.hip", "token.hip"]
SYM_SOURCES = ["update_sym.hip"]             # + update.hip compiled with -DPPO_WITH_SYM
HEADERS = ["ppo_common.h", "update_common.h", os.path.join("..", "..", "include", "ppo_hip.h")]
FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC",
         "-fhip-fp32-correctly-rounded-divide-sqrt"]
# token.hip: no packed fp32 instructions (some of their forms have been seen to give wrong results on this GPU)
SOURCE_FLAGS = {"token.hip": ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]}


def _stale(lib, sources):
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    deps = [os.path.join(CSRC, s) for s in sources + HEADERS] + [os.path.abspath(__file__)]   # (update_vjp.hip includes update.hip)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(jobs, verbose):
    """jobs: (source, object, extra flags); all at once (six or seven files)."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    procs = []
    for src, obj, extra in jobs:
        cmd = [hipcc] + FLAGS + SOURCE_FLAGS.get(src, []) + list(extra) + ["-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((subprocess.Popen(cmd), cmd))
    for p, cmd in procs:
        if p.wait() != 0:
            raise RuntimeError("hipcc failed: " + " ".join(cmd))


def _link(objs, lib, verbose):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC"] + objs + ["-o", lib]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def build_fastcall(force=False, verbose=True):
    """The ctypes-free per-step binding (csrc/fastcall.c): a CPython extension compiled with the host C
    compiler against this interpreter's headers; it links against nothing else."""
    import sysconfig
    src = os.path.join(CSRC, "fastcall.c")
    if not force and os.path.exists(FASTCALL) and os.path.getmtime(FASTCALL) >= os.path.getmtime(src):
        return FASTCALL
    cmd = [os.environ.get("CC", "gcc"), "-O2", "-shared", "-fPIC", "-Wall", "-I" + sysconfig.get_paths()["include"],
           src, "-o", FASTCALL]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return FASTCALL


def build_token_ops(force=False, verbose=True):
    """The binding of ppo_amd.tokens (csrc/token_torch.cpp): host C++ against torch's headers and libraries.  It calls
    libppo_hip.so by address and is not linked against it."""
    import sysconfig
    import torch
    src = os.path.join(CSRC, "token_torch.cpp")
    deps = [src, os.path.join(HERE, "..", "include", "ppo_hip.h"), os.path.abspath(__file__)]
    if not force and os.path.exists(TOKEN_OPS) and all(os.path.getmtime(TOKEN_OPS) >= os.path.getmtime(d) for d in deps):
        return TOKEN_OPS
    at = os.path.dirname(torch.__file__)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for inc in (os.path.join(at, "include"), os.path.join(at, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], "/opt/rocm/include"):
        cmd += ["-isystem", inc]
    cmd += [src, "-o", TOKEN_OPS, "-L" + os.path.join(at, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch",
            "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return TOKEN_OPS


def build(force=False, verbose=True, variant=None, extra_flags=()):
    """Compile every HIP source for gfx950 and link the C-ABI shared libraries.  Returns the product
    library's path; build.last_action says what happened ("compiled" or "up to date").
    variant / extra_flags: diagnostic builds (e.g. -DPPO_TANH_ACCURATE) go to
    libppo_hip_<variant>.so (with the symmetric kernel inside), selected at run time with the
    PPO_HIP_LIB environment variable."""
    if variant is not None:
        objdir = os.path.join(HERE, f"build_{variant}")
        os.makedirs(objdir, exist_ok=True)
        srcs = SOURCES + SYM_SOURCES
        obj = lambda s: os.path.join(objdir, s.replace(".hip", ".o"))
        _compile([(s, obj(s), list(extra_flags) + ["-DPPO_WITH_SYM"]) for s in srcs], verbose)
        lib = os.path.join(HERE, f"libppo_hip_{variant}.so")
        _link([obj(s) for s in srcs], lib, verbose)
        return lib
    build_fastcall(force, verbose)
    build_token_ops(force, verbose)
    if not force and not _stale(LIB, SOURCES) and not _stale(LIB_SYM, SOURCES + SYM_SOURCES):
        build.last_action = "up to date"
        return LIB
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    obj = lambda s: os.path.join(objdir, s.replace(".hip", ".o"))
    upd_sym = os.path.join(objdir, "update_withsym.o")
    _compile([(s, obj(s), []) for s in SOURCES] + [(s, obj(s), []) for s in SYM_SOURCES] +
             [("update.hip", upd_sym, ["-DPPO_WITH_SYM"])], verbose)
    _link([obj(s) for s in SOURCES], LIB, verbose)
    _link([obj(s) for s in SOURCES if s != "update.hip"] + [upd_sym] + [obj(s) for s in SYM_SOURCES],
          LIB_SYM, verbose)
    build.last_action = "compiled"
    return LIB


build.last_action = None


if __name__ == "__main__":
    # python -m ppo_amd.build [--force] [--variant NAME -DFLAG ...]
    args = sys.argv[1:]
    if "--variant" in args:
        i = args.index("--variant")
        build(variant=args[i + 1], extra_flags=[a for a in args[i + 2:] if a.startswith("-")])
    else:
        build(force="--force" in args)
        print("libppo_hip:", build.last_action)
