"""Build libqattn.so (gfx950) in-tree with hipcc.

    python -m qattention_amd.build

The library is a plain C-ABI shared object: it links only the HIP runtime.
When loaded into a process that has already imported torch, the dynamic
linker resolves libamdhip64.so.7 to torch's copy, so torch's streams and
allocations are valid handles for it.

_calls.so, a CPython module of the host compiler, takes the serving calls from
torch tensors to that C ABI; it links torch's libraries, which the process has
loaded by then.  It shortens the way to the library and is no part of it: without
a host compiler or the headers it is left out, and the calls go through Python.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libqattn.so")
OBJ_DIR = os.path.join(PKG_DIR, "_build")
SOURCES = ["tree_attn.hip", "subtree_stream.hip", "prefix_attn.hip", "paged_attn.hip", "prompt_attn.hip",
           "kv_pages.hip", "quant_pages.hip", "quant_attn.hip"]
HEADERS = ["qattn_common.h", "qattn_device.h", "kv_tiles.h", "dense_tiles.h", "paged_work.h", "quant_format.h", "tree_walk.h"]
CALLS_SOURCE = "calls.cpp"
CALLS_PATH = os.path.join(PKG_DIR, "_calls.so")
ARCH = os.environ.get("QATTN_ARCH", "gfx950")


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (expected /opt/rocm/bin/hipcc)")


def compile_flags() -> list:
    return [
        f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
        # packed fp32 VALU ops stay off (correctness issue on this platform)
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        # one-lane counter atomics stay single instructions: the atomic
        # optimizer would turn each into a wave reduction that waits for the
        # answer at once, where the subtree kernel overlaps it with its loads
        "-Xarch_device", "-mllvm=-amdgpu-atomic-optimizer-strategy=None",
        "-Wall", "-Wno-unused-function",
        # inline assembly must not clobber registers the compiler reserves
        # (M0, EXEC, VCC): such an asm statement is undefined behaviour
        "-Werror=inline-asm",
    ]


def _run(cmd, verbose):
    if verbose:
        print("[qattention_amd.build]", " ".join(cmd), flush=True)
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)


def _finish(proc, verbose):
    _, stderr = proc.communicate()
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in stderr.splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"{os.path.basename(proc.args[0])} failed ({proc.returncode}):\n{err}")
    if verbose and err.strip():
        print(err, file=sys.stderr)


def calls_command(out: str) -> list:
    """The host compiler's command for _calls.so."""
    import torch
    from torch.utils import cpp_extension

    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]
    return [
        os.environ.get("CXX") or shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
        "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(f"-I{d}" for d in include), "-o", out, os.path.join(CSRC, CALLS_SOURCE),
        "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python",
    ]


def _start_calls(out: str, verbose: bool):
    """The compiler of the call module at work, or what kept it from starting."""
    try:
        return _run(calls_command(out), verbose)
    except (ImportError, OSError) as e:
        return e


def _finish_calls(proc, out: str, verbose: bool) -> None:
    """Puts the call module in its place; one that cannot be built is left out, and
    so is an older one, which may not fit the library."""
    try:
        if isinstance(proc, Exception):
            raise proc
        _finish(proc, verbose)
        os.replace(out, CALLS_PATH)
    except (ImportError, OSError, RuntimeError) as e:
        if os.path.exists(CALLS_PATH):
            os.remove(CALLS_PATH)
        print(f"[qattention_amd.build] no {os.path.basename(CALLS_PATH)}, serving calls go through Python: {e}",
              file=sys.stderr, flush=True)


def build(verbose: bool = True) -> str:
    """Compile every HIP source into qattention_amd/libqattn.so and the call
    module into qattention_amd/_calls.so (always rebuilds).

    Each source is compiled to an object in its own hipcc process (they run
    in parallel), then the objects are linked into the shared library."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs, procs = [], []
    for s in SOURCES:
        obj = os.path.join(OBJ_DIR, os.path.splitext(s)[0] + ".o")
        objs.append(obj)
        procs.append(_run([_hipcc(), *compile_flags(), "-c", "-o", obj, os.path.join(CSRC, s)], verbose))
    calls_tmp = CALLS_PATH + ".tmp"
    calls = _start_calls(calls_tmp, verbose)
    for proc in procs:
        _finish(proc, verbose)
    tmp = LIB_PATH + ".tmp"
    _finish(_run([_hipcc(), f"--offload-arch={ARCH}", "-shared", "-o", tmp, *objs], verbose), verbose)
    os.replace(tmp, LIB_PATH)
    _finish_calls(calls, calls_tmp, verbose)
    return LIB_PATH


def is_stale() -> bool:
    if not os.path.exists(LIB_PATH) or not os.path.exists(CALLS_PATH):
        return True
    t = min(os.path.getmtime(LIB_PATH), os.path.getmtime(CALLS_PATH))
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS + [CALLS_SOURCE]]
    deps.append(os.path.join(PKG_DIR, "..", "include", "qattn.h"))
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


if __name__ == "__main__":
    print(build())
