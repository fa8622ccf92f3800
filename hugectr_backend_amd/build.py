"""In-tree build of the native libraries (hipcc, gfx950 only).

    python -m hugectr_backend_amd.build [--force] [--jobs N]

Outputs (git-ignored, shipped to the GPU box by gpurun):
    hugectr_backend_amd/lib/libhps_amd.so         engine + C ABI (include/hps_amd.h)
    hugectr_backend_amd/lib/libtriton_hps.so      Triton backend shell: exports only TRITONBACKEND_*
    hugectr_backend_amd/lib/libtriton_mock_core.so  TEST INFRASTRUCTURE: stand-in for tritonserver's core
"""
from __future__ import annotations

import argparse
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata, util
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
ROOT = PKG.parent
# HPS_AMD_LIB_DIR / HPS_AMD_EXTRA_FLAGS: an instrumented variant of the libraries next to the product build
# (tests/test_sanitizers.py builds the shell with -fsanitize=address into a scratch directory this way)
_ALT = os.environ.get("HPS_AMD_LIB_DIR")
LIB = Path(_ALT) if _ALT else PKG / "lib"
OBJ = Path(_ALT) / "obj" if _ALT else PKG / "build"

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
CXXFLAGS = ["-O3", "-std=c++17", "-fPIC", "-Wall", "-Wextra", "-Wno-unused-parameter", "-pthread",
            f"-I{ROOT / 'include'}", f"-I{CSRC}", *os.environ.get("HPS_AMD_EXTRA_FLAGS", "").split()]
# device code only: some packed fp32 instructions that hipcc makes of plain float code have given wrong results on this chip
HIPFLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

ENGINE_SRCS = [
    "common/json.cpp",
    "common/config.cpp",
    "ps/thread_pool.cpp",
    "ps/host_table.cpp",
    "ps/volatile_tier.cpp",
    "ps/update_source.cpp",
    "cache/kernels.hip",
    "cache/shard_kernels.hip",
    "cache/shard_session.cpp",
    "cache/entry_kernels.hip",
    "cache/shard_entry.cpp",
    "cache/direct_kernels.hip",
    "cache/copy_engines.cpp",
    "cache/segcopy_kernels.hip",
    "cache/probe_kernels.hip",
    "cache/qrows_kernels.hip",
    "cache/multi_gpu_probe.cpp",
    "cache/engine.cpp",
    "cache/parameter_server.cpp",
    "dense/dense_kernels.hip",
    "dense/fused_kernels.hip",
    "dense/dense.cpp",
    "dense/linear_kernels.hip",
    "dense/group_rows.hip",
    "dense/linear.cpp",
]
CAPI_SRCS = ["c_api.cpp"]
TRITON_SRCS = [
    "triton/hps.cpp",
    "triton/backend_state.cpp",
    "triton/model_state.cpp",
    "triton/model_instance_state.cpp",
    "triton/timer.cpp",
    "triton/roctx.cpp",
]
MOCK_SRCS = ["mock_triton/mock_core.cpp"]


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(" ".join(map(str, cmd)) + "\n" + r.stdout + r.stderr)
        raise RuntimeError(f"build step failed: {cmd[0]} ... {cmd[-1]}")
    return r


def _flags(src: Path) -> list:
    return HIPFLAGS if src.suffix == ".hip" else []


def _deps_stamp(src: Path) -> str:
    """Hash of the source and every header under csrc/ + include/ (coarse but safe)."""
    h = hashlib.sha1()
    h.update(src.read_bytes())
    for d in (CSRC, ROOT / "include"):
        for p in sorted(d.rglob("*.h")):
            h.update(p.read_bytes())
    h.update(" ".join(CXXFLAGS + _flags(src)).replace(str(ROOT), ".").encode())     # (a tree that was copied elsewhere is as good)
    return h.hexdigest()


def _compile(rel: str, force: bool) -> Path:
    src = CSRC / rel
    obj = OBJ / (rel.replace("/", "__") + ".o")
    stamp = obj.with_suffix(".stamp")
    want = _deps_stamp(src)
    if not force and obj.exists() and stamp.exists() and stamp.read_text() == want:
        return obj
    obj.parent.mkdir(parents=True, exist_ok=True)
    cmd = [HIPCC, f"--offload-arch={ARCH}", *CXXFLAGS, *_flags(src), "-c", str(src), "-o", str(obj)]
    _run(cmd)
    stamp.write_text(want)
    return obj


def _link(out: Path, objs, extra=()):
    out.parent.mkdir(parents=True, exist_ok=True)
    _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(out), *map(str, objs), "-pthread", *extra,
          *os.environ.get("HPS_AMD_EXTRA_LDFLAGS", "").split()])


def _rocm_include() -> Path:
    """The headers that belong to HIPCC."""
    beside = Path(shutil.which(HIPCC) or HIPCC).parent.parent / "include"
    return beside if (beside / "hip").is_dir() else Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "include"


def _torch_home():
    spec = util.find_spec("torch")     # (found, not imported)
    return Path(list(spec.submodule_search_locations)[0]) if spec and spec.submodule_search_locations else None


def torch_module_lacks(home, python_include: Path, rocm_include: Path, cxx: str):
    """What the operators' calls on torch tensors cannot be built without here, or None.  A host that only serves through the plugin has no
    torch, one of another kind or no Python headers; the libraries and the tools need none of it."""
    if home is None:
        return "torch"
    for f in (home / "lib" / "libc10_hip.so", home / "include" / "c10" / "hip" / "HIPStream.h", python_include / "Python.h",
              rocm_include / "hip" / "hip_runtime_api.h"):
        if not f.exists():
            return str(f)
    return None if shutil.which(cxx) else cxx


def _torch_module(src: Path, out: Path, cxx: str):
    """The operators' calls on torch tensors, a CPython module.  Its hps_* entries come from libhps_amd.so, which hps.py loads first."""
    import torch
    home = Path(torch.__file__).resolve().parent
    dirs = [home / "include", home / "include" / "torch" / "csrc" / "api" / "include", _rocm_include(), sysconfig.get_paths()["include"]]
    _run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{ROOT / 'include'}", *(f"-isystem{d}" for d in dirs), str(src),
          "-o", str(out), f"-L{home / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"])


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> dict:
    jobs = jobs or min(8, os.cpu_count() or 1)
    groups = {"engine": ENGINE_SRCS, "capi": CAPI_SRCS}
    if (CSRC / "triton" / "hps.cpp").exists():
        groups["triton"] = TRITON_SRCS
    if (CSRC / "mock_triton" / "mock_core.cpp").exists():
        groups["mock"] = MOCK_SRCS
    all_srcs = sorted({s for g in groups.values() for s in g})
    with ThreadPoolExecutor(jobs) as ex:
        objs = dict(zip(all_srcs, ex.map(lambda s: _compile(s, force), all_srcs)))
    outs = {}

    def newer(out: Path, deps) -> bool:
        return force or not out.exists() or any(o.stat().st_mtime > out.stat().st_mtime for o in deps)

    eng = [objs[s] for s in ENGINE_SRCS]
    out = LIB / "libhps_amd.so"
    deps = eng + [objs[s] for s in CAPI_SRCS]
    if newer(out, deps):
        _link(out, deps)
    outs["hps_amd"] = out
    if "triton" in groups:
        out = LIB / "libtriton_hps.so"
        deps = eng + [objs[s] for s in TRITON_SRCS]
        if newer(out, deps):
            # export only TRITONBACKEND_* like the reference's libtriton_hps.ldscript
            _link(out, deps, [f"-Wl,--version-script={CSRC / 'triton' / 'libtriton_hps.ldscript'}"])
        outs["triton_hps"] = out
    if "mock" in groups:
        out = LIB / "libtriton_mock_core.so"
        deps = [objs[s] for s in MOCK_SRCS]
        if newer(out, deps):
            _link(out, deps, ["-ldl"])
        outs["mock_core"] = out
    # native tools next to the libraries (binaries are git-ignored like the libraries; they travel with gpurun)
    tool_src = ROOT / "tools" / "triton_abi_bench.cpp"
    if tool_src.exists() and "mock" in groups:
        out = LIB / "triton_abi_bench.bin"
        if force or not out.exists() or out.stat().st_mtime < max(tool_src.stat().st_mtime,
                                                                   (CSRC / "mock_triton" / "mock_core.h").stat().st_mtime,
                                                                   (CSRC / "common" / "hps_hash.h").stat().st_mtime):
            _run([HIPCC, f"--offload-arch={ARCH}", "-O2", "-std=c++17", "-Wall", "-Wno-unused-result", str(tool_src), "-o", str(out),
                  "-ldl", "-pthread"])
        outs["triton_abi_bench"] = out
    cxx = os.environ.get("CXX", "g++")
    lacks = torch_module_lacks(_torch_home(), Path(sysconfig.get_paths()["include"]), _rocm_include(), cxx)
    if lacks:                                       # (the Python classes of the operators say that they need the module)
        print(f"hps_torch_calls.so left out: no {lacks}", file=sys.stderr)
    else:
        out = LIB / "hps_torch_calls.so"
        src = CSRC / "python" / "torch_calls.cpp"
        stamp = OBJ / "python__torch_calls.stamp"
        want = f"{_deps_stamp(src)} torch {metadata.version('torch')}"      # another torch: another module
        if force or not out.exists() or not stamp.exists() or stamp.read_text() != want:
            _torch_module(src, out, cxx)
            stamp.write_text(want)
        outs["torch_calls"] = out
    if verbose:
        for k, v in outs.items():
            print(f"{k}: {v}")
    return outs


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    a = ap.parse_args()
    build(force=a.force, jobs=a.jobs, verbose=True)
