"""Build libggmlc_b200.so in-tree (ggmlc_b200/libggmlc_b200.so) with nvcc for sm_100a.

    python -m ggmlc_b200.build [--force]

Objects go to ggmlc_b200/_build/; a source is recompiled when it or any header in csrc/ is
newer than its object.  The shared library links the CUDA runtime statically so it loads in
any process of this image (with or without torch).  Where torch is installed, the binding of the
4-bit KV cache operators (_kv_q4.so) is built against it as well.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libggmlc_b200.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found (CUDA 12.9 toolkit required to build ggmlc_b200)")
    return cand


def _flags(src: Path) -> list[str]:
    common = ["-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-lineinfo", "-I", str(CSRC),
              "-I", str(PKG.parent / "include")]
    if src.suffix == ".cu":
        return common + ARCH + ["--expt-relaxed-constexpr", "-Xptxas", "-O3"]
    return common + ARCH


def _compile(src: Path) -> Path:
    obj = BUILD / (src.name + ".o")
    cmd = [nvcc(), "-c", str(src), "-o", str(obj)] + _flags(src)
    if src.suffix != ".cu":
        cmd += ["-x", "cu"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted([p for p in CSRC.iterdir() if p.suffix in (".cu", ".cpp")])
    headers = [p for p in CSRC.iterdir() if p.suffix in (".h", ".cuh")]
    headers.append(PKG.parent / "include" / "ggmlc_b200.h")
    newest_header = max(h.stat().st_mtime for h in headers)
    todo = []
    for s in sources:
        obj = BUILD / (s.name + ".o")
        if force or not obj.exists() or obj.stat().st_mtime < max(s.stat().st_mtime, newest_header):
            todo.append(s)
    if todo:
        with cf.ThreadPoolExecutor(max_workers=min(len(todo), os.cpu_count() or 4)) as ex:
            for obj in ex.map(_compile, todo):
                if verbose:
                    print("compiled", obj.name)
    objs = [BUILD / (s.name + ".o") for s in sources]
    if force or todo or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), "-shared", "-o", str(tmp)] + [str(o) for o in objs] + ARCH + [
            "-Xlinker", "--no-undefined", "-lcuda", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    build_bench_tool(force)
    build_torch_binding(force)
    return LIB


TOOL_SRC = PKG / "tools" / "ggmlc_bench.cpp"
TOOL = PKG / "ggmlc-bench"


def build_bench_tool(force: bool = False) -> Path:
    """ggmlc_b200/ggmlc-bench: the reference's benchmark CLI over the C ABI (host C++ only)."""
    if not force and TOOL.exists() and TOOL.stat().st_mtime >= max(
            TOOL_SRC.stat().st_mtime, LIB.stat().st_mtime):
        return TOOL
    cxx = shutil.which("g++") or "g++"
    cmd = [cxx, "-O2", "-std=c++17", "-o", str(TOOL), str(TOOL_SRC), "-I",
           str(PKG.parent / "include"), "-L", str(PKG), "-lggmlc_b200", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"ggmlc-bench build failed:\n{r.stdout}\n{r.stderr}")
    return TOOL


BINDING_SRC = PKG / "bindings" / "kv_q4.cpp"
BINDING = PKG / "_kv_q4.so"
BINDING_FOR = BUILD / "_kv_q4.for"  # what it was built against


def torch_build() -> str | None:
    """What the torch binding is compiled against (interpreter, torch and its ABI), None where torch
    with its C++ headers and CUDA is not installed.  Found without importing torch, which takes seconds."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    root = Path(list(spec.submodule_search_locations)[0])
    needs = ("include/torch/csrc/utils/pybind.h", "lib/libc10_cuda.so", "lib/libtorch_python.so")
    if not all((root / f).exists() for f in needs):
        return None
    version = root / "version.py"
    tag = version.read_text() if version.exists() else ""
    return "\n".join([sys.version, str(root), tag])


def build_torch_binding(force: bool = False) -> Path | None:
    """ggmlc_b200/_kv_q4.so: the torch binding of the 4-bit KV cache operators (host C++ against
    torch's headers and the library above), built anew when the source, the header, torch or the
    interpreter changes.  None where there is no torch to build it against: only ggmlc_b200.kv_q4
    needs it, the engine does not."""
    against = torch_build()
    if against is None:
        return None
    header = PKG.parent / "include" / "ggmlc_b200.h"
    if not force and BINDING.exists() and BINDING.stat().st_mtime >= max(
            BINDING_SRC.stat().st_mtime, header.stat().st_mtime) and (
            BINDING_FOR.exists() and BINDING_FOR.read_text() == against):
        return BINDING
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cxx = shutil.which("g++") or "g++"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-o", str(tmp), str(BINDING_SRC),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-DTORCH_EXTENSION_NAME=_kv_q4", "-I", str(PKG.parent / "include"),
           "-I", sysconfig.get_paths()["include"],
           "-I", str(Path(nvcc()).resolve().parents[1] / "include")]
    for p in include_paths():
        cmd += ["-isystem", p]
    cmd += ["-L", str(PKG), "-lggmlc_b200", "-Wl,-rpath,$ORIGIN"]
    for p in library_paths():
        cmd += ["-L", p]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"torch binding build failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)
    BUILD.mkdir(exist_ok=True)
    BINDING_FOR.write_text(against)
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
