"""Build libfgw_mha.so in-tree with nvcc for sm_100a, and the Python binding of the serving-step operators.

Each ``csrc/*.cu`` compiles to an object under ``_build/`` in parallel; the objects link into
``fgw_b200/_lib/libfgw_mha.so`` with the CUDA runtime linked statically, so the library only
needs the NVIDIA driver at run time. ``csrc/fgw_torch.cpp`` becomes ``fgw_b200/_lib/fgw_torch.so`` beside it (a
Python extension on torch's headers that calls the library; left out where torch is not installed). Re-running is incremental (objects newer than their
sources and headers are kept).

    python -m fgw_b200.build [--force] [--jobs N]
"""
import argparse
import concurrent.futures
import importlib.metadata
import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

PACKAGE = pathlib.Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIB_DIR = PACKAGE / "_lib"
LIB = LIB_DIR / "libfgw_mha.so"
BINDING = LIB_DIR / "fgw_torch.so"
BINDING_SOURCE = CSRC / "fgw_torch.cpp"
BINDING_STAMP = BUILD / "fgw_torch.built_for"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# Host code keeps separate multiplies and adds (no fused multiply-add contraction): the host split choice
# (fgw_split_choice.cu) must round like its Python restatement to make the same picks.
CFLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
          "--expt-relaxed-constexpr", "-DNDEBUG", "-Xcompiler", "-ffp-contract=off", f"-I{INCLUDE}", f"-I{CSRC}"]


def nvcc():
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(found):
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build libfgw_mha.so")
    return found


def _stale(obj, src, headers):
    if not obj.exists():
        return True
    stamp = obj.stat().st_mtime
    return any(p.stat().st_mtime > stamp for p in [src, *headers])


def _compile(src, obj, extra):
    cmd = [nvcc(), *ARCH, *CFLAGS, *extra, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return proc.stderr


def _version(package):
    """Version and place of an installed package, without importing it; None if there is none."""
    spec = importlib.util.find_spec(package)
    return None if spec is None else f"{importlib.metadata.version(package)} {spec.origin}"


def binding_command(target, include=INCLUDE):
    """The compiler call that makes the Python binding for the torch of this interpreter."""
    import torch
    from torch.utils import cpp_extension

    includes = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"], str(include)]
    libraries = cpp_extension.library_paths("cuda")
    return ["g++", "-shared", "-fPIC", "-O2", "-std=c++17", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=fgw_torch",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[flag for path in includes for flag in ("-isystem", path)], str(BINDING_SOURCE), "-o", str(target),
            f"-L{LIB_DIR}", *[f"-L{path}" for path in libraries], "-lfgw_mha", "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]


def _build_binding():
    tmp = BINDING.with_suffix(".so.tmp")
    proc = subprocess.run(binding_command(tmp), capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SOURCE.name}:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, BINDING)


def build(force=False, jobs=None, verbose_ptxas=False):
    """Compile every kernel translation unit, link the shared library and build the binding; returns the library's path."""
    BUILD.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))
    extra = ["-Xptxas", "-v"] if verbose_ptxas else []
    objects = [BUILD / (s.stem + ".o") for s in sources]
    todo = [(s, o) for s, o in zip(sources, objects) if force or verbose_ptxas or _stale(o, s, headers)]
    logs = {}
    if todo:
        workers = jobs or min(len(todo), os.cpu_count() or 4)
        with concurrent.futures.ThreadPoolExecutor(workers) as pool:
            futures = {pool.submit(_compile, s, o, extra): s for s, o in todo}
            for fut in concurrent.futures.as_completed(futures):
                logs[futures[fut].name] = fut.result()
    if todo or not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objects):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objects)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
        os.replace(tmp, LIB)
    # the binding is compiled against the interpreter's and torch's headers, which are not among its sources
    built_for = f"torch {_version('torch')}\npython {sys.version}\n"
    if _version("torch") is None:
        print("the binding of the serving-step operators is left out: built without torch")
    elif (force or _stale(BINDING, BINDING_SOURCE, sorted(INCLUDE.glob("*.h")))
          or not BINDING_STAMP.exists() or BINDING_STAMP.read_text() != built_for):
        _build_binding()
        BINDING_STAMP.write_text(built_for)
    if verbose_ptxas:
        for name, text in sorted(logs.items()):
            print(f"== {name}\n{text}")
    return LIB


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--jobs", type=int, default=None)
    parser.add_argument("--ptxas", action="store_true", help="print -Xptxas -v register/smem usage")
    args = parser.parse_args(argv)
    path = build(force=args.force, jobs=args.jobs, verbose_ptxas=args.ptxas)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main())
