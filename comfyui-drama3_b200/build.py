"""Build the sm_100a shared library in place: drama3_b200/libdrama3_b200.so.

    python comfyui-drama3_b200/build.py [--force]

nvcc cross-compiles for sm_100a on a machine without a GPU. The translation units compile side by side, each into an
object under _build/ that is rebuilt when a file it was compiled from is newer; the library is linked from them.
"""
import argparse
import concurrent.futures
import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
SOURCES = [HERE / "csrc" / "drama3_b200.cu", HERE / "csrc" / "lines.cu", HERE / "csrc" / "pack.cpp"]
DEPENDS = sorted((HERE / "csrc").glob("*.c*")) + [ROOT / "include" / "drama3_b200.h"]
OUTPUT = HERE / "drama3_b200" / "libdrama3_b200.so"
OBJECTS = HERE / "_build"
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xptxas", "-warn-spills", "-diag-suppress", "177,128"]


def nvcc():
    for candidate in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if candidate and (os.path.sep not in candidate or Path(candidate).exists()):
            return candidate
    raise RuntimeError("nvcc not found")


def stale():
    if not OUTPUT.exists():
        return True
    built = OUTPUT.stat().st_mtime
    return any(p.stat().st_mtime > built for p in DEPENDS)


def compiled_from(depfile):
    """The files of this repository that a make-style dependency file names, or None without one."""
    if not depfile.exists():
        return None
    names = depfile.read_text().replace("\\\n", " ").split(":", 1)[1].split()
    return [p for p in map(Path, names) if ROOT in p.resolve().parents]


def compile_unit(source, force, verbose):
    """The object of one translation unit, compiled if it is missing or older than a file it was compiled from."""
    obj = OBJECTS / (source.name + ".o")
    dep = obj.with_suffix(".d")
    made = obj.stat().st_mtime if obj.exists() else 0.0
    files = compiled_from(dep)
    if not force and files and all(p.exists() and p.stat().st_mtime <= made for p in files):
        return obj
    tmp = obj.with_suffix(".o.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-MD", "-MF", str(dep), "-c", "-o", str(tmp), str(source)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=HERE)
    os.replace(tmp, obj)
    return obj


def build(force=False, verbose=False):
    """Compile the library if it is missing or older than its sources; returns its path."""
    if not force and not stale():
        return OUTPUT
    OBJECTS.mkdir(exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(lambda source: compile_unit(source, force, verbose), SOURCES))
    tmp = OUTPUT.with_suffix(".so.tmp")
    subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", str(tmp), *map(str, objects)], check=True, cwd=HERE)
    os.replace(tmp, OUTPUT)
    return OUTPUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=True))
    sys.exit(0)
