"""Build in-tree, from one compilation of the csrc/*.cu files (in parallel) for sm_100a:
  saient-quartz_b200/libquartz_b200.so  the CUDA library (what the tests and the benchmark load)
  saient-quartz_b200/libkernels.a       the same objects as a static archive under the name the reference's
                                        build.rs links (`static=kernels` + `cudart`, build.rs:52-72)
and saient-quartz_b200/libquartz_host.so (the C++ host side of the decode step, a pure client of the C ABI)."""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libquartz_b200.so")
ARCHIVE = os.path.join(HERE, "libkernels.a")
HOST_LIB = os.path.join(HERE, "libquartz_host.so")
HOST_SRC = os.path.join(HERE, "host", "forward_state.cpp")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def compiler():
    return os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")


def compile_command():
    arch = os.environ.get("QUARTZ_CUDA_ARCH", "sm_100a")   # same variable as the reference's build.rs:33
    cc = arch.replace("sm_", "compute_")
    cmd = [compiler(), "-O3", "-std=c++17", "-gencode", f"arch={cc},code={arch}", "-lineinfo", "-Xcompiler", "-fPIC", "-c"]
    return cmd + os.environ.get("QUARTZ_NVCC_FLAGS", "").split()   # extra compiler flags (e.g. -DNAME=value)


def made_by(path, cmd):
    """Was `path` made by this command?  (Recorded beside it once it was finished.)"""
    return os.path.exists(path) and os.path.exists(path + ".cmd") and open(path + ".cmd").read() == " ".join(cmd)


def forget(path):
    if os.path.exists(path + ".cmd"):
        os.remove(path + ".cmd")


def record(path, cmd):
    with open(path + ".cmd", "w") as f:
        f.write(" ".join(cmd))


def up_to_date(cmd):
    """The library and the archive are newer than all they are made from, this file too, and come from the same command."""
    if not made_by(LIB, cmd) or not os.path.exists(ARCHIVE):
        return False
    t = os.path.getmtime(LIB)
    hdr = os.path.join(HERE, "..", "include", "quartz_b200.h")
    return all(os.path.getmtime(s) <= t for s in sources() + [hdr, os.path.abspath(__file__)])


def included(src, seen=None):
    """`src` and every file of this tree that it includes, directly or not."""
    seen = set() if seen is None else seen
    if src not in seen:
        seen.add(src)
        for name in re.findall(r'^#include "([^"]+)"', open(src).read(), re.M):
            path = os.path.normpath(os.path.join(os.path.dirname(src), name))
            if os.path.exists(path):
                included(path, seen)
    return seen


def object_current(src, obj, cmd):
    """The object is newer than its source, all that it includes and this file, and was made by the same command."""
    if not os.path.exists(obj) or any(os.path.getmtime(f) > os.path.getmtime(obj) for f in included(src) | {os.path.abspath(__file__)}):
        return False
    return made_by(obj, cmd)


def build_host(force=False):
    hdrs = [os.path.join(HERE, "host", "forward_state.h"), os.path.join(HERE, "host", "gguf_loader.h"),
            os.path.join(HERE, "..", "include", "quartz_b200.h")]
    srcs = [HOST_SRC, os.path.join(HERE, "host", "gguf_loader.cpp"), os.path.join(HERE, "host", "model_loader.cpp")]
    if (not force and os.path.exists(HOST_LIB)
            and all(os.path.getmtime(p) <= os.path.getmtime(HOST_LIB) for p in srcs + [LIB] + hdrs)):
        return HOST_LIB
    tmp = HOST_LIB + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", tmp] + srcs + ["-L" + HERE, "-lquartz_b200",
           "-Wl,-rpath,$ORIGIN"]
    subprocess.check_call(cmd)
    os.replace(tmp, HOST_LIB)   # a reader never sees a half-written library
    return HOST_LIB


def build(force=False, verbose=False):
    cmd = compile_command()
    if not force and up_to_date(cmd):
        build_host()
        return LIB
    forget(LIB)
    show = ["-Xptxas", "-v"] if verbose else []
    objs, running = [], []
    for src in (s for s in sources() if s.endswith(".cu")):
        obj = os.path.join(HERE, os.path.splitext(os.path.basename(src))[0] + ".o")
        objs.append(obj)
        if not force and object_current(src, obj, cmd):
            continue
        forget(obj)
        running.append((src, obj, subprocess.Popen(cmd + show + ["-o", obj, src])))
    failed = []
    for src, obj, p in running:
        if p.wait() != 0:
            failed.append(src)
        else:
            record(obj, cmd)
    if failed:
        raise RuntimeError("nvcc failed on " + ", ".join(failed))
    tmp = LIB + ".tmp"
    subprocess.check_call(cmd[:1] + cmd[3:5] + ["-shared", "-o", tmp] + objs)
    os.replace(tmp, LIB)   # a reader never sees a half-written library
    tmp = ARCHIVE + ".tmp"
    if os.path.exists(tmp):
        os.remove(tmp)
    subprocess.check_call(["ar", "rcs", tmp] + objs)
    os.replace(tmp, ARCHIVE)
    record(LIB, cmd)
    build_host(force=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
