"""CPU test: an object file is used again only if it came from the same command and nothing that it includes has changed."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def build():
    spec = importlib.util.spec_from_file_location("qz_build", os.path.join(ROOT, "saient-quartz_b200", "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_objects_are_used_again_only_as_they_are(build, tmp_path):
    (tmp_path / "b.cuh").write_text("int b;\n")
    (tmp_path / "a.cuh").write_text('#include "b.cuh"\n')
    (tmp_path / "a.cu").write_text('#include "a.cuh"\n#include <stdio.h>\n')
    src, obj, cmd = str(tmp_path / "a.cu"), str(tmp_path / "a.o"), ["nvcc", "-O3"]
    assert not build.object_current(src, obj, cmd)
    (tmp_path / "a.o").write_text("")
    now = os.path.getmtime(obj) + 1000
    os.utime(obj, (now, now))
    assert not build.object_current(src, obj, cmd)            # nobody knows how it was made
    (tmp_path / "a.o.cmd").write_text("nvcc -O3")
    assert build.object_current(src, obj, cmd)
    assert not build.object_current(src, obj, cmd + ["-DX"])
    os.utime(str(tmp_path / "b.cuh"), (now + 1, now + 1))     # a header of a header
    assert not build.object_current(src, obj, cmd)


class Compiler:
    """Stands in for the compiler and the linker: writes what it was asked for, `made` names the objects compiled."""
    def __init__(self, fail=()):
        self.made, self.fail = [], fail

    def Popen(self, cmd):
        src, obj = cmd[-1], cmd[-2]
        assert not os.path.exists(obj + ".cmd")       # nothing claims to know how an object was made while it is made
        self.made.append(os.path.basename(obj))
        with open(obj, "w") as f:
            f.write("object")
        bad = os.path.basename(src) in self.fail

        class Done:
            def wait(self):
                return 1 if bad else 0
        return Done()

    def check_call(self, cmd):
        out = cmd[cmd.index("-o") + 1] if "-o" in cmd else cmd[2]
        with open(out, "w") as f:
            f.write("library")


@pytest.fixture()
def tree(build, tmp_path, monkeypatch):
    (tmp_path / "pkg" / "csrc").mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "quartz_b200.h").write_text("")
    for n in ("a.cu", "b.cu"):
        (tmp_path / "pkg" / "csrc" / n).write_text("int x;\n")
    pkg = tmp_path / "pkg"
    for name, path in (("HERE", pkg), ("CSRC", pkg / "csrc"), ("LIB", pkg / "libquartz_b200.so"), ("ARCHIVE", pkg / "libkernels.a")):
        monkeypatch.setattr(build, name, str(path))
    monkeypatch.setattr(build, "build_host", lambda force=False: None)
    for name in ("QUARTZ_NVCC_FLAGS", "QUARTZ_CUDA_ARCH", "CUDA_HOME"):
        monkeypatch.delenv(name, raising=False)

    def run(fail=(), **kw):
        c = Compiler(fail)
        monkeypatch.setattr(build.subprocess, "Popen", c.Popen)
        monkeypatch.setattr(build.subprocess, "check_call", c.check_call)
        build.build(**kw)
        return sorted(c.made)
    return run


def test_another_command_builds_again(build, tree, monkeypatch):
    assert tree() == ["a.o", "b.o"]
    assert tree() == []
    for name, value in (("QUARTZ_NVCC_FLAGS", "-DX=1"), ("QUARTZ_CUDA_ARCH", "sm_103a"), ("CUDA_HOME", "/opt/other")):
        monkeypatch.setenv(name, value)
        assert tree() == ["a.o", "b.o"], name
        assert tree() == []
    for name in ("QUARTZ_NVCC_FLAGS", "QUARTZ_CUDA_ARCH", "CUDA_HOME"):
        monkeypatch.delenv(name)
    assert tree() == ["a.o", "b.o"]                  # and back
    now = os.path.getmtime(build.LIB) + 100
    os.utime(os.path.join(build.CSRC, "a.cu"), (now, now))
    made = tree()
    assert "a.o" in made
    assert tree(force=True) == ["a.o", "b.o"]


def test_a_build_that_failed_is_not_taken_for_one_that_did_not(build, tree, monkeypatch):
    assert tree() == ["a.o", "b.o"]
    monkeypatch.setenv("QUARTZ_NVCC_FLAGS", "-DX=1")
    with pytest.raises(RuntimeError):
        tree(fail=("b.cu",))
    monkeypatch.delenv("QUARTZ_NVCC_FLAGS")          # b.o is the other command's, whatever was recorded before
    assert tree() == ["a.o", "b.o"]
    assert tree() == []
