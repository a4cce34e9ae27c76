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
