"""The incremental build of the CUDA library, with a stand-in for the compiler."""
import importlib.util
import os
import stat

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = """#!/bin/sh
# writes the files that it is asked for; one line per call
out=; dep=; src=
echo "$@" >> "$CUDA_HOME/calls"
while [ $# -gt 0 ]; do
  case "$1" in
    -o) out=$2; shift;;
    -MF) dep=$2; shift;;
    -c) src=$2; shift;;
  esac
  shift
done
[ -n "$dep" ] && echo "$out: $src" > "$dep"
echo built > "$out"
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(ROOT, "mps-deform-conv_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    nvcc = tmp_path / "cuda" / "bin" / "nvcc"
    nvcc.parent.mkdir(parents=True)
    nvcc.write_text(FAKE)
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("CUDA_HOME", str(tmp_path / "cuda"))
    for name in ("CSRC", "INCLUDE", "LIBDIR", "BUILD"):
        monkeypatch.setattr(b, name, str(tmp_path / name.lower()))
        os.makedirs(getattr(b, name), exist_ok=True)
    monkeypatch.setattr(b, "LIB", str(tmp_path / "libdir" / "lib.so"))
    for name in ("a.cu", "b.cu", "c.cu"):
        (tmp_path / "csrc" / name).write_text("")

    def compiled():
        """Files compiled since the last time it was asked."""
        calls = tmp_path / "cuda" / "calls"
        lines = calls.read_text().splitlines() if calls.exists() else []
        calls.write_text("")
        return sorted(os.path.basename(w) for l in lines for k, w in enumerate(l.split()) if k and l.split()[k - 1] == "-c")

    b.compiled = compiled
    b.age = lambda name, seconds: os.utime(tmp_path / "csrc" / name, (os.path.getmtime(b.LIB) + seconds,) * 2)
    return b


def test_only_what_changed_is_compiled(build):
    build.build_lib()
    assert build.compiled() == ["a.cu", "b.cu", "c.cu"]
    build.age("b.cu", 10)
    build.build_lib()
    assert build.compiled() == ["b.cu"]


def test_objects_of_other_flags_are_not_linked(build):
    """One edit after a change of flags compiles every file with the new ones."""
    build.build_lib()
    build.compiled()
    build.NVCC_FLAGS = [*build.NVCC_FLAGS, "-DOTHER"]
    build.age("b.cu", 10)
    build.build_lib()
    assert build.compiled() == ["a.cu", "b.cu", "c.cu"]
