"""When the in-tree build compiles again, with stand-ins for nvcc and g++ that write down what they were called with."""

import importlib.util
import os
import stat

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COMPILER = """#!/bin/sh
if [ "$1" = "--version" ]; then cat "%(dir)s/version"; exit 0; fi
echo "$@" >> "%(dir)s/calls"
[ -e "%(dir)s/broken" ] && exit 1
while [ $# -gt 0 ]; do if [ "$1" = "-o" ]; then echo built > "$2"; fi; shift; done
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module over a tree of two sources and a header, and `ran()`: what was compiled and linked since."""
    tools, csrc = tmp_path / "tools", tmp_path / "csrc"
    tools.mkdir(), csrc.mkdir()
    (tools / "version").write_text("compiler 1\n")
    for name in ("nvcc", "g++"):
        exe = tools / name
        exe.write_text(COMPILER % {"dir": tools})
        exe.chmod(exe.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("PATH", str(tools) + os.pathsep + os.environ["PATH"])
    (csrc / "a.cu").write_text('#include "shared.cuh"\n')
    (csrc / "b.cu").write_text("int b;\n")
    (csrc / "shared.cuh").write_text("int a;\n")
    (csrc / "tensor_calls.cpp").write_text("int c;\n")
    for f in csrc.iterdir():
        os.utime(f, (1e9, 1e9))
    spec = importlib.util.spec_from_file_location("_ftk_build_under_test", os.path.join(ROOT, "fusedtok_b200", "_build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for name, value in dict(HERE=str(tmp_path), CSRC=str(csrc), LIB=str(tmp_path / "lib.so"), BOUNDS_LIB=str(tmp_path / "bounds.so"),
                            SOURCES=["a.cu", "b.cu"], OBJECTS=str(tmp_path / "build"), BINDING=str(tmp_path / "_tensors.so")).items():
        monkeypatch.setattr(module, name, value)

    def ran():
        calls = tools / "calls"
        lines = calls.read_text().splitlines() if calls.exists() else []
        calls.write_text("")
        made = [os.path.basename(x.split("-o ")[1].split()[0]) for x in lines]
        return sorted(made), lines
    module.ran, module.tools, module.csrc = ran, tools, csrc
    return module


EVERYTHING = sorted(["a.o", "b.o", "a_FTK_BOUNDS.o", "b_FTK_BOUNDS.o", "lib.so", "bounds.so", "_tensors.so"])


def test_nothing_is_built_twice(build):
    build.build_all()
    assert build.ran()[0] == EVERYTHING
    build.build_all()
    build.build()
    assert build.ran()[0] == []
    build.build_all(force=True)
    assert build.ran()[0] == EVERYTHING


def test_a_changed_header_compiles_what_includes_it(build):
    build.build_all()
    build.ran()
    os.utime(build.csrc / "shared.cuh")
    build.build_all()
    assert build.ran()[0] == sorted(["a.o", "a_FTK_BOUNDS.o", "lib.so", "bounds.so"])


def test_changed_flags_compile_everything_again(build, monkeypatch):
    build.build_all()
    build.ran()
    monkeypatch.setattr(build, "NVCC_FLAGS", build.NVCC_FLAGS + ["-lineinfo2"])
    build.build_all()
    made, lines = build.ran()
    assert made == [n for n in EVERYTHING if n != "_tensors.so"]
    assert all("-lineinfo2" in x for x in lines if " -c " in x)
    monkeypatch.setattr(build, "NVCC_FLAGS", build.NVCC_FLAGS[:-1])
    build.build()
    assert build.ran()[0] == ["a.o", "b.o", "lib.so"]


def test_changed_link_flags_and_sources_link_again(build, monkeypatch):
    build.build_all()
    build.ran()
    monkeypatch.setattr(build, "LINK_FLAGS", build.LINK_FLAGS + ["-lm"])
    build.build_all()
    assert build.ran()[0] == ["bounds.so", "lib.so"]
    monkeypatch.setattr(build, "SOURCES", ["a.cu"])
    build.build_all()
    assert build.ran()[0] == ["bounds.so", "lib.so"]


def test_another_compiler_compiles_everything_again(build):
    build.build_all()
    build.ran()
    (build.tools / "version").write_text("compiler 2\n")
    build.build_all()
    assert build.ran()[0] == EVERYTHING


def test_a_verbose_build_compiles_what_it_reports(build):
    build.build_all()
    build.ran()
    build.build(verbose=True)
    made, lines = build.ran()
    assert made == ["a.o", "b.o", "lib.so"]
    assert all("-Xptxas -v" in x for x in lines if " -c " in x)
    build.build_all()
    assert build.ran()[0] == []                             # (the report changes nothing of what is built)


def test_what_failed_is_compiled_again(build):
    build.build_all()
    build.ran()
    os.utime(build.csrc / "b.cu")
    (build.tools / "broken").write_text("")
    with pytest.raises(RuntimeError):
        build.build()
    (build.tools / "broken").unlink()
    build.ran()
    build.build()
    assert build.ran()[0] == ["b.o", "lib.so"]


def test_a_moved_tree_is_up_to_date(build, monkeypatch, tmp_path):
    """The commands hold paths of the tree; where the tree lies does not matter to what they build."""
    build.build_all()
    build.ran()
    where = tmp_path / "moved"
    where.mkdir()
    for name in ("csrc", "build", "lib.so", "bounds.so", "_tensors.so"):
        os.rename(tmp_path / name, where / name)
    for name in ("HERE", "CSRC", "LIB", "BOUNDS_LIB", "OBJECTS", "BINDING"):
        monkeypatch.setattr(build, name, getattr(build, name).replace(str(tmp_path), str(where)))
    build.build_all()
    assert build.ran()[0] == []


def test_a_variant_is_built_where_it_is_asked_for(build, tmp_path):
    build.build_all()
    build.ran()
    other = str(tmp_path / "other.so")
    assert build.build(out=other) == other and os.path.exists(other)
    assert build.build(defines=["FTK_X"], out=other) == other
    assert build.ran()[0] == sorted(["other.so", "a_FTK_X.o", "b_FTK_X.o", "other.so"])


def test_without_a_compiler_what_is_there_is_used(build, monkeypatch):
    build.build_all()
    build.ran()
    monkeypatch.setenv("PATH", "")
    assert build.build_all() == build.LIB and build.build() == build.LIB
    os.utime(build.csrc / "b.cu")
    with pytest.raises(FileNotFoundError):
        build.build()
