"""build.py makes an object again where the command that compiles it has changed (another compiler, Python, torch or flag),
and links again where the list of objects has."""
import ctypes
import importlib.util
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("boxconv_b200_build_under_test", os.path.join(ROOT, "box-convolutions_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "OBJECTS", str(tmp_path / "objects"))
    return module


def source(tmp_path, name, text):
    path = tmp_path / name
    path.write_text(text)
    os.utime(path, (1, 1))      # (older than every object)
    return str(path)


def test_another_command_makes_another_object(build, tmp_path):
    src = source(tmp_path, "value.cpp", "extern \"C\" int value() { return VALUE; }\n")
    made = lambda *flags: build.compile_all(["g++", "-fPIC", *flags], [src], False, False)  # noqa: E731
    one, new = made("-DVALUE=1")
    assert new
    assert made("-DVALUE=1") == (one, False)
    two, new = made("-DVALUE=2")
    assert new and open(two[0], "rb").read() != open(one[0], "rb").read()
    # and back: the object is the first command's again
    again, _ = made("-DVALUE=1")
    out = str(tmp_path / "lib.so")
    build.link(["g++", "-shared"], [], out, again, False)
    assert ctypes.CDLL(out).value() == 1


def test_what_the_compiler_is_counts(build, tmp_path):
    src = source(tmp_path, "f.cpp", "int f() { return 3; }\n")
    assert build.compile_all(["g++"], [src], False, False)[1]
    assert not build.compile_all(["g++"], [src], False, False)[1]
    assert build.compile_all(["g++"], [src], False, False, also="torch 99")[1]
    other = tmp_path / "other"      # (a compiler of the same place and another version)
    for version, new in (("1", True), ("1", False), ("2", True)):
        other.write_text("#!/bin/sh\nif [ \"$1\" = --version ]; then echo %s; else exec g++ \"$@\"; fi\n" % version)
        other.chmod(0o755)
        assert build.compile_all([str(other)], [src], False, False)[1] == new


def test_a_source_that_is_gone_is_linked_no_more(build, tmp_path):
    a = source(tmp_path, "a.cpp", "extern \"C\" int a() { return 1; }\n")
    b = source(tmp_path, "b.cpp", "extern \"C\" int b() { return 2; }\n")
    out = str(tmp_path / "lib.so")
    assert build.link(["g++", "-shared"], [], out, build.compile_all(["g++", "-fPIC"], [a, b], False, False)[0], False)
    assert not build.link(["g++", "-shared"], [], out, build.compile_all(["g++", "-fPIC"], [a, b], False, False)[0], False)
    assert build.link(["g++", "-shared"], [], out, build.compile_all(["g++", "-fPIC"], [a], False, False)[0], False)
    assert "b" not in symbols(out) and "a" in symbols(out)


def symbols(path):
    return {line.split()[-1] for line in subprocess.check_output(["nm", "-D", "--defined-only", path], text=True).splitlines()}
