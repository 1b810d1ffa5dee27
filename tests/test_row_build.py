"""The row operators' Python extension: when make builds it, and what loading a wrong one says."""
import os
import shutil
import stat
import subprocess

import pytest

from armnet_hip import native

Error = native.ArmnetNativeError


def script(path, text):
    path.write_text("#!/bin/sh\n" + text + "\n")
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return str(path)


@pytest.fixture
def make(tmp_path):
    """runs make for the extension alone, with a compiler that only counts and an interpreter that says which torch it has"""
    if not shutil.which("make"):
        pytest.skip("no make")
    log = tmp_path / "compiled"
    log.write_text("")
    script(tmp_path / "g++", f'echo x >> {log}\nwhile [ "$1" != "-o" ]; do shift; done\n: > "$2"')
    env = dict(os.environ, PATH=f"{tmp_path}:{os.environ['PATH']}")
    env.pop("MAKEFLAGS", None)

    def run(python, target="rows"):
        out = subprocess.run(["make", "-C", native.CSRC, target, f"ROWS_OUT={tmp_path}/rows.so", f"OBJDIR={tmp_path}/obj", f"PYTHON={python}"],
                             env=env, capture_output=True, text=True)
        assert out.returncode == 0, out.stdout + out.stderr
        return len(log.read_text().split()), (tmp_path / "rows.so").exists()

    return run


def test_the_extension_follows_torch_and_the_interpreter(make, tmp_path):
    python = lambda says: script(tmp_path / "python", f"echo {says}")      # noqa: E731
    assert make(python("cpython-310 2.10.0")) == (1, True)
    assert make(python("cpython-310 2.10.0")) == (1, True)       # up to date
    assert make(python("cpython-310 2.11.0")) == (2, True)       # another torch
    assert make(python("cpython-312 2.11.0")) == (3, True)       # another interpreter
    assert make(python("cpython-312 2.11.0")) == (3, True)


def test_the_c_libraries_need_no_torch(make, tmp_path):
    assert make(script(tmp_path / "python", "exit 1")) == (0, False)
    assert make(str(tmp_path / "nowhere")) == (0, False)


def test_the_default_target_builds_both():
    text = open(os.path.join(native.CSRC, "Makefile")).read()
    assert "\nall: libs rows\n" in text and "\nlibs: $(OUT) $(IO_OUT)\n" in text


def fresh(monkeypatch):
    native.rows()
    monkeypatch.setattr(native, "_rows", None)


def test_an_extension_for_other_entries_is_refused(monkeypatch):
    """the entries' signatures are compiled in"""
    fresh(monkeypatch)
    monkeypatch.setattr(native, "ABI_VERSION", native.ABI_VERSION + 1)
    with pytest.raises(Error, match="ABI"):
        native.rows()
    assert native._rows is None


def test_an_extension_that_cannot_be_loaded_says_what_to_do(monkeypatch, tmp_path):
    fresh(monkeypatch)
    bad = tmp_path / "_armnet_rows.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(native, "ROWS_PATH", str(bad))
    with pytest.raises(Error, match="build"):
        native.rows()
    monkeypatch.setattr(native, "ROWS_PATH", str(tmp_path / "nowhere.so"))
    with pytest.raises(Error, match="missing"):
        native.rows()
