"""What `make` under csrc/ builds, by its own account (make -n: nothing is built)."""
import os
import subprocess
import sys
import sysconfig

import pytest

from berth_b200 import _lib


def _plan(*args):
    return subprocess.run(["make", "-n", "-B", "-C", _lib.CSRC, *args], capture_output=True, text=True)


@pytest.mark.parametrize("python", ["python3", "/nowhere/python"])
def test_the_c_library_alone_needs_no_python(python):
    """A C or Rust host's `make`: the library, on a machine without an interpreter too."""
    r = _plan(f"PYTHON={python}")
    assert r.returncode == 0, r.stderr
    assert "libberth_b200.so" in r.stdout and "bind.c" not in r.stdout and "nowhere" not in r.stdout + r.stderr


def test_the_callers_are_of_one_interpreter():
    """`make bind`: against the headers of the interpreter that is named, under the name that only such interpreters load."""
    r = _plan("bind", f"PYTHON={sys.executable}")
    assert r.returncode == 0, r.stderr
    compiled = [line for line in r.stdout.splitlines() if "bind.c" in line]
    assert len(compiled) == 1 and "-I" + sysconfig.get_paths()["include"] + " " in compiled[0]
    assert "_bind" + sysconfig.get_config_var("EXT_SUFFIX") in compiled[0] and "libberth_b200.so" in r.stdout
    r = _plan("bind", "PYTHON=/nowhere/python")
    assert r.returncode != 0 and "/nowhere/python" in r.stderr


def test_the_loaded_callers_are_this_interpreter_s():
    if not os.path.exists(_lib.SO_PATH):
        _lib.build()
    assert _lib.bind().__file__.endswith("_bind" + sysconfig.get_config_var("EXT_SUFFIX"))


def test_build_asks_for_both(monkeypatch):
    """_lib.build() builds the callers of the interpreter that it runs in."""
    asked = []
    monkeypatch.setattr(_lib.subprocess, "run", lambda cmd, **kw: asked.append((cmd, kw)))
    _lib.build()
    (cmd, kw), = asked
    assert cmd[0] == "make" and "bind" in cmd and f"PYTHON={sys.executable}" in cmd and kw["check"]
