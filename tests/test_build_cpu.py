"""The build with and without torch, and with another torch than last time."""

import os
import subprocess
import sys

import pytest


def test_library_builds_without_torch():
    """An interpreter without site-packages has no torch: the library is all there is to build."""
    from lightgbm_rs_b200 import build

    build.build()
    code = ("import importlib.util as u, sys\n"
            "s = u.spec_from_file_location('b', sys.argv[1])\n"
            "m = u.module_from_spec(s)\n"
            "s.loader.exec_module(m)\n"
            "assert u.find_spec('torch') is None\n"
            "print(m.build(), m.build_binding())\n")
    r = subprocess.run([sys.executable, "-S", "-E", "-c", code, build.__file__],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == [build.LIB, "None"]


def test_binding_is_rebuilt_for_another_torch(monkeypatch):
    pytest.importorskip("torch")
    from lightgbm_rs_b200 import build

    obj = os.path.join(build.BUILD, "experts_torch.cpp.o")
    assert build.build_binding() == build.BINDING
    assert not build._binding_stale(obj)
    monkeypatch.setattr(build, "_torch_stamp", lambda: "another")
    assert build._binding_stale(obj)
