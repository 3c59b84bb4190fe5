"""What the build needs: the library and the C++ shim no torch, the binding the torch and Python that it is loaded into."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """build.py with its targets in a folder of their own and compilers that only write their output."""
    from kiln_b200 import build
    for name in ("LIB", "HOST_LIB", "BINDING"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    calls = []

    def run(cmd, **_):
        calls.append(os.path.basename(cmd[cmd.index("-o") + 1]).replace(".new", ""))
        tag = [c.split("=", 1)[1].strip('"') for c in cmd if c.startswith("-DKB_BUILT_FOR")]
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("".join(f"[{t}]" for t in tag))
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build.subprocess, "run", run)
    return build, calls


def test_without_torch(recorded, monkeypatch, capsys):
    build, calls = recorded
    found = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else found(name, *a))
    assert build.build() == build.LIB and build.build_host() == build.HOST_LIB
    assert calls == ["libkiln_b200.so", "libkiln_engine_ops.so"] and not os.path.exists(build.BINDING)
    assert build.build_binding() is None and "torch" in capsys.readouterr().err


def test_library_first_and_nothing_twice(recorded):
    build, calls = recorded
    build.build()
    build.build()
    assert calls == ["libkiln_b200.so", "_kiln_torch.so"]


def test_binding_of_another_torch_is_rebuilt(recorded, monkeypatch):
    build, calls = recorded
    build.build_binding()
    build.build_binding()
    assert calls == ["_kiln_torch.so"]
    tag = build.torch_tag
    monkeypatch.setattr(build, "torch_tag", lambda d: tag(d).replace("torch ", "torch 9."))
    build.build_binding()
    build.build_binding()
    assert calls == ["_kiln_torch.so"] * 2


def test_binding_of_another_torch_is_not_loaded(built_lib):
    code = ("import kiln_b200.build as b, kiln_b200.ops as o\n"
            "assert o._b().built_for == b.torch_tag(__import__('os').path.dirname(__import__('torch').__file__))\n"
            "o._binding = None; b.torch_tag = lambda d: 'torch 0.1, other'\n"
            "try: o._b()\nexcept ImportError as e: assert 'torch 0.1' in str(e) and 'kiln_b200.build' in str(e)\nelse: raise SystemExit(3)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
