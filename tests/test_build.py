"""When the library and the binding are built, with the compilers played by a fake."""

import os

import pytest

from ktir_cpu_b200 import build as B


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """Targets in a folder of the test's own; compilers that only leave their output."""
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("built")

    class Process:
        returncode = 0

        def __init__(self, cmd, **kw):
            run(cmd)

        def communicate(self):
            return b"", b""

    monkeypatch.setattr(B, "HERE", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "_serving.so"))
    monkeypatch.setattr(B, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(B.subprocess, "Popen", Process)
    monkeypatch.setattr(B.subprocess, "check_call", run)
    return commands


def test_builds_once(fake):
    assert not B.up_to_date()
    B.build()
    n = len(fake)
    assert n and os.path.exists(B.LIB) and os.path.exists(B.BINDING) and B.up_to_date()
    B.build()
    assert len(fake) == n


def test_without_torch_the_library_alone_is_built(fake, monkeypatch):
    monkeypatch.setattr(B, "_torch", lambda: None)
    B.build()
    assert os.path.exists(B.LIB) and not os.path.exists(B.BINDING) and B.up_to_date()
    assert not any("serving_binding.cpp" in part for cmd in fake for part in cmd)


def test_another_torch_wants_another_binding(fake, monkeypatch):
    B.build()
    assert B.up_to_date()
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "0.0.1")
    assert not B.up_to_date()
    n = len(fake)
    B.build()
    assert len(fake) > n and B.up_to_date()
