"""CPU: when the library and its C++ host side are built again."""
from __future__ import annotations

import pytest

from rus_b200 import build


@pytest.fixture
def built(tmp_path, monkeypatch):
    """Paths of their own and a compiler that writes its output file; returns the files compiled."""
    compiled = []

    def run(cmd, check):
        from pathlib import Path

        out = Path(cmd[cmd.index("-o") + 1])
        out.write_bytes(b"")
        compiled.append(out.name)

    for name in ("LIB_PATH", "HOST_PATH", "HOST_ABI"):
        monkeypatch.setattr(build, name, tmp_path / getattr(build, name).name)
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "compile_command", lambda: ["nvcc", "-o", "?"])
    return compiled


def test_what_is_up_to_date_stays(built):
    build.build_library()
    assert built == ["liblmce.so.tmp", "_host.so.tmp"]
    assert build.LIB_PATH.exists() and build.HOST_PATH.exists()
    build.build_library()
    assert len(built) == 2
    build.build_library(force=True)
    assert len(built) == 4


@pytest.mark.parametrize("change", ["torch", "python", "unknown"])
def test_another_torch_or_interpreter_rebuilds_the_host_side(built, monkeypatch, change):
    """Its sources' times do not tell: _lib.host() refuses it and asks for a build, which has to act."""
    build.build_library()
    del built[:]
    if change == "torch":
        import torch

        monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    elif change == "python":
        monkeypatch.setattr(build.sys.implementation, "cache_tag", "cpython-399")
    else:
        build.HOST_ABI.unlink()
    build.build_library()
    assert built == ["_host.so.tmp"]
    build.build_library()
    assert len(built) == 1
