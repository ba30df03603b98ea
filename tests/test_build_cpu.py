"""The build step: what it takes for up to date, and that processes that build at the same
time do not write to one file.  The compilers are replaced by a function that writes a file."""

import subprocess

import pytest
import torch

from qgemv_b200 import build


class Compiler:
    """Stands for nvcc and g++: writes the output named after -o, as process `pid`."""

    def __init__(self, monkeypatch, tmp_path):
        self.outputs, self.meanwhile = [], None
        monkeypatch.setattr(build, "PKG_DIR", tmp_path)
        monkeypatch.setattr(build, "LIB_PATH", tmp_path / "libqgemv_b200.so")
        monkeypatch.setattr(build, "torch_command", lambda out: ["g++", "-o", str(out)])
        monkeypatch.setattr(build, "up_to_date", lambda out=None: False)
        monkeypatch.setattr(subprocess, "run", self.run)
        (tmp_path.parent / "include").mkdir(exist_ok=True)
        (tmp_path.parent / "include" / "qgemv_b200.h").touch()

    def run(self, cmd, **_):
        out = cmd[cmd.index("-o") + 1]
        self.outputs.append(out)
        with open(out, "w") as f:
            f.write(f"made by {len(self.outputs)}")
        if self.meanwhile is not None:
            other, self.meanwhile = self.meanwhile, None
            other()
        return subprocess.CompletedProcess(cmd, 0, "", "")


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    (tmp_path / "pkg").mkdir()
    return Compiler(monkeypatch, tmp_path / "pkg")


def test_torch_front_end_belongs_to_the_installed_torch(compiler, monkeypatch):
    first = build.build_torch()
    assert len(compiler.outputs) == 1 and first.exists()
    assert build.build_torch() == first and len(compiler.outputs) == 1
    monkeypatch.setattr(torch, "__version__", "99.1.0+cu1")
    other = build.build_torch()  # compiled against other headers
    assert len(compiler.outputs) == 2 and other != first and other.exists()


@pytest.mark.parametrize("make", ["build", "build_torch"])
def test_builds_at_the_same_time_write_apart(compiler, monkeypatch, make):
    pid = [100]
    monkeypatch.setattr(build.os, "getpid", lambda: pid[0])

    def other_process():
        pid[0] = 200
        getattr(build, make)(force=True)
        pid[0] = 100

    compiler.meanwhile = other_process
    path = getattr(build, make)(force=True)
    assert len(set(compiler.outputs)) == 2
    assert path.read_text().startswith("made by")  # whole, whichever was renamed last
    assert list(path.parent.glob("*.tmp*")) == []
