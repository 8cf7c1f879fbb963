"""When the CPython binding is rebuilt (the compiler is a stand-in)."""
import os
import subprocess

import pytest

from butterfly_b200 import build


@pytest.fixture
def calls(tmp_path, monkeypatch):
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("built")
        os.utime(out, (2 ** 33, 2 ** 33))  # newer than every source
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "NATIVE", str(tmp_path / "_native.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", run)
    return made


def test_built_once_and_again_for_another_torch(calls, monkeypatch):
    build._build_binding()
    build._build_binding()
    assert len(calls) == 1
    monkeypatch.setattr(build.metadata, "version", lambda name: "99.0")
    build._build_binding()
    build._build_binding()
    assert len(calls) == 2


def test_a_failed_build_is_tried_again(calls, monkeypatch):
    build._build_binding()
    monkeypatch.setattr(build.metadata, "version", lambda name: "99.0")
    good = build.subprocess.run
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: subprocess.CompletedProcess(cmd, 1, "", "no"))
    with pytest.raises(RuntimeError):
        build._build_binding()
    monkeypatch.setattr(build.subprocess, "run", good)
    build._build_binding()
    assert len(calls) == 2
