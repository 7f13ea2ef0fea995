"""The build of the serving operators' extension module, without a GPU and without compiling anything."""
import os
import subprocess

import pytest

from pto_isa_b200 import build


@pytest.fixture()
def dry(monkeypatch, tmp_path):
    """build() with every target stale, its outputs in a folder of their own and its commands recorded; a command that names
    torch_fast.cpp fails when `fail` is set."""
    class Dry:
        commands, fail, here = [], False, tmp_path

    def call(cmd, **kw):
        Dry.commands.append(" ".join(cmd))
        if Dry.fail and "torch_fast.cpp" in Dry.commands[-1]:
            raise subprocess.CalledProcessError(1, cmd)
    Dry.commands = []
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "_stale", lambda target, deps: True)
    monkeypatch.setattr(build.subprocess, "check_call", call)
    return Dry


def test_build_goes_on_without_the_extension_module(dry):
    (dry.here / "_fast.so").write_text("of an older build")
    dry.fail = True
    with pytest.warns(UserWarning, match="extension module"):
        assert build.build() == build.LIB
    for shim in build.SHIMS.values():
        assert any(shim in c for c in dry.commands)
    assert not os.path.exists(dry.here / "_fast.so")


def test_build_makes_the_extension_module(dry, recwarn):
    build.build()
    assert sum("torch_fast.cpp" in c for c in dry.commands) == 1 and not [w for w in recwarn if "extension module" in str(w.message)]
