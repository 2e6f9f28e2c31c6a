"""The compiled host path (csrc/autograd.cpp) is taken only if it was compiled against the entry points it calls, and two processes that
build it at the same time do not write one file."""

import os
import re
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_one_abi_version_everywhere():
    from cute_kernels import _C, _native

    header = open(os.path.join(ROOT, "include", "cute_hip.h")).read()
    (version,) = re.findall(r"#define CK_ABI_VERSION (\d+)", header)
    assert int(version) == _C._ABI_VERSION == _C.load_library().ck_abi_version() == _native.load().abi_version


@pytest.mark.parametrize("built_for", [None, "older", "newer"])
def test_an_extension_built_for_other_signatures_is_refused(monkeypatch, built_for):
    from cute_kernels import _C, _native

    module = types.SimpleNamespace(load=lambda *args: pytest.fail("connected to the library"))
    if built_for is not None:
        module.abi_version = _C._ABI_VERSION + (1 if built_for == "newer" else -1)
    monkeypatch.setattr(_native, "_module", None)
    monkeypatch.setattr(_native, "_import", lambda path: module)
    with pytest.raises(RuntimeError, match="rebuild"):
        _native.load()
    assert _native._module is None


def test_each_process_builds_into_a_file_of_its_own(monkeypatch, tmp_path):
    from cute_kernels import _build

    monkeypatch.setattr(_build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(_build, "AUTOGRAD_PATH", str(tmp_path / "cute_autograd.so"))
    written = []

    def run(cmd, **kwargs):
        target = cmd[cmd.index("-o") + 1]
        written.append(target)
        with open(target, "w") as f:
            f.write("built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(_build.subprocess, "run", run)
    for pid in (11, 12):
        monkeypatch.setattr(_build.os, "getpid", lambda: pid)
        assert _build.build_autograd() == str(tmp_path / "cute_autograd.so")
    assert len(set(written)) == 2 and os.listdir(tmp_path) == ["cute_autograd.so"]
