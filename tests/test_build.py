"""When the native binaries are built again, and what importing a stale extension says."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

from pagedcore_b200 import build
from tests.conftest import ROOT


@pytest.fixture
def extension(tmp_path, monkeypatch):
    """A fresh extension of this torch in a folder of its own; its builds are recorded, not made."""
    monkeypatch.setattr(build, "EXTENSION", tmp_path / "_int4_ops.so")
    monkeypatch.setattr(build, "EXTENSION_STAMP", tmp_path / "_int4_ops.built_for")
    monkeypatch.setattr(build, "_library_up_to_date", lambda: True)
    builds = []
    monkeypatch.setattr(build, "_run", lambda command, tmp, target, verbose: (builds.append(command), target.write_bytes(b"")))
    build.build()
    assert len(builds) == 1 and build.up_to_date()
    return builds


@pytest.mark.parametrize("what", ["torch", "python", "no record", "source"])
def test_the_extension_is_built_again_when_what_it_depends_on_changes(what, extension, tmp_path, monkeypatch) -> None:
    import torch

    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    elif what == "python":
        monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-other")
    elif what == "no record":
        build.EXTENSION_STAMP.unlink()
    else:
        os.utime(build.EXTENSION, (1, 1))
    assert not build.up_to_date()
    build.build()
    assert len(extension) == 2 and build.up_to_date()
    build.build()
    assert len(extension) == 2  # nothing left to do


def test_an_extension_of_another_torch_is_not_taken() -> None:
    code = (
        "import torch; torch.__version__ = '9.9.9'\n"
        "try:\n    import pagedcore_b200.int4\n"
        "except ImportError as error:\n    print(error, '|', error.__cause__)\n"
    )
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert "python -m pagedcore_b200.build" in done.stdout and "torch 9.9.9" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("lacks", ["Python's headers", "torch", "CUDA"])
def test_the_library_is_built_without_what_only_the_extension_needs(lacks, tmp_path, monkeypatch, capsys) -> None:
    import torch

    if lacks == "Python's headers":
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    elif lacks == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)  # importing it raises ImportError
    else:
        (tmp_path / "include" / "ATen").mkdir(parents=True)
        (tmp_path / "include" / "ATen" / "ATen.h").touch()
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    library = tmp_path / "libpagedkv.so"
    monkeypatch.setattr(build, "LIBRARY", library)
    monkeypatch.setattr(build, "EXTENSION", tmp_path / "_int4_ops.so")
    monkeypatch.setattr(build, "EXTENSION_STAMP", tmp_path / "_int4_ops.built_for")
    monkeypatch.setattr(build, "_run", lambda command, tmp, target, verbose: target.write_bytes(b""))
    assert not build.up_to_date()
    assert build.build() == library and library.exists() and not build.EXTENSION.exists()
    assert lacks in capsys.readouterr().err and build.up_to_date()


def test_an_extension_that_does_not_say_what_it_was_built_for_is_not_taken() -> None:
    code = (
        "import sys, types, pagedcore_b200\n"
        "pagedcore_b200._int4_ops = sys.modules['pagedcore_b200._int4_ops'] = types.ModuleType('_int4_ops')\n"
        "try:\n    import pagedcore_b200.int4\n"
        "except ImportError as error:\n    print(error, '|', error.__cause__)\n"
    )
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert "python -m pagedcore_b200.build" in done.stdout and "earlier form" in done.stdout, done.stdout + done.stderr
