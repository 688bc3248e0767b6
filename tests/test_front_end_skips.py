"""Only the front end's absence turns a failed test into a skip: run in pytest processes of their own."""

from __future__ import annotations

import importlib.util
import os
from pathlib import Path
import subprocess
import sys

import pytest

TESTS = Path(__file__).resolve().parent


def outcomes(folder: Path, source: str) -> str:
    (folder / "test_it.py").write_text(source)
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(folder), str(TESTS)]))
    done = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "conftest", "-p", "no:cacheprovider",
                           f"--rootdir={folder}", str(folder / "test_it.py")],
                          cwd=folder, env=env, capture_output=True, text=True, timeout=120)
    return done.stdout.strip().splitlines()[-1]


BROKEN = """
def test_import():
    import chomikgrad.{name}

def test_child():
    raise RuntimeError("the child ended: ModuleNotFoundError: No module named '{name}' (chomikgrad's rank 1)")
"""


def test_broken_imports_of_an_installed_package_fail(tmp_path):
    (tmp_path / "chomikgrad").mkdir()
    (tmp_path / "chomikgrad" / "__init__.py").write_text("")
    (tmp_path / "chomikgrad" / "whole.py").write_text("import chomikgrad.lost")
    assert outcomes(tmp_path, BROKEN.format(name="whole")).startswith("2 failed")
    child = "def test_it():\n    raise RuntimeError(\"ModuleNotFoundError: No module named 'chomikgrad'\")\n"
    assert outcomes(tmp_path, child).startswith("1 failed")  # a child that lost its path
    assert outcomes(tmp_path, "import chomikgrad.whole\n").startswith("1 error")


@pytest.mark.skipif(importlib.util.find_spec("chomikgrad") is not None, reason="the front end is installed")
def test_only_the_missing_front_end_skips(tmp_path):
    assert outcomes(tmp_path, "import chomikgrad\n").startswith("1 skipped")
    assert outcomes(tmp_path, BROKEN.format(name="tensor")).startswith("1 failed, 1 skipped")
    child = "def test_it():\n    raise RuntimeError(\"ModuleNotFoundError: No module named 'chomikgrad'\")\n"
    assert outcomes(tmp_path, child).startswith("1 skipped")
    assert outcomes(tmp_path, "import other_chomikgrad\n").startswith("1 error")
    rank = "def test_it():\n    got = repr(ModuleNotFoundError(\"No module named '{}'\"))\n    assert not got, got\n"
    assert outcomes(tmp_path, rank.format("chomikgrad")).startswith("1 skipped")
    assert outcomes(tmp_path, rank.format("whole")).startswith("1 failed")
