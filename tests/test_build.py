"""The build of the torch binding: not needed for the C library, and done again when the torch it was built against changes.
A stand-in compiler and a stand-in python; nothing is compiled."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "orda-knowledge-distillation-kernel_amd" / "csrc"
pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def script(path, text):
    path.write_text("#!/bin/sh\n" + text)
    path.chmod(0o755)
    return str(path)


@pytest.fixture
def make(tmp_path):
    binding, log = tmp_path / "lib" / "binding.so", tmp_path / "compiled"
    compiler = script(tmp_path / "cxx", f'echo "$@" >> {log}\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')

    def run(python, target=str(binding)):
        env = {k: v for k, v in os.environ.items() if not k.startswith("MAKE")}
        out = subprocess.run(["make", "-C", str(CSRC), f"BUILD={tmp_path}/build", f"TOUT={binding}", f"CXX={compiler}",
                              f"PYTHON={python}", target], env=env, capture_output=True, text=True, timeout=60)
        return out, (log.read_text().splitlines() if log.exists() else [])

    run.binding = binding
    return run


def test_without_torch_the_binding_is_left_out(make, tmp_path):
    none = script(tmp_path / "none", "exit 1\n")
    for _ in range(2):
        out, compiled = make(none)
        assert out.returncode == 0, out.stderr
        assert "cannot import torch" in out.stdout and compiled == [] and not make.binding.exists()


def test_another_torch_builds_it_again(make, tmp_path):
    one, two = (script(tmp_path / n, f"echo -DORDA_TORCH={n}\n") for n in ("one", "two"))
    for python, builds in ((one, 1), (one, 1), (two, 2), (two, 2)):
        out, compiled = make(python)
        assert out.returncode == 0, out.stderr
        assert len(compiled) == builds and make.binding.exists()
    assert "-DORDA_TORCH=one" in compiled[0] and "-DORDA_TORCH=two" in compiled[1]


def test_the_binding_is_compiled_with_warnings(make, tmp_path):
    _, compiled = make(script(tmp_path / "one", "echo -DORDA_TORCH=1\n"))
    assert "-Wall" in compiled[0].split() and "-w" not in compiled[0].split()
