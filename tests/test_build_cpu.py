"""Which compiler the operator library is built with."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "relation-lm_b200" / "csrc"

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="make is not installed")


def compiler_of(*arguments, **environment):
    env = {k: v for k, v in os.environ.items() if k not in ("CXX", "HOST_CXX", "MAKEFLAGS")}
    dry = subprocess.run(["make", "-n", "-C", str(CSRC), "-W", "torch_ops.cpp", "torch_ops.o", *arguments], env={**env, **environment},
                         capture_output=True, text=True, check=True)
    line = next(x for x in dry.stdout.splitlines() if " -O2 " in x)
    return line.split()[0]


@pytest.mark.parametrize("where", ("environment", "command line"))
@pytest.mark.parametrize("runtime,chosen", [("/usr/lib/libstdc++.so", True), ("libstdc++.so", False)])
def test_a_chosen_compiler_builds_the_operators_if_its_runtime_is_shared(tmp_path, where, runtime, chosen):
    compiler = tmp_path / "c++"
    compiler.write_text(f"#!/bin/sh\necho {runtime}\n")
    compiler.chmod(0o755)
    got = compiler_of(CXX=str(compiler)) if where == "environment" else compiler_of(f"CXX={compiler}")
    assert got == (str(compiler) if chosen else "g++")
    assert compiler_of(f"HOST_CXX={compiler}") == str(compiler)


def test_without_a_choice():
    assert compiler_of() == "g++"
