"""CPU: what the build files build, and which libraries a process maps."""
import os
import subprocess
import sys

import pytest

from transformer_vae_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def planned(*goals):
    """The commands that make would run for a tree without anything built (nothing is run)."""
    return subprocess.run(["make", "-n", "-B", "-C", _lib.CSRC, *goals], capture_output=True, text=True, check=True).stdout


def test_the_library_is_built_without_torch():
    # the C interface's users have neither torch's headers nor, perhaps, a Python
    plan = planned()
    assert "libtvae_hip.so" in plan and "host.cpp" not in plan and "python" not in plan
    plan = planned("all", "host")
    assert "libtvae_hip.so" in plan and "host.cpp" in plan
