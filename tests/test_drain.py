"""The copies that may be in flight when a kernel's producers stop early, checked on the CPU (no kernel is made
to give up on a GPU for it)."""
import os
import subprocess

from conftest import PKG

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_copy_in_flight_is_waited_for(tmp_path):
    exe = tmp_path / "drain"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(PKG, "csrc"),
                    os.path.join(HERE, "cpu_checks", "drain_check.cpp"), "-o", str(exe)], check=True)
    runs, bad = map(int, subprocess.run([str(exe)], capture_output=True, check=True).stdout.split())
    assert runs > 10000 and bad == 0
