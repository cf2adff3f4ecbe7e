"""The library's makefile where the interpreter has no torch to build against."""
import os
import shutil
import subprocess

from conftest import PKG

MODULE = "_pt_b200_torch.so"


def _make(tmp_path, *args):
    return subprocess.run(["make", "-C", PKG, f"TORCHMOD={tmp_path}/{MODULE}", *args], capture_output=True, text=True)


def test_without_torch_the_library_alone_is_built(tmp_path):
    false = shutil.which("false")
    done = _make(tmp_path, f"PYTHON={false}")
    assert done.returncode == 0 and f"{MODULE} is not built" in done.stdout, done.stdout + done.stderr
    assert os.path.exists(os.path.join(PKG, "libpt_b200.so")) and not os.listdir(tmp_path)
    assert _make(tmp_path, f"PYTHON={false}", "torch").returncode != 0


def test_a_module_that_does_not_compile_fails_the_build(tmp_path):
    done = _make(tmp_path, f"HOSTCXX={shutil.which('false')}")
    assert done.returncode != 0
