"""The transformer-layer operators' host side, without a GPU: the argument structs as ctypes packs
them, and the refusals that need no device."""
import os
import re
import subprocess
import tempfile

import pytest

import pt_b200

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"pt_b200_linear_args": "_LINEAR", "pt_b200_linear_grad_args": "_LINEAR_GRAD",
           "pt_b200_norm_args": "_NORM", "pt_b200_norm_grad_args": "_NORM_GRAD"}


def _fields(name):
    text = open(os.path.join(REPO, "include", "pt_b200.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
    out = []
    for decl in body.split(";"):
        if decl.strip():
            first, *rest = decl.split(",")
            out += [re.findall(r"\w+", first)[-1]] + [re.findall(r"\w+", r)[-1] for r in rest]
    return out


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_packed_structs_match_the_header(name):
    """Field i packed with the value i + 1 reads back as i + 1 through the C struct."""
    fields = _fields(name)
    packed = getattr(pt_b200.Operators, STRUCTS[name]).pack(*range(1, len(fields) + 1))
    src = ['#include <stdio.h>', '#include "pt_b200.h"', "int main(void){", f"  {name} a;",
           "  if (fread(&a, sizeof a, 1, stdin) != 1 || getchar() != EOF) return 1;"]
    src += [f'  printf("%lld\\n", (long long)a.{f});' for f in fields]
    src.append("  return 0;}")
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "p.c"), "w").write("\n".join(src))
        subprocess.run(["gcc", "-w", "-std=gnu11", "-I", os.path.join(REPO, "include"),
                        os.path.join(d, "p.c"), "-o", os.path.join(d, "p")], check=True)
        got = subprocess.run([os.path.join(d, "p")], input=packed, capture_output=True, check=True).stdout
    assert [int(v) for v in got.split()] == list(range(1, len(fields) + 1))


def test_null_handles_are_refused():
    lib = pt_b200.lib()
    ops = pt_b200.Operators
    assert lib.pt_b200_linear(None, None, bytes(ops._LINEAR.size)) == -1
    assert b"NULL handle" in lib.pt_b200_last_error()
    assert lib.pt_b200_linear_backward(None, None, bytes(ops._LINEAR_GRAD.size)) == -1
    assert lib.pt_b200_layer_norm(None, None, bytes(ops._NORM.size)) == -1
    assert lib.pt_b200_layer_norm_backward(None, None, bytes(ops._NORM_GRAD.size)) == -1
    assert lib.pt_b200_ops_sync(None, None) == -1
    assert lib.pt_b200_linear_backward_work(None, bytes(ops._LINEAR_GRAD.size)) == 0
    lib.pt_b200_ops_destroy(None)


def test_no_such_device():
    with pytest.raises(pt_b200.PtB200Error, match="out of range"):
        pt_b200.Operators(device=63)


def test_cpu_tensors_are_refused():
    """The torch entry points turn a tensor elsewhere down before the handle is used; there is no CPU
    path."""
    torch = pytest.importorskip("torch")
    call, t = pt_b200._torch_module(), torch.zeros(2, 4)
    for fn, args in (("linear", (t, t, None, None, 0, 0.1, False)),
                     ("linear_backward", (t, t, t, None, 0, 0.1, True, True, True)),
                     ("layer_norm", (t, None, None, 1e-5)),
                     ("layer_norm_backward", (t, t, None, t, t, True, True, True))):
        with pytest.raises(pt_b200.PtB200Error, match="on cuda:0, got torch.float32 on cpu"):
            getattr(call, fn)(1, 0, *args)
        with pytest.raises(pt_b200.PtB200Error, match="have been closed"):
            getattr(call, fn)(0, 0, *args)
        with pytest.raises(pt_b200.PtB200Error, match="needs a tensor"):
            getattr(call, fn)(1, 0, None, *args[1:])
        with pytest.raises(TypeError, match="arguments are needed"):
            getattr(call, fn)(1, 0)
