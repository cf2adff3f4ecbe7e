"""Arguments that the operators' C entries turn down on the host, without a GPU: the checks come
before the device is touched, so a block of zeros stands in for the handle."""
import ctypes as C

import pytest

import pt_b200

OPS = pt_b200.Operators
HANDLE = (C.c_uint8 * 256)()
A = 1 << 20     # an address for tensors, aligned to everything
SIZES = {0: 4, 1: 2, 2: 2}


def _call(entry, struct, args):
    return entry(C.addressof(HANDLE), None, struct.pack(*args.values()))


def _linear(dtype, **kw):
    a = dict(dtype=dtype, act=5, rows=6, n_in=24, n_out=40, x=A, w=A, bias=A, res=A, y=A, pre=A, ldx=24, ldw=24,
             ldr=40, ldy=40, ldp=40, work=0, nbytes=0, slope=0.0)
    return _call(pt_b200.lib().pt_b200_linear, OPS._LINEAR, {**a, **kw})


def _linear_backward(dtype, **kw):
    a = dict(dtype=dtype, act=5, rows=6, n_in=24, n_out=40, dy=A, x=A, w=A, pre=A, dx=A, dw=A, db=A, lddy=40, ldx=24,
             ldw=24, ldp=40, lddx=24, lddw=24, work=0, nbytes=0, slope=0.0)
    return _call(pt_b200.lib().pt_b200_linear_backward, OPS._LINEAR_GRAD, {**a, **kw})


def _layer_norm(dtype, **kw):
    a = dict(dtype=dtype, eps=1e-5, rows=6, cols=24, x=A, gamma=A, beta=A, y=A, mean=A, rstd=A, ldx=24, ldy=24)
    return _call(pt_b200.lib().pt_b200_layer_norm, OPS._NORM, {**a, **kw})


def _layer_norm_backward(dtype, **kw):
    a = dict(dtype=dtype, reserved=0, rows=6, cols=24, dy=A, x=A, gamma=A, mean=A, rstd=A, dx=A, dgamma=A, dbeta=A,
             lddy=24, ldx=24, lddx=24, work=0, nbytes=0)
    return _call(pt_b200.lib().pt_b200_layer_norm_backward, OPS._NORM_GRAD, {**a, **kw})


# (call, its tensors of the call's type, its fp32 tensors)
CALLS = {"linear": (_linear, ["x", "w", "bias", "res", "y", "pre"], []),
         "linear_backward": (_linear_backward, ["dy", "x", "w", "pre", "dx", "dw", "db"], []),
         "layer_norm": (_layer_norm, ["x", "gamma", "beta", "y"], ["mean", "rstd"]),
         "layer_norm_backward": (_layer_norm_backward, ["dy", "x", "gamma", "dx", "dgamma", "dbeta"],
                                 ["mean", "rstd"])}
CASES = [(c, t, dt, SIZES[dt]) for c in CALLS for dt in SIZES for t in CALLS[c][1]]
CASES += [(c, t, dt, 4) for c in CALLS for dt in SIZES for t in CALLS[c][2]]


@pytest.mark.parametrize("name,which,dtype,size", CASES)
def test_pointers_between_elements(name, which, dtype, size):
    """Every tensor of every call, off by one byte up to one less than an element."""
    call, launches = CALLS[name][0], pt_b200.kernel_launches()
    for off in range(1, size):
        assert call(dtype, **{which: A + off}) == -1
        said = pt_b200.lib().pt_b200_last_error().decode()
        assert said.startswith(f"pt_b200_{name}:") and ("aligned" in said or "need" in said), said
        assert "device" not in said
    assert pt_b200.kernel_launches() == launches
