"""The transformer-layer operators on rows that lie far apart: element offsets over 2^31 in every matrix of
a call, inputs and outputs, through the C entries.  The same call with rows close together (and of the
same alignment) has to give the same bits."""
import pytest

import pt_b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    o = pt_b200.Operators(0)
    yield o
    o.sync()
    o.close()


def _far(rows, near):
    """A row stride that puts the last of `rows` rows over 2^31 elements, of near's alignment."""
    ld = ((1 << 31) // (rows - 1) // 64 + 2) * 64 + near % 64
    assert (rows - 1) * ld > 1 << 31 and (ld - near) % 8 == 0
    return ld


class Matrices:
    """Matrices side by side as columns of one wide tensor, `shift` elements off its alignment."""

    def __init__(self, rows, widths, dtype, ld, shift):
        self.at, end = {}, shift
        for name, width in widths.items():
            self.at[name] = (end, width)
            end += (width + 15) // 16 * 16
        assert end <= ld
        self.wide, self.ld = torch.empty(rows, ld, dtype=dtype, device="cuda"), ld

    def __getitem__(self, name):
        begin, width = self.at[name]
        return self.wide[:, begin:begin + width]

    def ptr(self, name):
        return self[name].data_ptr()


def _rand(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _work(need):
    return torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")


def _linear(ops, m, dtype, rows, n_in, n_out, w, b):
    args = [TYPES[dtype], 6, rows, n_in, n_out, m.ptr("x"), w.data_ptr(), b.data_ptr(), m.ptr("r"), m.ptr("y"),
            m.ptr("pre"), m.ld, n_in, m.ld, m.ld, m.ld, 0, 0, 0.0]
    need = ops._lib.pt_b200_linear_work(ops.h, ops._LINEAR.pack(*args))
    work = _work(need)
    args[16], args[17] = work.data_ptr(), need
    assert ops._lib.pt_b200_linear(ops.h, ops._stream(), ops._LINEAR.pack(*args)) == 0


def _linear_backward(ops, m, dtype, rows, n_in, n_out, w):
    dw, db = torch.empty_like(w), torch.empty(n_out, dtype=dtype, device="cuda")
    args = [TYPES[dtype], 6, rows, n_in, n_out, m.ptr("r"), m.ptr("x"), w.data_ptr(), m.ptr("pre"), m.ptr("dx"),
            dw.data_ptr(), db.data_ptr(), m.ld, m.ld, n_in, m.ld, m.ld, n_in, 0, 0, 0.0]
    need = ops._lib.pt_b200_linear_backward_work(ops.h, ops._LINEAR_GRAD.pack(*args))
    work = _work(need)
    args[18], args[19] = work.data_ptr(), need
    assert ops._lib.pt_b200_linear_backward(ops.h, ops._stream(), ops._LINEAR_GRAD.pack(*args)) == 0
    return dw, db


# the few-rows kernel, the products in tiles, fp32 against a few channels; aligned rows and others
@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("dtype,rows,n_in,n_out", [
    (torch.bfloat16, 3, 96, 72), (torch.float32, 3, 96, 72), (torch.bfloat16, 200, 96, 72), (torch.float16, 200, 97, 71),
    (torch.float32, 200, 192, 136), (torch.float32, 9500, 130, 25), (torch.float32, 9500, 256, 16)])
def test_linear(ops, dtype, rows, n_in, n_out, shift):
    near = 1024 + (0 if shift == 0 else 8 + shift)
    w, b = _rand(1, n_out, n_in, dtype=dtype), _rand(2, n_out, dtype=dtype)
    x, r = _rand(3, rows, n_in, dtype=dtype), _rand(4, rows, n_out, dtype=dtype)
    got = []
    for ld in (near, _far(rows, near)):
        m = Matrices(rows, {"x": n_in, "r": n_out, "y": n_out, "pre": n_out, "dx": n_in}, dtype, ld, shift)
        m["x"].copy_(x)
        m["r"].copy_(r)
        _linear(ops, m, dtype, rows, n_in, n_out, w, b)
        dw, db = _linear_backward(ops, m, dtype, rows, n_in, n_out, w)
        got.append([m[k].clone() for k in ("y", "pre", "dx")] + [dw, db])
        del m
    assert torch.allclose(got[0][1].float(), x.float() @ w.float().T + b.float(), rtol=0.02, atol=0.2)
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_and_their_gradient(ops, dtype):
    """w's and dw's rows, of which a layer has as many as channels."""
    rows, n_in, n_out, near = 150, 96, 40, 1024
    x, dy, w = _rand(1, rows, n_in, dtype=dtype), _rand(2, rows, n_out, dtype=dtype), _rand(3, n_out, n_in, dtype=dtype)
    got = []
    for ld in (near, _far(n_out, near)):
        m = Matrices(n_out, {"w": n_in, "dw": n_in}, dtype, ld, 0)
        m["w"].copy_(w)
        dx = torch.empty_like(x)
        args = [TYPES[dtype], 0, rows, n_in, n_out, dy.data_ptr(), x.data_ptr(), m.ptr("w"), 0, dx.data_ptr(),
                m.ptr("dw"), 0, n_out, n_in, m.ld, 0, n_in, m.ld, 0, 0, 0.0]
        need = ops._lib.pt_b200_linear_backward_work(ops.h, ops._LINEAR_GRAD.pack(*args))
        work = _work(need)
        args[18], args[19] = work.data_ptr(), need
        assert ops._lib.pt_b200_linear_backward(ops.h, ops._stream(), ops._LINEAR_GRAD.pack(*args)) == 0
        got.append([ops.linear(x[:n], m["w"]) for n in (3, rows)] + [dx, m["dw"].clone()])
        del m
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("dtype,rows,cols", [(torch.bfloat16, 3, 96), (torch.bfloat16, 300, 513), (torch.float32, 300, 1000),
                                             (torch.float16, 2000, 64), (torch.bfloat16, 5, 20000)])
def test_layer_norm(ops, dtype, rows, cols, shift):
    near = 4 * ((cols + 63) // 64 * 64) + 64 + (0 if shift == 0 else 8 + shift)
    x, dy, gamma = (_rand(i, *s, dtype=dtype) for i, s in ((1, (rows, cols)), (2, (rows, cols)), (3, (cols,))))
    got = []
    for ld in (near, _far(rows, near)):
        m = Matrices(rows, {"x": cols, "dy": cols, "y": cols, "dx": cols}, dtype, ld, shift)
        m["x"].copy_(x)
        m["dy"].copy_(dy)
        mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        assert ops._lib.pt_b200_layer_norm(ops.h, ops._stream(), ops._NORM.pack(
            TYPES[dtype], EPS, rows, cols, m.ptr("x"), gamma.data_ptr(), 0, m.ptr("y"), mean.data_ptr(), rstd.data_ptr(),
            m.ld, m.ld)) == 0
        dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
        need = ops._lib.pt_b200_layer_norm_backward_work(ops.h, rows, cols)
        work = _work(need)
        assert ops._lib.pt_b200_layer_norm_backward(ops.h, ops._stream(), ops._NORM_GRAD.pack(
            TYPES[dtype], 0, rows, cols, m.ptr("dy"), m.ptr("x"), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            m.ptr("dx"), dg.data_ptr(), db.data_ptr(), m.ld, m.ld, m.ld, work.data_ptr(), need)) == 0
        got.append([m["y"].clone(), m["dx"].clone(), mean, rstd, dg, db])
        del m
    assert torch.allclose(got[0][2], x.float().mean(1), atol=1e-5)
    assert all(torch.equal(p, q) for p, q in zip(*got))
