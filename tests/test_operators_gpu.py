"""The transformer-layer operators on the GPU against plain float64 formulas.

Tolerances are bounds, derived from the operation and not from what the kernels give.  u is the
stored type's unit roundoff, E = 2^-24 that of fp32.  A sum of n products in fp32, in any order and
with adds that may truncate, is off by at most (n + 16) 2E sum|terms|; the 16 covers operands held
as sums of parts.  An activation (slope at most 1.13) adds 16 E of its argument for its own
evaluation, and storing a value adds u times it (2^-25 where fp16 is denormal).
"""
import ctypes as C
import math

import pytest

import pt_b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

E = 2.0 ** -24
U = {torch.float32: E, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = 2.0 ** -25
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
SLOPE = 0.1
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    o = pt_b200.Operators(0)
    yield o
    o.sync()
    o.close()


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _close(got, want, bound):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert worst <= 0.0, f"error {err.max().item():.3g}, over its bound by {worst:.3g}"


def _act(p, act):
    F = torch.nn.functional
    return {"none": lambda t: t, "leaky": lambda t: F.leaky_relu(t, SLOPE), "relu": F.relu,
            "gelu": F.gelu, "silu": F.silu}[act](p)


def _dact(p, act):
    if act == "none":
        return torch.ones_like(p)
    q = p.detach().clone().requires_grad_()
    (g,) = torch.autograd.grad(_act(q, act).sum(), q)
    return g


def _linear_case(seed, dtype, rows, n_in, n_out):
    g = _gen(seed)
    x = _randn(g, rows, n_in).to(dtype)
    w = (_randn(g, n_out, n_in) / math.sqrt(n_in)).to(dtype)
    b = (0.1 * _randn(g, n_out)).to(dtype)
    r = _randn(g, rows, n_out).to(dtype)
    return x, w, b, r


def _check_linear(got, x, w, b, r, act, pre=None):
    dt = x.dtype
    xd, wd = x.double(), w.double()
    want_pre = xd @ wd.T
    mass = xd.abs() @ wd.abs().T
    if b is not None:
        want_pre, mass = want_pre + b.double(), mass + b.double().abs()
    e_pre = (x.shape[-1] + 16) * 2 * E * mass
    if pre is not None:
        _close(pre, want_pre, e_pre + U[dt] * (want_pre.abs() + e_pre) + TINY)
    y = _act(want_pre, act)
    e = 1.13 * e_pre + 16 * E * want_pre.abs()
    if r is not None:
        y = y + r.double()
        e = e + 2 * E * (y.abs() + r.double().abs())
    _close(got, y, e + U[dt] * (y.abs() + e) + TINY)


def _check_linear_backward(got, dy, x, w, pre, act):
    dt = dy.dtype
    u = U[dt] if dt != torch.float32 else 2 * E
    dx, dw, db = got
    dyd, xd, wd = dy.double(), x.double(), w.double()
    g = dyd * (_dact(pre.double(), act) if pre is not None else 1.0)
    eg = 16 * E * dyd.abs() * (1 + pre.double().abs()) if act != "none" else torch.zeros_like(g)
    round_g = u * g.abs() + eg + (TINY if dt == torch.float16 and act != "none" else 0.0)
    rows, n_out = dy.shape
    if dx is not None:
        e = (n_out + 16) * 2 * E * (g.abs() @ wd.abs()) + 1.01 * round_g @ wd.abs()
        want = g @ wd
        _close(dx, want, e + U[dt] * (want.abs() + e) + TINY)
    if dw is not None:
        e = (rows + 16) * 2 * E * (g.abs().T @ xd.abs()) + 1.01 * round_g.T @ xd.abs()
        want = g.T @ xd
        _close(dw, want, e + U[dt] * (want.abs() + e) + TINY)
    if db is not None:
        e = (rows + 16) * 2 * E * g.abs().sum(0) + eg.sum(0)
        want = g.sum(0)
        _close(db, want, e + U[dt] * (want.abs() + e) + TINY)


# one token to several tiles of tokens; widths of one, odd, under, at and over a tile
ROWS = [1, 2, 3, 5, 8, 9, 16, 17, 31, 64, 65, 127, 128, 130, 257, 600]
WIDTHS = [(1, 1), (7, 5), (16, 24), (64, 128), (65, 127), (192, 768), (193, 515), (768, 192), (1000, 40),
          (2056, 136)]
LINEAR_CASES = [(r, *WIDTHS[(3 * i + j) % len(WIDTHS)]) for i, r in enumerate(ROWS) for j in (0, 5)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,n_in,n_out", LINEAR_CASES)
def test_linear(ops, dtype, rows, n_in, n_out):
    x, w, b, r = _linear_case(rows + n_in, dtype, rows, n_in, n_out)
    act = ["none", "leaky", "relu", "gelu", "silu"][(rows + n_out) % 5]
    y, pre = ops.linear(x, w, b, residual=r, act=act, slope=SLOPE, save_pre=True)
    _check_linear(y, x, w, b, r, act, pre)
    _check_linear(ops.linear(x, w), x, w, None, None, "none")


@pytest.mark.parametrize("rows,n_in,n_out", [(40000, 64, 1), (40001, 67, 7), (30000, 3, 8), (19434, 100, 9),
                                             (19433, 129, 16), (19434, 192, 17), (9501, 130, 25), (16385, 256, 32),
                                             (9500, 1000, 4)])
def test_linear_many_rows_few_channels(ops, rows, n_in, n_out):
    x, w, b, r = _linear_case(rows + n_in, torch.float32, rows, n_in, n_out)
    y, pre = ops.linear(x, w, b, residual=r, act="silu", save_pre=True)
    _check_linear(y, x, w, b, r, "silu", pre)
    x, w, _, _ = _linear_case(rows + n_in, torch.float32, rows, n_in + 3, n_out)   # rows that are not aligned
    x, w = x[:, 1:-2], w[:, 2:-1]
    _check_linear(ops.linear(x, w), x, w, None, None, "none")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ["none", "leaky", "relu", "gelu", "silu"])
def test_linear_activations(ops, dtype, act):
    for rows in (4, 150):
        x, w, b, r = _linear_case(11, dtype, rows, 72, 200)
        w = w * 3        # arguments well into both tails
        y, pre = ops.linear(x, w, b, act=act, slope=SLOPE, save_pre=True)
        _check_linear(y, x, w, b, None, act, pre)
        _check_linear_backward(ops.linear_backward(r, x, w, pre=pre, act=act, slope=SLOPE), r, x, w, pre, act)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,n_in,n_out", LINEAR_CASES)
def test_linear_backward(ops, dtype, rows, n_in, n_out):
    x, w, b, dy = _linear_case(rows + n_out, dtype, rows, n_in, n_out)
    pre = (x.float() @ w.float().T + b.float()).to(dtype)
    act = ["gelu", "none", "silu", "relu", "leaky"][(rows + n_in) % 5]
    _check_linear_backward(ops.linear_backward(dy, x, w, pre=pre, act=act, slope=SLOPE), dy, x, w, pre, act)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_long_contraction(ops, dtype):
    """Sums over many terms: in the forward pass over the inputs, in dW over the rows."""
    x, w, b, r = _linear_case(5, dtype, 40, 9000, 136)
    _check_linear(ops.linear(x, w, b), x, w, b, None, "none")
    x, w, b, dy = _linear_case(6, dtype, 12000, 136, 72)
    _check_linear_backward(ops.linear_backward(dy, x, w), dy, x, w, None, "none")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_backward_parts(ops, dtype):
    """Each gradient alone equals the one of the whole call."""
    x, w, b, dy = _linear_case(3, dtype, 200, 72, 136)
    for act in ("none", "gelu"):
        whole = ops.linear_backward(dy, x, w, pre=dy, act=act)
        for i in range(3):
            need = dict(zip(("need_dx", "need_dw", "need_db"), (j == i for j in range(3))))
            part = ops.linear_backward(dy, x, w, pre=dy, act=act, **need)
            assert [p is not None for p in part] == list(need.values())
            assert torch.equal(part[i], whole[i])


def _strided(t, left, right):
    """t as a column slice of a wider tensor whose other columns are NaN."""
    wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), dtype=t.dtype, device="cuda")
    out = wide[:, left:left + t.shape[1]]
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("left,right", [(0, 8), (8, 8), (1, 0), (3, 2)])
@pytest.mark.parametrize("rows", [3, 150])
def test_strides_and_alignment(ops, dtype, left, right, rows):
    x, w, b, r = _linear_case(9, dtype, rows, 96, 136)
    xs, ws, rs = (_strided(t, left, right) for t in (x, w, r))
    _check_linear(ops.linear(xs, ws, b, residual=rs, act="gelu"), x, w, b, r, "gelu")
    _check_linear_backward(ops.linear_backward(rs, xs, ws, pre=rs, act="silu"), r, x, w, r, "silu")
    gamma, beta = x[0], x[1]
    y, mean, rstd = ops.layer_norm(xs, gamma, beta)
    _check_norm(y, mean, rstd, x, gamma, beta)
    _check_norm_backward(ops.layer_norm_backward(_strided(y, left, right), xs, gamma, mean, rstd), y, x,
                         gamma, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_leading_dimensions(ops, dtype):
    x, w, b, r = _linear_case(8, dtype, 30, 40, 56)
    y = ops.linear(x.view(2, 3, 5, 40), w, b, residual=r.view(2, 3, 5, 56))
    assert y.shape == (2, 3, 5, 56) and torch.equal(y.view(30, 56), ops.linear(x, w, b, residual=r))
    assert torch.equal(ops.linear(x[0], w, b), ops.linear(x[:1], w, b)[0])
    n, mean, rstd = ops.layer_norm(x.view(2, 15, 40))
    assert n.shape == (2, 15, 40) and mean.shape == rstd.shape == (2, 15)
    d = ops.layer_norm_backward(n, x.view(2, 15, 40), None, mean, rstd)
    e = ops.layer_norm_backward(n.view(30, 40), x, None, mean.view(30), rstd.view(30))
    assert d[0].shape == (2, 15, 40) and all(torch.equal(p.view(q.shape), q) for p, q in zip(d, e))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_no_rows(ops, dtype):
    x, w, b, _ = _linear_case(1, dtype, 1, 24, 40)
    e = x[:0]
    dy = torch.empty(0, 40, dtype=dtype, device="cuda")
    y, pre = ops.linear(e, w, b, act="gelu", save_pre=True)
    assert y.shape == pre.shape == (0, 40)
    dx, dw, db = ops.linear_backward(dy, e, w, pre=pre, act="gelu")
    assert dx.shape == (0, 24) and not dw.any() and not db.any() and dw.shape == (40, 24)
    n, mean, rstd = ops.layer_norm(e)
    assert n.shape == (0, 24) and mean.shape == (0,)
    dx, dg, db = ops.layer_norm_backward(n, e, None, mean, rstd)
    assert dx.shape == (0, 24) and not dg.any() and not db.any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [4, 300])
def test_not_finite_stays_in_its_row(ops, dtype, rows):
    x, w, b, r = _linear_case(21, dtype, rows, 200, 136)
    bad = x.clone()
    bad[1, 3], bad[2, 150] = float("nan"), float("inf")
    keep = [i for i in range(rows) if i not in (1, 2)]
    for act in ("none", "relu", "gelu"):
        y, z = ops.linear(bad, w, b, act=act), ops.linear(x, w, b, act=act)
        assert torch.equal(y[keep], z[keep])
        assert y[1].isnan().all()
        assert not y[2].isfinite().all()
    y, mean, rstd = ops.layer_norm(bad)
    z, _, _ = ops.layer_norm(x)
    assert torch.equal(y[keep], z[keep]) and y[1].isnan().all() and y[2].isnan().any()
    # a NaN left in the padding beside the rows is never read
    _check_linear(ops.linear(_strided(x, 3, 5), w, b), x, w, b, None, "none")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_large_and_small_magnitudes(ops, dtype):
    """Values near the type's ends: products that stay finite come out as such."""
    hi = {torch.float32: 1e18, torch.bfloat16: 1e18, torch.float16: 100.0}[dtype]
    for rows in (3, 200):
        x, w, b, r = _linear_case(23, dtype, rows, 136, 72)
        _check_linear(ops.linear(x * hi, w * hi), x * hi, w * hi, None, None, "none")
        lo = {torch.float32: 1e-15, torch.bfloat16: 1e-15, torch.float16: 1e-3}[dtype]
        _check_linear(ops.linear(x * lo, w, None), x * lo, w, None, None, "none")


def test_f32_extremes(ops):
    """The largest fp32 values as operands (their leading part must not round up to infinity)."""
    top = torch.finfo(torch.float32).max
    for rows in (2, 200):
        x = torch.zeros(rows, 96, device="cuda")
        x[:, 0] = top
        x[:, 1] = -top
        w = torch.zeros(40, 96, device="cuda")
        w[:, 0] = 0.5
        w[::2, 1] = 0.25
        y = ops.linear(x, w)
        _check_linear(y, x, w, None, None, "none")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_same_bits_again(ops, dtype):
    x, w, b, dy = _linear_case(31, dtype, 700, 264, 328)
    first = [ops.linear(x, w, b, act="gelu"), *ops.linear_backward(dy, x, w, pre=dy, act="gelu"),
             *ops.layer_norm_backward(x, x, w[0], dy[:, 0].float().clone(), dy[:, 1].float().clone())]
    for _ in range(5):
        again = [ops.linear(x, w, b, act="gelu"), *ops.linear_backward(dy, x, w, pre=dy, act="gelu"),
                 *ops.layer_norm_backward(x, x, w[0], dy[:, 0].float().clone(), dy[:, 1].float().clone())]
        assert all(torch.equal(p, q) for p, q in zip(first, again))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_runs_on_the_current_stream(ops, dtype):
    """Inputs made on a side stream are read after they are made, without a wait on the host."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x, w, b, _ = _linear_case(33, dtype, 400, 256, 256)
        for _ in range(20):
            x = ops.linear(x, w, b, act="gelu")
            x, _, _ = ops.layer_norm(x)
    s.synchronize()
    z, w, b, _ = _linear_case(33, dtype, 400, 256, 256)
    for _ in range(20):
        z = ops.linear(z, w, b, act="gelu")
        z, _, _ = ops.layer_norm(z)
        ops.sync()
    assert torch.equal(x, z)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_graph_capture(ops, dtype):
    x, w, b, dy = _linear_case(35, dtype, 300, 128, 192)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y, pre = ops.linear(x, w, b, act="gelu", save_pre=True)
        grads = ops.linear_backward(dy, x, w, pre=pre, act="gelu")
        n, mean, rstd = ops.layer_norm(y)
        ngrads = ops.layer_norm_backward(y, y, None, mean, rstd)
    x.copy_(x.flip(0))
    g.replay()
    torch.cuda.synchronize()
    want, wpre = ops.linear(x, w, b, act="gelu", save_pre=True)
    assert torch.equal(y, want)
    assert all(torch.equal(p, q) for p, q in zip(grads, ops.linear_backward(dy, x, w, pre=wpre, act="gelu")))
    wn, wm, wr = ops.layer_norm(want)
    assert torch.equal(n, wn)
    assert all(torch.equal(p, q) for p, q in zip(ngrads, ops.layer_norm_backward(want, want, None, wm, wr)))


@pytest.mark.parametrize("rows", [3, 200])
def test_offsets_over_32_bits(ops, rows):
    """Rows that start more than 2^32 bytes apart in one tensor."""
    ld = ((1 << 31) // rows // 8 + 128) * 8
    wide = torch.empty(rows, ld, dtype=torch.bfloat16, device="cuda")
    x, w, b, r = _linear_case(41, torch.bfloat16, rows, 96, 96)
    wide[:, :96] = x
    wide[:, 128:224] = r
    xs, rs = wide[:, :96], wide[:, 128:224]
    assert xs.stride(0) * (rows - 1) * 2 >= (1 << 32) - (1 << 31)
    assert torch.equal(ops.linear(xs, w, b, residual=rs), ops.linear(x, w, b, residual=r))
    assert all(torch.equal(p, q) for p, q in zip(ops.linear_backward(rs, xs, w), ops.linear_backward(r, x, w)))
    y, mean, rstd = ops.layer_norm(xs)
    assert torch.equal(y, ops.layer_norm(x)[0])
    assert all(torch.equal(p, q) for p, q in zip(ops.layer_norm_backward(rs, xs, None, mean, rstd),
                                                 ops.layer_norm_backward(r, x, None, mean, rstd)))


def test_in_place_through_the_c_entry(ops):
    """y in the residual's buffer, the norm over its own input, dx over dy."""
    for rows in (4, 260):
        x, w, b, r = _linear_case(51, torch.bfloat16, rows, 128, 128)
        want = ops.linear(x, w, b, residual=r, act="silu")
        z = r.clone()
        args = [1, 6, rows, 128, 128, x.data_ptr(), w.data_ptr(), b.data_ptr(), z.data_ptr(), z.data_ptr(),
                0, 128, 128, 128, 128, 0, 0, 0, 0.0]
        need = ops._lib.pt_b200_linear_work(ops.h, ops._LINEAR.pack(*args))
        work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        args[16], args[17] = work.data_ptr(), need
        assert ops._lib.pt_b200_linear(ops.h, ops._stream(), ops._LINEAR.pack(*args)) == 0
        assert torch.equal(z, want)
        n, mean, rstd = ops.layer_norm(x)
        z = x.clone()
        assert ops._lib.pt_b200_layer_norm(ops.h, ops._stream(), ops._NORM.pack(
            1, EPS, rows, 128, z.data_ptr(), 0, 0, z.data_ptr(), 0, 0, 128, 128)) == 0
        assert torch.equal(z, n)
        want, _, _ = ops.layer_norm_backward(r, x, None, mean, rstd)
        z = r.clone()
        assert ops._lib.pt_b200_layer_norm_backward(ops.h, ops._stream(), ops._NORM_GRAD.pack(
            1, 0, rows, 128, z.data_ptr(), x.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), z.data_ptr(),
            0, 0, 128, 128, 128, 0, 0)) == 0
        assert torch.equal(z, want)


# ------------------------------------------------------------------------------------ layer norm
def _check_norm(y, mean, rstd, x, gamma, beta, eps=EPS):
    dt, cols = x.dtype, x.shape[1]
    xd = x.double()
    m = xd.mean(1)
    v = (xd - m[:, None]).square().mean(1)
    rs = (v + eps) ** -0.5
    e_mean = (cols + 4) * E * xd.abs().mean(1)
    _close(mean, m, e_mean)
    # deviations off by e_mean + 2E(|x| + |mean|); their squares' sum by (cols + 8) E
    e_dev = (e_mean + 2 * E * (m.abs() + xd.abs().amax(1)))[:, None] * torch.ones_like(xd)
    dev = (xd - m[:, None]).abs()
    e_var = (2 * dev * e_dev + e_dev ** 2).mean(1) + (cols + 8) * E * v
    e_rs = rs * (0.5 * e_var / (v + eps) * (1 + e_var / (v + eps)) + 4 * E)
    _close(rstd, rs, e_rs)
    xhat = (xd - m[:, None]) * rs[:, None]
    e = e_dev * rs[:, None] + dev * e_rs[:, None] + e_dev * e_rs[:, None] + 2 * E * xhat.abs()
    want = xhat
    if gamma is not None:
        want, e = want * gamma.double(), e * gamma.double().abs()
    if beta is not None:
        want = want + beta.double()
    e = e + 4 * E * (want.abs() + (xhat * (gamma.double() if gamma is not None else 1)).abs())
    _close(y, want, e + U[dt] * (want.abs() + e) + TINY)


def _check_norm_backward(got, dy, x, gamma, mean, rstd):
    dt, (rows, cols) = x.dtype, x.shape
    dx, dg, db = got
    d, xd, m, rs = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    gm = gamma.double() if gamma is not None else torch.ones(cols, device="cuda", dtype=torch.float64)
    xhat, g = (xd - m) * rs, d * gm
    e_xh = 4 * E * (xd.abs() + m.abs()) * rs.abs()
    s1, s2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    e1 = (cols + 8) * E * g.abs().mean(1, keepdim=True)
    e2 = (cols + 8) * E * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    if dx is not None:
        want = rs * (g - s1 - xhat * s2)
        e = rs.abs() * (e1 + xhat.abs() * e2 + e_xh * (s2.abs() + e2)
                        + 8 * E * (g.abs() + s1.abs() + (xhat * s2).abs()))
        _close(dx, want, e + U[dt] * (want.abs() + e) + TINY)
    if dg is not None:
        want = (d * xhat).sum(0)
        e = (rows + 16) * E * (d * xhat).abs().sum(0) + (d.abs() * e_xh).sum(0)
        _close(dg, want, e + U[dt] * (want.abs() + e) + TINY)
    if db is not None:
        want = d.sum(0)
        e = (rows + 16) * E * d.abs().sum(0)
        _close(db, want, e + U[dt] * (want.abs() + e) + TINY)


NORM_CASES = [(1, 1), (3, 2), (1, 192), (5, 192), (1, 4096), (17, 33), (40, 256), (33, 257), (9, 264),
              (700, 192), (130, 512), (70, 1000), (12, 1024), (12, 1025), (12, 1032), (6, 2048), (5, 2056),
              (7, 4096), (5, 4099), (3, 8192), (3, 8200), (2, 16384), (2, 16385), (9, 20000), (3000, 64),
              (4500, 40)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", NORM_CASES)
def test_layer_norm(ops, dtype, rows, cols):
    g = _gen(rows + cols)
    x = (_randn(g, rows, cols) + 0.5).to(dtype)
    gamma, beta = (1 + 0.1 * _randn(g, cols)).to(dtype), (0.1 * _randn(g, cols)).to(dtype)
    dy = _randn(g, rows, cols).to(dtype)
    _check_norm(*ops.layer_norm(x, gamma, beta, eps=EPS), x, gamma, beta)
    y, mean, rstd = ops.layer_norm(x, eps=EPS)
    _check_norm(y, mean, rstd, x, None, None)
    _check_norm_backward(ops.layer_norm_backward(dy, x, gamma, mean, rstd), dy, x, gamma, mean, rstd)
    _check_norm_backward(ops.layer_norm_backward(dy, x, None, mean, rstd), dy, x, None, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("cols", [100, 101, 1000, 1001, 3000, 6000, 10000])
def test_layer_norm_backward_few_rows(ops, dtype, cols):
    """Around the row counts where one block, a cluster of two to eight, and many blocks take over."""
    g = _gen(cols)
    x, dy = _randn(g, 130, cols).to(dtype), _randn(g, 130, cols).to(dtype)
    gamma = _randn(g, cols).to(dtype)
    _, mean, rstd = ops.layer_norm(x)
    for rows in (1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129):
        n = slice(0, rows)
        got = ops.layer_norm_backward(dy[n], x[n], gamma, mean[n], rstd[n])
        _check_norm_backward(got, dy[n], x[n], gamma, mean[n], rstd[n])


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("cols", [3, 37, 512, 1003])
def test_layer_norm_begins_anywhere(ops, dtype, cols):
    """Tensors that begin, and whose rows lie, at any element of a 16-byte piece."""
    g = _gen(cols)
    rows, n = 41, 41 * (cols + 5) + 9
    fx, fd = _randn(g, n).to(dtype), _randn(g, n).to(dtype)
    gamma = _randn(g, cols).to(dtype)
    for begin in range(9):
        for pad in (0, 1, 5):
            ld = cols + pad
            x = fx[begin:begin + rows * ld].view(rows, ld)[:, :cols]
            dy = fd[8 - begin:8 - begin + rows * ld].view(rows, ld)[:, :cols]
            y, mean, rstd = ops.layer_norm(x, gamma, eps=EPS)
            _check_norm(y, mean, rstd, x, gamma, None)
            _check_norm_backward(ops.layer_norm_backward(dy, x, gamma, mean, rstd), dy, x, gamma, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_layer_norm_backward_parts(ops, dtype):
    for rows, cols in ((50, 200), (20, 2048), (4, 17000)):
        g = _gen(cols)
        x, dy = _randn(g, rows, cols).to(dtype), _randn(g, rows, cols).to(dtype)
        gamma = _randn(g, cols).to(dtype)
        _, mean, rstd = ops.layer_norm(x)
        whole = ops.layer_norm_backward(dy, x, gamma, mean, rstd)
        for i in range(3):
            need = dict(zip(("need_dx", "need_dgamma", "need_dbeta"), (j == i for j in range(3))))
            part = ops.layer_norm_backward(dy, x, gamma, mean, rstd, **need)
            assert [p is not None for p in part] == list(need.values())
            assert torch.equal(part[i], whole[i])


def test_layer_norm_constant_and_offset_rows(ops):
    """A row without spread (rstd is 1 / sqrt(eps)) and one whose mean is far from its spread: the
    variance is of the deviations, not a difference of large sums."""
    g = _gen(77)
    for cols in (96, 1000, 3000):
        x = _randn(g, 4, cols)
        x[0] = 3.25
        x[1] = 0.0
        x[2] = x[2] * 0.01 + 1000.0
        y, mean, rstd = ops.layer_norm(x, eps=EPS)
        _check_norm(y, mean, rstd, x, None, None)
        assert not y[1].any()


def test_gradients_against_differences(ops):
    """<gradient, v> against central differences of the float64 loss sum(y * dy) along v."""
    h, rows, n_in, n_out = 1e-4, 40, 56, 72
    x, w, b, dy = _linear_case(61, torch.float32, rows, n_in, n_out)
    for act in ("none", "gelu", "silu"):
        _, pre = ops.linear(x, w, b, act=act, save_pre=True)
        grads = ops.linear_backward(dy, x, w, pre=pre, act=act)
        base = [t.double() for t in (x, w, b)]

        def loss(t):
            return (_act(t[0] @ t[1].T + t[2], act) * dy.double()).sum()

        for i in range(3):
            v = _randn(_gen(70 + i), *base[i].shape).double()
            moved = [[t + s * h * v if j == i else t for j, t in enumerate(base)] for s in (1, -1)]
            want = ((loss(moved[0]) - loss(moved[1])) / (2 * h)).item()
            got = (grads[i].double() * v).sum().item()
            scale = (grads[i].double() * v).abs().sum().item()
            # fp32 gradients (2^-24 a term, some hundred terms) and h^2 of the third derivative
            assert abs(got - want) <= 1e-5 * scale + h * h * 10 * v.abs().sum().item(), (act, i)
    gamma = 1 + 0.1 * _randn(_gen(80), n_out)
    beta = 0.1 * _randn(_gen(81), n_out)
    z = dy * 1.5 + 0.3
    t = _randn(_gen(82), rows, n_out)
    _, mean, rstd = ops.layer_norm(z, gamma, beta, eps=EPS)
    grads = ops.layer_norm_backward(t, z, gamma, mean, rstd)
    base = [q.double() for q in (z, gamma, beta)]

    def nloss(q):
        return (torch.nn.functional.layer_norm(q[0], (n_out,), q[1], q[2], EPS) * t.double()).sum()

    for i in range(3):
        v = _randn(_gen(90 + i), *base[i].shape).double()
        moved = [[q + s * h * v if j == i else q for j, q in enumerate(base)] for s in (1, -1)]
        want = ((nloss(moved[0]) - nloss(moved[1])) / (2 * h)).item()
        got = (grads[i].double() * v).sum().item()
        scale = (grads[i].double() * v).abs().sum().item()
        assert abs(got - want) <= 1e-5 * scale + h * h * 10 * v.abs().sum().item(), i


# -------------------------------------------------------------------------------------- refusals
def test_refusals(ops):
    x, w, b, r = _linear_case(1, torch.float32, 6, 24, 40)
    Err = pt_b200.PtB200Error
    launches = pt_b200.kernel_launches()
    for call, what in [
        (lambda: ops.linear(x.double(), w.double()), "float32, bfloat16 or float16"),
        (lambda: ops.linear(x.cpu(), w.cpu()), "on cuda:0"),
        (lambda: ops.linear(x, w.cpu()), "w: needs"),
        (lambda: ops.linear(x, w.bfloat16()), "w: needs"),
        (lambda: ops.linear(x, w[:, :23]), "do not fit"),
        (lambda: ops.linear(x, w[0]), "do not fit"),
        (lambda: ops.linear(x, w, b[:39]), "bias: needs 40"),
        (lambda: ops.linear(x, w, b[::2]), "bias: needs 40"),
        (lambda: ops.linear(x, w, b, residual=r[:5]), "residual: needs 6 rows of 40"),
        (lambda: ops.linear(x, w, b, act="tanh"), "act is one of"),
        (lambda: ops.linear(x.T.contiguous().T, w), "not contiguous"),
        (lambda: ops.linear(x[:1].expand(6, 24), w), "rows overlap"),
        (lambda: ops.linear(x.as_strided((2, 2, 24), (24, 72, 1)), w), "no common row stride"),
        (lambda: ops.linear_backward(r, x, w, act="gelu"), "needs pre"),
        (lambda: ops.linear_backward(r[:5], x, w), "x: needs 5 rows"),
        (lambda: ops.linear_backward(r, x, w.T), "do not fit"),
        (lambda: ops.linear_backward(r, x, w, need_dx=False, need_dw=False, need_db=False), "nothing"),
        (lambda: ops.layer_norm(x, b[:24].bfloat16()), "gamma: needs 24"),
        (lambda: ops.layer_norm(x, b), "gamma: needs 24"),
        (lambda: ops.layer_norm(x, eps=-1.0), "eps"),
        (lambda: ops.layer_norm(x[:, :0]), "no columns"),
        (lambda: ops.layer_norm_backward(x, x, None, b[:5], b[:6]), "mean: needs 6"),
        (lambda: ops.layer_norm_backward(x, x[:5], None, b[:6], b[:6]), "x: needs 6 rows"),
        (lambda: ops.layer_norm_backward(x, x, None, b[:6], b[:6], need_dx=False, need_dgamma=False,
                                         need_dbeta=False), "nothing"),
    ]:
        with pytest.raises(Err, match=what):
            call()
    assert pt_b200.kernel_launches() == launches


def test_refusals_of_the_c_entries(ops):
    """Arguments that the host must turn down before any launch, through the C ABI itself."""
    L, h = ops._lib, ops.h
    x, w, b, r = _linear_case(1, torch.bfloat16, 6, 24, 40)
    y = torch.empty_like(r)
    launches = pt_b200.kernel_launches()

    def linear(**kw):
        a = dict(dtype=1, act=0, rows=6, n_in=24, n_out=40, x=x.data_ptr(), w=w.data_ptr(), bias=0, res=0,
                 y=y.data_ptr(), pre=0, ldx=24, ldw=24, ldr=0, ldy=40, ldp=0, work=0, nbytes=0, slope=0.0)
        a.update(kw)
        return L.pt_b200_linear(h, None, ops._LINEAR.pack(*a.values()))

    for kw in (dict(dtype=3), dict(act=3), dict(rows=-1), dict(n_in=0), dict(n_out=-4), dict(x=0), dict(w=0),
               dict(y=0), dict(ldx=23), dict(ldw=23), dict(ldy=39), dict(res=r.data_ptr(), ldr=39),
               dict(pre=y.data_ptr(), ldp=39), dict(x=x.data_ptr() + 1), dict(n_in=1 << 40)):
        assert linear(**kw) == -1, kw
        assert b"pt_b200_linear" in L.pt_b200_last_error()

    def grad(**kw):
        a = dict(dtype=1, act=5, rows=6, n_in=24, n_out=40, dy=r.data_ptr(), x=x.data_ptr(), w=w.data_ptr(),
                 pre=r.data_ptr(), dx=x.data_ptr(), dw=w.data_ptr(), db=b.data_ptr(), lddy=40, ldx=24, ldw=24,
                 ldp=40, lddx=24, lddw=24, work=0, nbytes=0, slope=0.0)
        a.update(kw)
        return L.pt_b200_linear_backward(h, None, ops._LINEAR_GRAD.pack(*a.values()))

    for kw in (dict(), dict(work=1 << 20, nbytes=64), dict(act=4), dict(dy=0), dict(pre=0), dict(lddy=3),
               dict(x=0), dict(w=0), dict(lddx=3), dict(lddw=3), dict(dx=0, dw=0, db=0), dict(rows=-1)):
        assert grad(**kw) == -1, kw
    assert b"pt_b200_linear_backward" in L.pt_b200_last_error()

    def norm(**kw):
        a = dict(dtype=1, eps=1e-5, rows=6, cols=24, x=x.data_ptr(), g=0, b=0, y=y.data_ptr(), m=0, rs=0,
                 ldx=24, ldy=24)
        a.update(kw)
        return L.pt_b200_layer_norm(h, None, ops._NORM.pack(*a.values()))

    for kw in (dict(dtype=9), dict(eps=-1.0), dict(rows=-1), dict(cols=0), dict(x=0), dict(y=0), dict(ldx=20),
               dict(ldy=20)):
        assert norm(**kw) == -1, kw

    n = 300      # rows that need workspace (a few do without)
    st, big, out = torch.zeros(n, device="cuda"), x.repeat(n // 6, 1), x.repeat(n // 6, 1)
    assert L.pt_b200_layer_norm_backward_work(h, n, 24) > 0

    def norm_grad(**kw):
        a = dict(dtype=1, res=0, rows=n, cols=24, dy=big.data_ptr(), x=big.data_ptr(), g=0, m=st.data_ptr(),
                 rs=st.data_ptr(), dx=out.data_ptr(), dg=b.data_ptr(), db=0, lddy=24, ldx=24, lddx=24, work=0,
                 nbytes=0)
        a.update(kw)
        return L.pt_b200_layer_norm_backward(h, None, ops._NORM_GRAD.pack(*a.values()))

    for kw in (dict(), dict(m=0), dict(rs=0), dict(dx=0, dg=0), dict(dy=0), dict(x=0), dict(lddx=3)):
        assert norm_grad(**kw) == -1, kw
    assert pt_b200.kernel_launches() == launches
    ops.sync()
