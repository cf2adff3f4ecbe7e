"""How near the transformer-layer operators come to float64 where their sums or their operands are
extreme.  u is the stored type's unit roundoff."""
import math

import pytest

import pt_b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def ops():
    o = pt_b200.Operators(0)
    yield o
    o.sync()
    o.close()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _positive(seed, n, k, dtype):
    """[n][k] of values between a half and two, each row with a scale of its own (so that what comes of
    them is spread over the type's roundings)."""
    g = _gen(seed)
    t = 0.5 + 0.5 * torch.rand(n, k, generator=g, device="cuda")
    return (t * (1 + torch.rand(n, 1, generator=g, device="cuda"))).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("which", ["forward", "dw"])
def test_long_sums_of_one_sign_are_not_biased(ops, dtype, which):
    """The tensor core truncates each addition, so an accumulator of one sign loses up to 2^-23 of itself
    with every 16 of k.  One that takes 4096 of k at most loses 256 x 2^-24 on average or less; the mean
    over n outputs of their own rounding (under u each) is under 6 u / sqrt n."""
    n, k = 256, 1 << (18 if which == "forward" else 20)
    a, b = _positive(1, n, k, dtype), _positive(2, n, k, dtype)
    b = b * 2.0 ** -(k.bit_length() - 5)     # sums of some 30, within fp16
    if which == "forward":
        got = ops.linear(a, b)
        want = a.double() @ b.double().T
    else:
        a, b = a.T.contiguous(), b.T.contiguous()
        _, got, _ = ops.linear_backward(a, b, b[:n], need_dx=False, need_db=False)
        want = a.double().T @ b.double()
    off = ((got.double() - want) / want).mean().abs().item()
    assert off <= 256 * 2.0 ** -24 + 6 * U[dtype] / n, off


def _norm_error(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def _products(ops, x, w, dy):
    """The three products of a layer with their exact values and their lengths."""
    dx, dw, _ = ops.linear_backward(dy, x, w)
    xd, wd, dd = x.double(), w.double(), dy.double()
    return [("y", ops.linear(x, w), xd @ wd.T, x.shape[1]), ("dx", dx, dd @ wd, w.shape[0]),
            ("dw", dw, dd.T @ xd, x.shape[0])]


SHAPES = [(600, 768, 192), (300, 2056, 136), (257, 193, 515), (40, 9000, 136), (3616, 192, 768), (4, 4096, 1024),
          (9500, 130, 25)]


def _bound(k):
    """Relative 2-norm error of an fp32 product of k random terms: a chunk of 64 ends in four truncating
    additions (under 2^-23 each of what is there, half of that on average), k / 64 chunks are added with
    rounding to nearest, whose errors add up as a random walk does, and the terms' own errors (the products
    left out, the third planes' rounding) are under 2^-24 and as random as the terms."""
    return (4 + math.sqrt(k / 64)) * 2.0 ** -24


@pytest.mark.parametrize("rows,n_in,n_out", SHAPES)
def test_f32_products_hold_all_their_bits(ops, rows, n_in, n_out):
    g = _gen(rows)
    x, w, dy = _randn(g, rows, n_in), _randn(g, n_out, n_in), _randn(g, rows, n_out)
    for name, got, want, k in _products(ops, x, w, dy):
        assert _norm_error(got, want) <= _bound(k), name


# x dy and w scales that leave every product a normal number; 1.2e-38 is the smallest normal number, so some of
# the values themselves are denormal there
@pytest.mark.parametrize("sx,sw", [(1e-30, 1.0), (1e-34, 1.0), (1e-36, 10.0), (2e-38, 1000.0), (1e-18, 1e-17),
                                   (1.0, 1e-36), (1e30, 1e-34)])
@pytest.mark.parametrize("rows", [4, 600])
def test_f32_products_of_small_operands(ops, rows, sx, sw):
    g = _gen(7)
    x, w, dy = sx * _randn(g, rows, 192), sw * _randn(g, 256, 192), _randn(g, rows, 256)
    for name, got, want, k in _products(ops, x, w, dy):
        assert _norm_error(got, want) <= _bound(k), name
    for name, got, want, k in _products(ops, _randn(g, rows, 192), w, sx * dy):
        assert _norm_error(got, want) <= _bound(k), name


def test_bf16_products_of_small_operands(ops):
    """Rounded once, so under u of every output; normal numbers throughout."""
    g = _gen(8)
    for rows in (4, 600):
        x, w = (1e-30 * _randn(g, rows, 192)).bfloat16(), _randn(g, 256, 192).bfloat16()
        dy = _randn(g, rows, 256).bfloat16()
        for name, got, want, k in _products(ops, x, w, dy):
            assert _norm_error(got, want) <= U[torch.bfloat16], name


# x0 w0 + x1 w1: what is left of two terms that all but cancel lies in the product of two of the three parts
# (8 bits each) that an operand has; every step is exact
@pytest.mark.parametrize("x0,w0,x1,w1,want", [
    (1 + 2.0 ** -20, 1, -1, 1, 2.0 ** -20), (1, 1 + 2.0 ** -20, -1, 1, 2.0 ** -20),
    (1 + 2.0 ** -10, 1, -1, 1, 2.0 ** -10), (1, 1 + 2.0 ** -10, -1, 1, 2.0 ** -10),
    (1 + 2.0 ** -10, 1 + 2.0 ** -10, -1, 1 + 2.0 ** -9, 2.0 ** -20), (1, 1, 1, -0.5, 0.5)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -118, 2.0 ** 100])
def test_f32_terms_that_cancel(ops, x0, w0, x1, w1, want, scale):
    for rows, at in ((4, 1), (300, 1), (300, 15), (300, 63), (300, 150)):   # one MMA, one chunk, two chunks
        x, w = torch.zeros(rows, 192, device="cuda"), torch.zeros(200, 192, device="cuda")
        x[:, 0], x[:, at], w[:, 0], w[:, at] = x0 * scale, x1 * scale, w0, w1
        assert (ops.linear(x, w) == want * scale).all()
        dx, _, _ = ops.linear_backward(x, torch.zeros(rows, 200, device="cuda"), w.T.contiguous())
        assert (dx == want * scale).all()


def test_gelu_value_and_slope(ops):
    """E is fp32's unit roundoff.  h = Phi(-|p|) comes from a fit good to 1.1e-8 and to 1.1e-6 of h, an exponential
    whose argument carries three roundings (1.5 p^2 E of h), and some sixteen E for the exponential, the
    reciprocal and the arithmetic; 1 - h rounds once more.  Below 1e-37 the exponential ends."""
    e = 2.0 ** -24
    p = torch.linspace(-14, 14, 700001, device="cuda", dtype=torch.float64).float()
    p = torch.cat([p, torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30, 20.0, -20.0, 100.0, -100.0], device="cuda")])
    p = torch.cat([p, 3 * _randn(_gen(5), 300000)])[:, None]
    pd = p.double()
    h, phi = 0.5 * torch.erfc(pd.abs() * math.sqrt(0.5)), torch.exp(-0.5 * pd * pd) / math.sqrt(2 * math.pi)
    cdf = torch.where(pd < 0, h, 1 - h)
    e_exp = (1.5 * pd * pd + 16) * e
    e_cdf = torch.minimum(torch.full_like(h, 1.1e-8), 1.1e-6 * h) + h * e_exp + torch.where(pd < 0, 0.0, e / 2) + 1e-37
    one = torch.ones(1, 1, device="cuda")
    y, pre = ops.linear(p, one, act="gelu", save_pre=True)
    assert torch.equal(pre, p)
    value = pd * cdf
    over = ((y.double() - value).abs() - pd.abs() * e_cdf - e * value.abs()).max().item()
    assert over <= 0, over
    slope = cdf + pd * phi
    dx, _, _ = ops.linear_backward(torch.ones_like(p), p, one, pre=p, act="gelu")
    e_slope = e_cdf + (pd * phi).abs() * e_exp + pd.abs() * 1e-37 + 2 * e * (cdf + (pd * phi).abs())
    over = ((dx.double() - slope).abs() - e_slope).max().item()
    assert over <= 0, over
    n = _randn(_gen(6), 1 << 20, 1)
    off = (ops.linear(n, one, act="gelu").double() - torch.nn.functional.gelu(n.double())).square().mean().sqrt().item()
    assert off <= 3e-8, off     # half a rounding of values of about one


@pytest.mark.parametrize("which", ["alone", "whole"])
def test_f32_bias_gradient(ops, which):
    """A chain of n fp32 additions of random terms of equal size has a relative error of E sqrt((n + 1) / 6).  The
    sum over 3616 rows of 192 columns is one of eight rows in a block, of 452 blocks' sums over eight lanes and
    four turns (15), of those four in pairs (two levels), and of the eight lanes."""
    g = _gen(9)
    x, w, dy = _randn(g, 3616, 768), _randn(g, 192, 768), _randn(g, 3616, 192)
    alone = dict(need_dx=False, need_dw=False) if which == "alone" else {}
    db = ops.linear_backward(dy, x, w, **alone)[2]
    assert _norm_error(db, dy.double().sum(0)) <= 2.0 ** -24 * math.sqrt((9 + 16 + 3 + 9) / 6)
