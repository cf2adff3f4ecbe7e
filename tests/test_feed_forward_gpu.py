"""The feed-forward example: its gradients against float64 autograd of the same formula, and a
training run whose loss falls."""
import importlib.util
import os

import pytest

import pt_b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "feed_forward.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("feed_forward", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def ops():
    o = pt_b200.Operators(0)
    yield o
    o.sync()
    o.close()


def _reference(p, x, dy, act):
    """y and the gradients by torch's float64 autograd."""
    F = torch.nn.functional
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    xd = x.double().requires_grad_()
    h = F.layer_norm(xd, (x.shape[1],), q["gamma"], q["beta"], 1e-5)
    z = {"gelu": F.gelu, "relu": F.relu, "silu": F.silu}[act](F.linear(h, q["w1"], q["b1"]))
    y = xd + F.linear(z, q["w2"], q["b2"])
    grads = torch.autograd.grad(y, [xd, *q.values()], dy.double())
    return y, dict(zip(["x", *q], grads))


# Relative 2-norm errors.  fp32: each of the five chained products is good to some 2^-24 sqrt(n), a few
# 1e-6 in all.  bf16 / fp16: every intermediate (h, pre, z, dz, dpre, dh) is rounded once, errors of
# 2^-9 / 2^-12 rms each, adding up to under eight of them.
TOL = {torch.float32: 5e-6, torch.bfloat16: 8 * 2.0 ** -9, torch.float16: 8 * 2.0 ** -12}


@pytest.mark.parametrize("dtype", list(TOL), ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width,inner,act", [(1, 192, 768, "gelu"), (7, 192, 768, "gelu"),
                                                  (300, 192, 768, "silu"), (65, 129, 257, "gelu")])
def test_gradients(example, ops, dtype, rows, width, inner, act):
    layer = example.FeedForward(ops, width, inner, act, dtype)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    dy = torch.randn(rows, width, generator=gen, device="cuda").to(dtype)
    y, kept = layer.forward(x, keep=True)
    grads, dx = layer.backward(dy, kept)
    want_y, want = _reference(layer.p, x, dy, act)
    for name, got, ref in [("y", y, want_y), ("x", dx, want["x"])] + [(k, grads[k], want[k]) for k in grads]:
        err = (got.double() - ref).norm() / ref.norm()
        assert err <= TOL[dtype], (name, err.item())
    assert torch.equal(layer.forward(x), y)


@pytest.mark.parametrize("dtype", list(TOL), ids=["f32", "bf16", "f16"])
def test_training_reduces_the_loss(example, ops, dtype):
    layer, teacher = (example.FeedForward(ops, dtype=dtype, seed=s) for s in (0, 1))
    x = torch.randn(256, 192, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    losses = example.train(layer, x, teacher.forward(x), 30, rate=2.0)
    assert losses[-1] < 0.5 * losses[0], losses
