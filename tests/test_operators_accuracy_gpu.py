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
