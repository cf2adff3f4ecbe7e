"""The transformer-layer operators' documented edges on the GPU: buffers shared between inputs and
outputs, and arguments that must be turned down before a launch."""
import pytest

import pt_b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@pytest.fixture(scope="module")
def ops():
    o = pt_b200.Operators(0)
    yield o
    o.sync()
    o.close()


def _randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# a few rows (one cluster adds the sums), many (a second kernel does), rows that are not aligned, and
# rows wider than the registers hold
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(6, 128), (6, 129), (300, 128), (300, 131), (3000, 1000), (700, 3001),
                                       (40, 8192), (5, 16385), (40, 20000)])
def test_norm_gradient_over_dy(ops, dtype, rows, cols):
    """dx in dy's own buffer, with the sums over dy asked for too: the bits of a dx of its own."""
    x, dy = _randn(1, rows, cols, dtype=dtype), _randn(2, rows, cols, dtype=dtype)
    gamma = _randn(3, cols, dtype=dtype)
    _, mean, rstd = ops.layer_norm(x)
    want = ops.layer_norm_backward(dy, x, gamma, mean, rstd)
    dx, dgamma, dbeta = dy.clone(), torch.empty_like(gamma), torch.empty_like(gamma)
    need = ops._lib.pt_b200_layer_norm_backward_work(ops.h, rows, cols)
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    assert ops._lib.pt_b200_layer_norm_backward(ops.h, ops._stream(), ops._NORM_GRAD.pack(
        CODES[dtype], 0, rows, cols, dx.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), cols, cols, cols, work.data_ptr(),
        need)) == 0
    for got, ref in zip((dx, dgamma, dbeta), want):
        assert torch.equal(got, ref)


def test_tensors_whose_values_are_not_in_memory(ops):
    """A negated view and a zero tensor without memory are refused, in every place of every call."""
    z = torch.view_as_complex(_randn(1, 6, 8, 2)).conj().imag[:, :1]    # one column, a stride of 16
    assert z.is_neg() and z.stride(0) == 16
    launches = pt_b200.kernel_launches()
    with pytest.raises(pt_b200.PtB200Error, match="x: is a negated view"):
        ops.linear(z, _randn(2, 4, 1))
    m, v, s = _randn(3, 6, 24), _randn(4, 24), _randn(5, 6)
    w = _randn(6, 24, 24)
    calls = [(ops.linear, dict(x=m, w=w, bias=v, residual=m)),
             (ops.linear_backward, dict(dy=m, x=m, w=w, pre=m, act="gelu")),
             (ops.layer_norm, dict(x=m, gamma=v, beta=v)),
             (ops.layer_norm_backward, dict(dy=m, x=m, gamma=v, mean=s, rstd=s))]
    for call, args in calls:
        for name, t in args.items():
            if isinstance(t, torch.Tensor):
                with pytest.raises(pt_b200.PtB200Error, match=f"{name}: is a negated view"):
                    call(**{**args, name: torch._neg_view(t)})
                with pytest.raises(pt_b200.PtB200Error, match=f"{name}: is a tensor of zeros without memory"):
                    call(**{**args, name: torch._efficientzerotensor(t.shape, device="cuda")})
    assert pt_b200.kernel_launches() == launches
