"""torch.ops.moe_b200.router_select and .linear: fake shapes on CPU, results on the GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_fake_shapes(moe):
    moe.register_torch_ops()
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.moe_b200
    with FakeTensorMode() as m:
        l = m.from_tensor(torch.empty((7, 16)))
        ids, w = ops.router_select(l, 3, None, 4, 2, 2, "sigmoid", True, 2.5)
        assert ids.shape == (7, 3) and ids.dtype == torch.int32 and w.dtype == torch.float16
        x = m.from_tensor(torch.empty((7, 64), dtype=torch.bfloat16))
        k = m.from_tensor(torch.empty((24, 64), dtype=torch.bfloat16))
        assert ops.linear(x, k).shape == (7, 24) and ops.linear(x, k).dtype == torch.bfloat16
        assert ops.linear(x, k, None, "silu", True).shape == (7, 12)
        assert ops.linear(x, k, out_dtype=torch.float32).dtype == torch.float32


@pytest.mark.gpu
def test_same_as_front_end(moe):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    moe.register_torch_ops()
    ops = torch.ops.moe_b200
    x = torch.randn((33, 64), device="cuda").half()
    w = torch.randn((48, 64), device="cuda").half()
    b = torch.randn(48, device="cuda").half()
    assert torch.equal(ops.linear(x, w, b, "silu", True), moe.moe_linear(x, w, b, "silu", True))
    l = ops.linear(x, w, out_dtype=torch.float32)
    assert torch.equal(l, moe.moe_linear(x, w, out_dtype=torch.float32))
    bias = torch.randn(48, device="cuda") * 0.1
    a = ops.router_select(l, 4, bias, 8, 4, 2, "sigmoid", True, 2.5)
    c = moe.moe_router_select(l, 4, bias, 8, 4, 2, "sigmoid", True, 2.5)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
