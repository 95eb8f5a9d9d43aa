"""The error words of the linear kernels: a moe_linear's is the library's, read and cleared by
linear_device_error; the layer with a shared expert has its own, in its workspace.  A wait
that gives up is not made to happen: the library's word is written from the host."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_shared_layer import make, run  # noqa: E402


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def record(moe, code):
    """What a wait of a moe_linear that gave up would leave behind."""
    find = moe.lib()._ZN3moe17linear_error_wordEv  # int* moe::linear_error_word()
    find.restype = ctypes.c_void_p
    v = ctypes.c_int(code)
    torch.cuda.synchronize()
    assert ctypes.CDLL("libcudart.so.12").cudaMemcpy(ctypes.c_void_p(find()), ctypes.byref(v), ctypes.c_size_t(4), 1) == 0


def test_no_cpu_device(moe):
    with pytest.raises(moe.MoeError):
        moe.linear_device_error("cpu")


@pytest.mark.gpu
def test_reads_and_clears(moe, gpu):
    for T in (4, 40, 300, 2000):
        moe.moe_linear(torch.zeros((T, 512), device="cuda").half(), torch.zeros((1024, 512), device="cuda").half())
    assert moe.linear_device_error() == 0
    record(moe, 4)
    assert moe.linear_device_error("cuda") == 4
    assert moe.linear_device_error(torch.device("cuda", 0)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 17, 130, 300])
def test_layer_has_its_own(moe, gpu, T):
    H, E, K, I, Is = 256, 16, 2, 128, 256
    p = make(moe, T, H, E, K, I, Is, T)
    want = run(moe, p, K, 1, 1, 1)
    ws = torch.full((moe.moe_shared_layer_workspace_size(T, H, E, K, I, Is),), 255, dtype=torch.uint8, device="cuda")
    record(moe, 4)
    try:
        assert torch.equal(run(moe, p, K, 1, 1, 1, workspace=ws), want)
        assert moe.device_error(ws) == 0  # not another call's error, nor what the workspace held
        assert torch.equal(run(moe, p, K, 1, 1, 1, workspace=ws), want)
        assert moe.device_error(ws) == 0
    finally:
        left = moe.linear_device_error()
    assert left == 4  # whose call it is still learns of it


@pytest.mark.gpu
def test_layer_in_a_graph_has_its_own(moe, gpu):
    T, H, E, K, I, Is = 64, 256, 16, 4, 128, 256
    p = make(moe, T, H, E, K, I, Is, 2)
    want = run(moe, p, K, 4, 2, 2)
    ws = torch.full((moe.moe_shared_layer_workspace_size(T, H, E, K, I, Is),), 255, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(moe, p, K, 4, 2, 2, y=y, workspace=ws)
    record(moe, 8)
    try:
        for _ in range(2):
            ws.fill_(255)
            y.zero_()
            g.replay()
            assert torch.equal(y, want) and moe.device_error(ws) == 0
    finally:
        left = moe.linear_device_error()
    assert left == 8
