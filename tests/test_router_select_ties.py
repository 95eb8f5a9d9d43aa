"""Which logits moe_router_select tells apart: all that differ where no score is added to
anything, those whose scores differ in 64 bits otherwise."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 1500])  # a warp, and eight lanes, for a token
def test_saturated_sigmoids(moe, T):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    assert 1 / (1 + 2.718281828459045 ** -40) == 1 / (1 + 2.718281828459045 ** -41) == 1.0
    row = torch.full((16,), -5.0)
    row[2], row[3], row[9], row[10] = 40.0, 41.0, 44.0, 43.0
    l = row.expand(T, 16).contiguous().cuda()

    def ids(*args):
        return moe.moe_router_select(l, 4, *args, scoreFunc="sigmoid")[0].unique(dim=0).tolist()

    assert ids() == [[9, 10, 3, 2]]                     # by their logits
    assert ids(None, 4, 2, 1) == [[9, 10, 3, 2]]        # a group's value is one score: likewise
    assert ids(None, 4, 2, 2) == [[2, 3, 9, 10]]        # two scores are added: 1 + 1 and 1 + 1, ties
    assert ids(torch.zeros(16, device="cuda")) == [[2, 3, 9, 10]]  # a bias is added
