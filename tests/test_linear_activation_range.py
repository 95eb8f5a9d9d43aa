"""The activations of moe_linear from one end of fp32's range to the other, within the bounds
that stand beside them (linear.cu).  In units of 2^-24 of the result: the fast exponential of a
is off by 2 + 1.173 |a| ulp = 4 + 2.35 |a| units, the fast quotient by 4, every other operation
by 1, and a rounding of a by 1 unit of a shows as |a| units.
  silu, sigmoid: a = -z exact; 1 + e and the quotient: 4 + 2.35 |z| + 1 + 4, taken as 10 + 2.4 |z|.
  gelu: a = P(t) - z^2 / 2 with |P| <= 1.27; its rounding and the exponential 3.35 |a| + 4; the
    fit 2, Horner's steps 4, t twice 5, three products: 23 + 3.35 (z^2 / 2 + 1.3), taken as
    28 + 1.7 z^2.
  gelu_tanh: a = -u, seven roundings and the exponential 9.35 |u| + 4, sum and quotient 5.
A quotient by more than 2^126 is 0: an absolute |z| 2^-126 (sigmoid: 2^-126), and 1% of it for
the roundings above."""
import pytest

torch = pytest.importorskip("torch")

from test_linear import act64  # noqa: E402

ENDS = {"silu": (-100, 90), "sigmoid": (-100, 90), "gelu": (-15, 15), "gelu_tanh": (-12, 12)}


def bound(z, act):
    a = z.abs()
    u = 1.6 * (a + 0.0447 * a ** 3)
    return {"silu": 10 + 2.4 * a, "sigmoid": 10 + 2.4 * a, "gelu": 28 + 1.7 * z * z, "gelu_tanh": 9 + 9.4 * u}[act] * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 50, 200, 2500])
@pytest.mark.parametrize("act", sorted(ENDS))
def test_whole_range(moe, act, T):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    K = 64
    w = torch.eye(K, device="cuda").half()
    lo, hi = ENDS[act]
    near = {"silu": (-88.5, -86), "sigmoid": (-88.5, -86), "gelu": (-13.4, -12.9), "gelu_tanh": (-10.5, -10.1)}[act]
    for first, last in ((lo, hi), near, (-1, 1)):
        x = torch.linspace(first, last, T * K, device="cuda").view(T, K).half()
        y = moe.moe_linear(x, w, activation=act, out_dtype=torch.float32).double()
        z = x.double()
        want = act64(z, act)
        flush = 1.01 * 2.0 ** -126 * (1 if act == "sigmoid" else z.abs())
        off = (y - want).abs() - bound(z, act) * want.abs() - flush
        assert (off <= 0).all(), (act, T, z.flatten()[off.argmax()].item())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 300])
def test_past_the_range(moe, T):
    """Where exp is 0 or infinite: 0 or z, no NaN."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    z = torch.tensor([-65504.0, 65504.0, -1000.0, 1000.0, 0.0, -200.0, 200.0, -0.0], device="cuda").half()
    x = z.expand(T, 8).contiguous()
    w = torch.eye(8, device="cuda").half()
    for act in ("silu", "gelu", "gelu_tanh"):
        y = moe.moe_linear(x, w, activation=act, out_dtype=torch.float32)
        assert torch.equal(y, x.float().clamp_min(0)), act
    y = moe.moe_linear(x, w, activation="sigmoid", out_dtype=torch.float32)
    assert torch.equal(y, (x.float().sign() + 1) / 2)
