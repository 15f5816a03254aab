"""Gates far from zero in the feed-forward block, element by element.

With one token, x and dy of ones and an identity Wd, the gradients show what the epilogue computed for
each element: dwg's columns are dg = dh u act'(g), dwu's are du = dh act(g), dwd's rows are h = act(g) u.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan  # noqa: E402
import test_ffn_gpu as block  # noqa: E402

ACTS = ["silu", "gelu", "gelu_tanh"]


def elements(act, g, u, dh=1.0):
    """dg, du and h of the gates g with the values u, and dh everywhere."""
    n, dtype = g.numel(), g.dtype
    one = torch.ones(1, n, dtype=dtype, device="cuda")
    eye = torch.eye(n, dtype=dtype, device="cuda")
    plan = GatedFfnPlan(1, n, n, dtype=dtype, activation=act, training=True)
    out = [torch.empty_like(one)] + [torch.empty_like(eye) for _ in range(3)]
    plan.backward(one, eye, eye, eye * dh, g.view(1, n), u.view(1, n), one, *out)
    plan.check_status()
    plan.destroy()
    dwg, dwu, dwd = out[1:]
    assert all(torch.equal(t, t[:, :1].expand(n, n)) or t.isnan().any() for t in (dwg, dwu))
    return dwg[:, 0], dwu[:, 0], dwd[0]


def exact_act(act, v):
    """act and slope in 64 bits without the cancellation that the test looks for."""
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-v * 0.5 ** 0.5)
        return v * p, p + v * torch.exp(-0.5 * v * v) * (2 * torch.pi) ** -0.5
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * torch.sigmoid(-v))
    c = (2 / torch.pi) ** 0.5
    z = 2 * c * (v + 0.044715 * v ** 3)
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    return v * p, p + 2 * c * v * p * q * (1 + 3 * 0.044715 * v * v)


@pytest.mark.parametrize("act", ACTS)
def test_gates_at_the_end_of_the_type(act):
    """Up to the largest bf16: the slope is one or zero there, and act(g) is g or zero."""
    top = torch.finfo(torch.bfloat16).max
    g = torch.tensor([s * v for v in (1e30, 1e38, 2.2e38, 3e38, top) for s in (1, -1)], device="cuda").bfloat16()
    u = torch.full_like(g, 2.0 ** -10)
    dg, du, h = elements(act, g, u, dh=2.0 ** -8)
    zero = torch.zeros_like(g)
    on = g > 0
    # powers of two: every product is exact
    assert torch.equal(dg, torch.where(on, u * 2.0 ** -8, zero))
    assert torch.equal(du.abs(), torch.where(on, g * 2.0 ** -8, zero))
    assert torch.equal(h.abs(), torch.where(on, g * 2.0 ** -10, zero))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,lowest,dh", [(torch.bfloat16, -12.0, 1.0), (torch.float16, -5.5, 1024.0)])
def test_negative_gates_keep_their_digits(act, dtype, lowest, dh):
    """act(g) and its slope fall off like exp(-g^2 / 2) or exp(g) there, and no difference of larger
    numbers may stand in for them. Relative errors in fp32: the exponential 2 + 1.2 |z| steps of 2^-23 for
    an argument z, its argument 4 half steps times |z|; |z| is up to 67 where the value is above the
    smallest normal number, which makes 1e-5 + 1.6e-5. The factor beside gelu's exponential: 5e-7. The
    slope's two terms have opposite signs and differ by a factor of 3 at least, so that their errors come
    to twice as much: under 2^-13. Then one rounding to the type. The factor act(g) / g counts as zero
    under 2^-126."""
    g = torch.linspace(lowest, -4.0, 97, device="cuda").to(dtype)
    u = torch.full_like(g, 1.5)
    dg, du, h = elements(act, g, u, dh)
    a, slope = exact_act(act, g.double())
    small = 2.0 ** -126 * (1 + g.double().abs()) ** 4 * dh * 1.5 + block.tiny(dtype)
    rel = block.half_step(dtype) + 2.0 ** -13
    for name, got, want in (("dg", dg, dh * 1.5 * slope), ("du", du, dh * a), ("h", h, 1.5 * a)):
        block.within(got, want, rel * want.abs() + small, name)
    # the forward pass: y = act(x) x
    n = g.numel()
    eye = torch.eye(n, dtype=dtype, device="cuda") * (dh if dtype == torch.float16 else 1)
    plan = GatedFfnPlan(1, n, n, dtype=dtype, activation=act)
    y = torch.empty(1, n, dtype=dtype, device="cuda")
    one = torch.eye(n, dtype=dtype, device="cuda")
    plan.forward(g.view(1, n), one, one, eye, y)
    plan.check_status()
    plan.destroy()
    scale = float(eye[0, 0])
    want = scale * a * g.double()
    # h is rounded to the type before it meets Wd (a power of two)
    block.within(y[0], want, rel * want.abs() + scale * 12 * small, "y")


@pytest.mark.parametrize("act", ACTS)
def test_a_closed_gate_passes_nothing_however_large_the_rest(act):
    """dh u is beyond fp32 here, but the slope it is multiplied by is zero to 1e-80."""
    g = torch.full((40,), -200.0, device="cuda").bfloat16()
    dg, du, h = elements(act, g, torch.full_like(g, 1e30), dh=1e20)
    assert all(bool((t == 0).all()) for t in (dg, du, h))
