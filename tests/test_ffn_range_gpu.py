"""Gates far from zero in the feed-forward block, element by element.

With one token, x and dy of ones and an identity Wd, the gradients show what the epilogue computed for
each element: dwg's columns are dg = dh u act'(g), dwu's are du = dh act(g), dwd's rows are h = act(g) u.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan  # noqa: E402

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
