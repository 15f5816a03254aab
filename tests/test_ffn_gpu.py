"""The gated feed-forward block through its public plan, against the definition in 64 bits.

Tolerances are element-wise bounds built from the roundings the operator documents (u = half a
step of the operand type, finfo.eps / 2):
  * a sum of K products in the tensor core: each instruction adds 16 of them and truncates the
    fp32 accumulator, (K / 16 + 20) 2^-23 of the sum of the magnitudes;
  * the activation and its slope in fp32: the fast exponential's relative error grows with its
    argument, 2^-21 (1 + |v|), and the slope is a sum of terms up to 1 + |v|;
  * h, dg and du are rounded to the operand type (u), the results once more (u);
  * fp16 values below the normal range are off by up to half the smallest subnormal.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import _lib  # noqa: E402
from mlir_roller_b200.ffn import GatedFfnPlan  # noqa: E402

DTYPES = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh"]
# tokens, d_model, d_ff: one element, less than a k-block, odd widths, around the tile edges, a
# reduction worth splitting, several tiles each way
SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (7, 100, 33), (8, 128, 200), (33, 264, 1000), (120, 1024, 512),
          (121, 65, 129), (128, 256, 384), (129, 257, 255), (200, 72, 520), (300, 512, 1000), (513, 640, 328)]


def act64(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))


def slope64(name, v):
    if name == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 + v * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133


def acc(k):
    return (k / 16 + 20) * 2.0 ** -23


def make(tokens, d, f, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, s=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * s).to(dtype)

    return {"x": normal(tokens, d, s=scale), "wg": normal(f, d, s=2 * d ** -0.5), "wu": normal(f, d, s=d ** -0.5),
            "wd": normal(d, f, s=f ** -0.5), "dy": normal(tokens, d, s=0.5)}


def guarded(rows, cols, dtype, pad_rows=2, pad_cols=5, lead=0):
    """A rows x cols view inside a larger buffer filled with a value that no result takes."""
    buf = torch.full((rows + pad_rows, lead + cols + pad_cols), 777.0, dtype=dtype, device="cuda")
    return buf, buf[:rows, lead:lead + cols]


def untouched(buf, rows, cols, lead=0):
    out = buf.clone()
    out[:rows, lead:lead + cols] = 777.0
    return bool((out == 777.0).all())


def within(got, want, bound, what):
    diff = (got.double() - want).abs()
    bad = ~(diff <= bound)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got "
                             f"{got[tuple(i)].item()}, want {want[tuple(i)].item()}, bound {bound[tuple(i)].item()}")


def forward_bounds(s, act, dtype):
    """(y, g, u) in 64 bits and how far each may be off."""
    u_ = half_step(dtype)
    x, wg, wu, wd = (s[k].double() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.T, x @ wu.T
    eg, eu = acc(x.shape[1]) * (x.abs() @ wg.abs().T), acc(x.shape[1]) * (x.abs() @ wu.abs().T)
    a = act64(act, g)
    h = a * u
    ea = 1.2 * eg + 2.0 ** -21 * (1 + g.abs()) * a.abs()
    eh = ea * u.abs() + (a.abs() + ea) * eu
    eh = eh + u_ * (h.abs() + eh) + tiny(dtype)
    y = h @ wd.T
    ey = eh @ wd.abs().T + acc(h.shape[1]) * ((h.abs() + eh) @ wd.abs().T)

    def rounded(v, e):
        return e + u_ * (v.abs() + e) + tiny(dtype)

    return {"y": (y, rounded(y, ey)), "g": (g, rounded(g, eg)), "u": (u, rounded(u, eu))}


def backward_bounds(s, act, dtype):
    u_ = half_step(dtype)
    x, wg, wu, wd, g, u, dy = (s[k].double() for k in ("x", "wg", "wu", "wd", "g", "u", "dy"))
    tokens, d = x.shape
    f = wg.shape[0]
    a, b = act64(act, g), slope64(act, g)
    dh = dy @ wd
    edh = acc(d) * (dy.abs() @ wd.abs())
    fast = 2.0 ** -20 * (1 + g.abs()) ** 2          # act and slope: sums of terms up to 1 + |v|
    out = {}

    def product(value, error):                      # rounded to the operand type
        return value, error + u_ * (value.abs() + error) + tiny(dtype)

    dg, edg = product(dh * u * b, edh * (u * b).abs() + (dh.abs() + edh) * u.abs() * fast)
    du, edu = product(dh * a, edh * a.abs() + (dh.abs() + edh) * fast)
    h, eh = product(a * u, u.abs() * fast)

    def result(name, value, error):
        out[name] = (value, error + u_ * (value.abs() + error) + tiny(dtype))

    result("dx", dg @ wg + du @ wu,
           edg @ wg.abs() + edu @ wu.abs() + acc(2 * f) * ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()))
    result("dwg", dg.T @ x, edg.T @ x.abs() + acc(tokens) * ((dg.abs() + edg).T @ x.abs()))
    result("dwu", du.T @ x, edu.T @ x.abs() + acc(tokens) * ((du.abs() + edu).T @ x.abs()))
    result("dwd", dy.T @ h, dy.abs().T @ eh + acc(tokens) * (dy.abs().T @ (h.abs() + eh)))
    return out


def run_forward(s, act, dtype, save=True, max_tokens=None, plan=None):
    tokens, d = s["x"].shape
    f = s["wg"].shape[0]
    own = plan is None
    plan = plan or GatedFfnPlan(max_tokens or max(tokens, 1), d, f, dtype=dtype, activation=act)
    y = torch.empty(tokens, d, dtype=dtype, device="cuda")
    g, u = plan.new_saved(tokens) if save else (None, None)
    plan.forward(s["x"], s["wg"], s["wu"], s["wd"], y, g, u)
    plan.check_status()
    if own:
        plan.destroy()
    return y, g, u


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act,dtype", [("silu", torch.bfloat16), ("gelu", torch.float16), ("gelu_tanh", torch.bfloat16)])
def test_forward(shape, act, dtype):
    s = make(*shape, dtype, seed=1)
    want = forward_bounds(s, act, dtype)
    y, g, u = run_forward(s, act, dtype)
    within(g, *want["g"], "g")
    within(u, *want["u"], "u")
    within(y, *want["y"], "y")
    # without g and u the same y, bit for bit
    assert torch.equal(run_forward(s, act, dtype, save=False)[0], y)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_activation_and_type_over_a_wide_range(act, dtype):
    """Gates from far below zero to far above, where the exponentials run out of range."""
    s = make(64, 128, 256, dtype, seed=2, scale=30.0)
    want = forward_bounds(s, act, dtype)
    assert want["g"][0].abs().max() > 90
    y, g, u = run_forward(s, act, dtype)
    within(y, *want["y"], "y")


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 64, 64), (3, 5, 7), (7, 100, 33), (33, 264, 1000), (129, 257, 255),
                                   (200, 72, 520), (300, 512, 1000), (513, 640, 328), (65, 1024, 128)])
@pytest.mark.parametrize("act,dtype", [("silu", torch.bfloat16), ("gelu", torch.float16), ("gelu_tanh", torch.float16)])
def test_backward(shape, act, dtype):
    s = make(*shape, dtype, seed=3)
    tokens, d, f = shape
    plan = GatedFfnPlan(tokens, d, f, dtype=dtype, activation=act, training=True)
    y, s["g"], s["u"] = run_forward(s, act, dtype, plan=plan)
    outs = {k: torch.empty_like(s[v]) for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))}
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], **outs)
    plan.check_status()
    for name, (want, bound) in backward_bounds(s, act, dtype).items():
        within(outs[name], want, bound, name)
    plan.destroy()


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """The gradients against central differences of the block in 64 bits, along one direction for
    each operand: L = sum(dy * y). Besides the element-wise bounds of the gradients (summed along the
    direction) the saved g and u are rounded, which moves the slope's argument by u |g|, and the
    difference quotient is off by its step squared."""
    dtype = torch.float16
    tokens, d, f = 40, 48, 72
    s = make(tokens, d, f, dtype, seed=4)
    plan = GatedFfnPlan(tokens, d, f, dtype=dtype, activation=act, training=True)
    y, s["g"], s["u"] = run_forward(s, act, dtype, plan=plan)
    outs = {k: torch.empty_like(s[v]) for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))}
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], **outs)
    plan.check_status()

    def loss(x, wg, wu, wd):
        return (s["dy"].double() * ((act64(act, x @ wg.T) * (x @ wu.T)) @ wd.T)).sum()

    base = {k: s[k].double() for k in ("x", "wg", "wu", "wd")}
    bounds = backward_bounds(s, act, dtype)
    exact = dict(base, g=base["x"] @ base["wg"].T, u=base["x"] @ base["wu"].T, dy=s["dy"].double())
    unrounded = backward_bounds(exact, act, dtype)
    gen = torch.Generator(device="cuda").manual_seed(5)
    step = 1e-5
    for name, key in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd")):
        v = torch.randn(base[key].shape, generator=gen, device="cuda", dtype=torch.float64)
        up, down = dict(base), dict(base)
        up[key], down[key] = base[key] + step * v, base[key] - step * v
        slope = (loss(**up) - loss(**down)) / (2 * step)
        from_saved = (bounds[name][0] - unrounded[name][0]).abs()   # what rounding g and u moves
        tol = ((bounds[name][1] + from_saved) * v.abs()).sum() + 1e-6 * (1 + slope.abs())
        assert (outs[name].double() * v).sum().sub(slope).abs() <= tol, name
    plan.destroy()


@pytest.mark.parametrize("lead", [0, 3])
@pytest.mark.parametrize("tokens,d,f", [(50, 64, 96), (130, 72, 200), (20, 33, 47)])
def test_strided_operands_and_untouched_surroundings(tokens, d, f, lead):
    """Every operand a view into a wider buffer (its rows starting on odd addresses with lead = 3): the
    same results as from contiguous ones, and nothing else in the outputs' buffers changes."""
    dtype = torch.bfloat16
    s = make(tokens, d, f, dtype, seed=6)
    plan = GatedFfnPlan(tokens + 9, d, f, dtype=dtype, training=True)
    y, g, u = run_forward(s, "silu", dtype, plan=plan)
    outs = [torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd")]
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], g, u, s["dy"], *outs)
    v, bufs = {}, {}
    for k, t in {**s, "g": g, "u": u, "y": y, "dx": s["x"], "dwg": s["wg"], "dwu": s["wu"], "dwd": s["wd"]}.items():
        bufs[k], v[k] = guarded(*t.shape, dtype, lead=lead)
    for k in ("x", "wg", "wu", "wd", "dy"):
        v[k].copy_(s[k])
    plan.forward(v["x"], v["wg"], v["wu"], v["wd"], v["y"], v["g"], v["u"])
    plan.backward(v["x"], v["wg"], v["wu"], v["wd"], v["g"], v["u"], v["dy"], v["dx"], v["dwg"], v["dwu"], v["dwd"])
    plan.check_status()
    for k, want in (("y", y), ("g", g), ("u", u), ("dx", outs[0]), ("dwg", outs[1]), ("dwu", outs[2]), ("dwd", outs[3])):
        assert torch.equal(v[k], want), k
        assert untouched(bufs[k], *want.shape, lead=lead), k
    plan.destroy()


def test_no_tokens():
    plan = GatedFfnPlan(4, 40, 24, training=True)
    s = make(4, 40, 24, torch.bfloat16, seed=7)
    e = {k: s[k][:0] for k in ("x", "dy")}
    y = torch.empty_like(e["x"])
    g, u = plan.new_saved(0)
    plan.forward(e["x"], s["wg"], s["wu"], s["wd"], y, g, u)
    grads = {k: torch.full_like(s[v], 5.0) for k, v in (("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))}
    plan.backward(e["x"], s["wg"], s["wu"], s["wd"], g, u, e["dy"], torch.empty_like(e["x"]), **grads)
    plan.check_status()
    assert all(bool((t == 0).all()) for t in grads.values())
    plan.destroy()


def test_fewer_tokens_than_the_plan_holds():
    """One plan, calls of different lengths: nothing of a longer call shows in a shorter one."""
    dtype = torch.bfloat16
    plan = GatedFfnPlan(700, 136, 200, dtype=dtype, training=True)
    for i, tokens in enumerate((700, 3, 257, 1, 64)):
        s = make(tokens, 136, 200, dtype, seed=20 + i)
        y, s["g"], s["u"] = run_forward(s, "silu", dtype, plan=plan)
        within(y, *forward_bounds(s, "silu", dtype)["y"], "y")
        outs = {k: torch.empty_like(s[v]) for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))}
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], **outs)
        plan.check_status()
        for name, (want, bound) in backward_bounds(s, "silu", dtype).items():
            within(outs[name], want, bound, name)
    plan.destroy()


@pytest.mark.parametrize("tokens", [5, 200])
def test_a_token_that_is_not_finite_stays_by_itself(tokens):
    dtype = torch.bfloat16
    s = make(tokens, 256, 320, dtype, seed=8)
    plan = GatedFfnPlan(tokens, 256, 320, dtype=dtype)
    y0, g0, u0 = run_forward(s, "silu", dtype, plan=plan)
    s["x"][2, 7] = float("nan")
    s["x"][4, 3] = float("inf")
    y, g, u = run_forward(s, "silu", dtype, plan=plan)
    rest = [i for i in range(tokens) if i not in (2, 4)]
    assert torch.equal(y[rest], y0[rest]) and torch.equal(g[rest], g0[rest]) and torch.equal(u[rest], u0[rest])
    assert y[2].isnan().all() and not y[4].isfinite().any()
    plan.destroy()


def test_split_reductions_repeat_bit_for_bit():
    """Few tokens and long reductions are cut into parts; their order of arrival must not show."""
    dtype = torch.bfloat16
    s = make(20, 2048, 1024, dtype, seed=9)
    plan = GatedFfnPlan(20, 2048, 1024, dtype=dtype)
    first = run_forward(s, "gelu", dtype, plan=plan)
    for _ in range(20):
        again = run_forward(s, "gelu", dtype, plan=plan)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    plan.destroy()


def test_on_a_side_stream_and_in_a_graph():
    dtype = torch.bfloat16
    s = make(96, 256, 512, dtype, seed=10)
    plan = GatedFfnPlan(96, 256, 512, dtype=dtype, training=True)
    y, g, u = run_forward(s, "silu", dtype, plan=plan)
    outs = [torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd")]
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], g, u, s["dy"], *outs)
    torch.cuda.synchronize()
    ys, gs, us = torch.empty_like(y), torch.empty_like(g), torch.empty_like(u)
    again = [torch.zeros_like(t) for t in outs]
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.forward(s["x"], s["wg"], s["wu"], s["wd"], ys, gs, us)
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], gs, us, s["dy"], *again)
    fresh = make(96, 256, 512, dtype, seed=11)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ys, y) and all(torch.equal(a, b) for a, b in zip(again, outs))
    # new contents at the same addresses
    s["x"].copy_(fresh["x"])
    s["dy"].copy_(fresh["dy"])
    graph.replay()
    torch.cuda.synchronize()
    y2, g2, u2 = run_forward(s, "silu", dtype, plan=plan)
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], g2, u2, s["dy"], *outs)
    plan.check_status()
    assert torch.equal(ys, y2) and all(torch.equal(a, b) for a, b in zip(again, outs))
    with torch.cuda.stream(stream):
        plan.forward(s["x"], s["wg"], s["wu"], s["wd"], ys.zero_())
    stream.synchronize()
    assert torch.equal(ys, y2)
    plan.check_status()
    plan.destroy()


def test_capture_refuses_to_allocate():
    """An unaligned view the plan has no copy for yet: refused while capturing, fine afterwards."""
    dtype = torch.bfloat16
    s = make(8, 64, 64, dtype, seed=12)
    plan = GatedFfnPlan(8, 64, 64, dtype=dtype)
    wide = torch.zeros(8, 67, dtype=dtype, device="cuda")
    x = wide[:, 3:]
    x.copy_(s["x"])
    y = torch.empty_like(s["x"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(_lib.RollerError) as e:
            plan.forward(x, s["wg"], s["wu"], s["wd"], y)
        assert e.value.status == _lib.ERR_UNSUPPORTED
    plan.forward(x, s["wg"], s["wu"], s["wd"], y)
    want = run_forward(s, "silu", dtype, save=False, plan=plan)[0]
    assert torch.equal(y, want)
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        plan.forward(x, s["wg"], s["wu"], s["wd"], y.zero_())
    graph.replay()
    plan.check_status()
    assert torch.equal(y, want)
    plan.destroy()


def test_refusals():
    with pytest.raises(TypeError):
        GatedFfnPlan(4, 8, 8, dtype=torch.float32)
    with pytest.raises(ValueError):
        GatedFfnPlan(4, 8, 8, activation="relu")
    for bad in ((0, 8, 8), (4, 0, 8), (4, 8, 0), ((1 << 20) + 1, 8, 8)):
        with pytest.raises(_lib.RollerError) as e:
            GatedFfnPlan(*bad)
        assert e.value.status == _lib.ERR_INVALID
    plan = GatedFfnPlan(8, 16, 24)
    s = make(8, 16, 24, torch.bfloat16, seed=13)
    y = torch.empty_like(s["x"])
    w = (s["wg"], s["wu"], s["wd"])
    g, u = plan.new_saved(8)
    with pytest.raises(ValueError):
        plan.forward(s["x"], *w, y, g)                               # u missing
    with pytest.raises(TypeError):
        plan.forward(s["x"].half(), *w, y)
    with pytest.raises(ValueError):
        plan.forward(s["x"].cpu(), *w, y)
    with pytest.raises(ValueError):
        plan.forward(s["x"], s["wd"], s["wu"], s["wd"], y)           # shape
    with pytest.raises(ValueError):
        plan.forward(s["x"], s["wg"].T.contiguous().T, s["wu"], s["wd"], y)   # order
    with pytest.raises(ValueError):
        plan.forward(s["x"][:1].expand(8, 16), *w, y)                # overlapping rows
    with pytest.raises(_lib.RollerError) as e:
        big = torch.zeros(9, 16, dtype=torch.bfloat16, device="cuda")
        plan.forward(big, *w, torch.empty_like(big))
    assert e.value.status == _lib.ERR_TOO_LARGE
    with pytest.raises(_lib.RollerError) as e:
        plan.forward(s["x"], *w, s["x"])                             # in place
    assert e.value.status == _lib.ERR_INVALID
    outs = [torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd")]
    with pytest.raises(_lib.RollerError) as e:
        plan.backward(s["x"], *w, g, u, s["dy"], *outs)              # not a training plan
    assert e.value.status == _lib.ERR_UNSUPPORTED
    plan.check_status()
    plan.destroy()
    with pytest.raises(RuntimeError):
        plan.forward(s["x"], *w, y)


@pytest.mark.parametrize("act", ACTS)
def test_far_out_activations_stay_finite(act):
    # beyond 1.8e19 the square of g leaves fp32; the activation is g or zero there, its slope one or zero
    s = make(9, 40, 24, torch.bfloat16, 21)
    sign = torch.ones(9, 24, device="cuda")
    sign[::2] = -1
    s["g"] = (sign * 1e25).bfloat16()
    s["u"] = torch.full_like(s["g"], 1e-20)
    plan = GatedFfnPlan(9, 40, 24, activation=act, training=True)
    out = [torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd")]
    plan.backward(*(s[k] for k in ("x", "wg", "wu", "wd", "g", "u", "dy")), *out)
    plan.check_status()
    plan.destroy()
    a, slope = torch.where(sign > 0, s["g"].double(), 0.0), (sign > 0).double()
    # dg, du, h: one rounding each; the products: another, and their sums
    dh = s["dy"].double() @ s["wd"].double()
    dg, du, h = dh * s["u"].double() * slope, dh * a, a * s["u"].double()
    off = acc(40) * (s["dy"].double().abs() @ s["wd"].double().abs())
    u_ = half_step(torch.bfloat16)
    for got, parts in ((out[0], ((dg, off * s["u"].double() * slope, s["wg"].double()), (du, off * a, s["wu"].double()))),
                       (out[1], ((dg.T, (off * s["u"].double() * slope).T, s["x"].double()),)),
                       (out[2], ((du.T, (off * a).T, s["x"].double()),)),
                       (out[3], ((s["dy"].double().T, torch.zeros(40, 9, device="cuda", dtype=torch.float64), h),))):
        want = sum(p @ m for p, _, m in parts)
        # (u_ on either operand, whichever was rounded)
        bound = sum((e + (2 * u_ + acc(49) + 2.0 ** -20) * p.abs()) @ m.abs() for p, e, m in parts)
        within(got, want, bound + u_ * (want.abs() + bound) + tiny(torch.bfloat16), "gradient")


@pytest.mark.parametrize("shape", [(333, 768, 2048), (700, 1024, 1000), (300, 130, 4001), (70, 2050, 700)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_gradients_dealt_unevenly(shape, dtype):
    # the weights' tiles start beside dx's last wave, which leaves part of the SMs to them
    tokens, d, f = shape
    s = make(*shape, dtype, seed=22)
    plan = GatedFfnPlan(tokens, d, f, dtype=dtype, training=True)
    y, s["g"], s["u"] = run_forward(s, "silu", dtype, plan=plan)
    first = None
    for _ in range(3):
        out = {}
        bufs = {}
        for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd")):
            bufs[k], out[k] = guarded(*s[v].shape, dtype, pad_cols=8 if s[v].shape[1] % 8 == 0 else 3)
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], **out)
        plan.check_status()
        assert all(untouched(bufs[k], *out[k].shape) for k in out)
        if first is None:
            first = out
            for name, (want, bound) in backward_bounds(s, "silu", dtype).items():
                within(out[name], want, bound, name)
        assert all(torch.equal(first[k], out[k]) for k in out)
    plan.destroy()
