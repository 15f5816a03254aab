"""Every compiled kernel of the feed-forward block and of the orthogonalisation, with every split of its
reduction, against 64 bits (fused_shapes.py; bounds as in the tests of the single operators). Outputs lie in
larger buffers, so that a row or column too many shows as well."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan  # noqa: E402
import fused_shapes as shapes  # noqa: E402
import test_ffn_gpu as block  # noqa: E402
import test_orthogonal_gpu as ortho  # noqa: E402

ACTS = ["silu", "gelu", "gelu_tanh"]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("shape", shapes.BLOCK)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block(shape, dtype):
    tokens, d, f = shape
    act = ACTS[(tokens + d + f) % 3]
    s = block.make(*shape, dtype, seed=80)
    plan = GatedFfnPlan(tokens, d, f, dtype=dtype, activation=act, training=True)
    sizes = dict(y=(tokens, d), g=(tokens, f), u=(tokens, f), dx=(tokens, d), dwg=(f, d), dwu=(f, d), dwd=(d, f))
    bufs, out = {}, {}
    for k, (rows, cols) in sizes.items():
        # rows on 16 bytes where the width allows it, as in a program's own tensors
        bufs[k], out[k] = block.guarded(rows, cols, dtype, pad_cols=8 if cols % 8 == 0 else 3)
    plan.forward(s["x"], s["wg"], s["wu"], s["wd"], out["y"], out["g"], out["u"])
    s["g"], s["u"] = out["g"], out["u"]
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], *(out[k] for k in ("dx", "dwg", "dwu", "dwd")))
    plan.check_status()
    plan.destroy()
    for bounds in (block.forward_bounds, block.backward_bounds):
        for name, (want, bound) in bounds(s, act, dtype).items():
            block.within(out[name], want, bound, name)
    for k in sizes:
        assert block.untouched(bufs[k], *sizes[k]), k


@pytest.mark.parametrize("shape", shapes.UPDATE)
def test_update(shape):
    batch, rows, cols = shape
    dtype = TYPES[(batch + rows + cols) % 3]
    g = ortho.make(rows, cols, "plain", seed=81, batch=batch).to(dtype)
    g[0] = ortho.make(rows, cols, "decay", seed=82)[0].to(dtype)
    ortho.check(ortho.run(g), g)


def test_weight_gradients_over_offsets_beyond_32_bits():
    """270,000 tokens x 8192, 2.2e9 elements each of dg, du and h, which the weights' gradients sum over. The
    tokens are 1000, repeated, but for 80 of their own, at the end and where the offsets pass 2^31, whose dy
    is so large that the bound would not survive their being left out or read from elsewhere."""
    dtype, act = torch.bfloat16, "silu"
    tokens, d, f, base = 270_000, 64, 8192, 1000
    middle = 2 ** 31 // f
    own = torch.cat((torch.arange(middle - 20, middle + 20), torch.arange(tokens - 40, tokens))).cuda()
    s = block.make(base, d, f, dtype, seed=83)
    fresh = block.make(len(own), d, f, dtype, seed=84)
    x, dy = (s[k].repeat(tokens // base, 1) for k in ("x", "dy"))
    x[own], dy[own] = fresh["x"], fresh["dy"] * 1024
    plan = GatedFfnPlan(tokens, d, f, activation=act, training=True)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    g, u = plan.new_saved(tokens)
    plan.forward(x, s["wg"], s["wu"], s["wd"], y, g, u)
    out = dict(zip(("dwg", "dwu", "dwd"), (torch.empty_like(s[k]) for k in ("wg", "wu", "wd"))))
    plan.backward(x, s["wg"], s["wu"], s["wd"], g, u, dy, dx, *out.values())
    plan.check_status()
    plan.destroy()
    repeated = torch.ones(tokens, dtype=torch.bool, device="cuda")
    repeated[own] = False
    for first in range(0, tokens, base):       # repeated tokens have the same g and u
        r = repeated[first:first + base]
        assert torch.equal(g[first:first + base][r], g[:base][r]) and torch.equal(u[first:first + base][r], u[:base][r])

    def sums(rows, times):
        """Of these tokens: each gradient, how far roundings of its operands may move it, its magnitude."""
        v = {k: t.double() for k, t in rows.items()}
        wd, half = s["wd"].double(), block.half_step(dtype)
        a, b = block.act64(act, v["g"]), block.slope64(act, v["g"])
        dh, edh = v["dy"] @ wd, block.acc(d) * (v["dy"].abs() @ wd.abs())
        fast = 2.0 ** -20 * (1 + v["g"].abs()) ** 2
        result = {}
        for name, value, error, other in (
                ("dwg", dh * v["u"] * b, edh * (v["u"] * b).abs() + (dh.abs() + edh) * v["u"].abs() * fast, v["x"]),
                ("dwu", dh * a, edh * a.abs() + (dh.abs() + edh) * fast, v["x"]),
                ("dwd", a * v["u"], v["u"].abs() * fast, v["dy"])):
            error = error + half * (value.abs() + error) + block.tiny(dtype)
            three = (value.T @ other, error.T @ other.abs(), (value.abs() + error).T @ other.abs())
            result[name] = [times * (t.T if name == "dwd" else t) for t in three]
        return result

    whole = sums(dict(x=s["x"], dy=s["dy"], g=g[:base], u=u[:base]), tokens // base)
    gone = own % base
    replaced = sums(dict(x=s["x"][gone], dy=s["dy"][gone], g=g[:base][gone], u=u[:base][gone]), 1)
    added = sums(dict(x=x[own], dy=dy[own], g=g[own], u=u[own]), 1)
    for name, got in out.items():
        want = whole[name][0] - replaced[name][0] + added[name][0]
        bound = whole[name][1] + added[name][1] + block.acc(tokens) * (whole[name][2] + added[name][2])
        bound = bound + block.half_step(dtype) * (want.abs() + bound) + block.tiny(dtype)
        block.within(got, want, bound, name)
        for part in (slice(0, 40), slice(40, 80)):     # either group of tokens of their own matters
            alone = sums(dict(x=x[own[part]], dy=dy[own[part]], g=g[own[part]], u=u[own[part]]), 1)[name][0]
            assert (alone.abs() > bound).double().mean() > 0.25, name
