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
