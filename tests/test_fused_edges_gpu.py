"""Outputs of the feed-forward and orthogonalising plans whose rows start on 16 bytes and end anywhere: what lies
behind a row stays as it was."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan  # noqa: E402
import test_ffn_gpu as block  # noqa: E402


def behind(cols):
    """Columns to add for a row stride of a multiple of 16 bytes, one unit at least."""
    return 8 + -cols % 8


@pytest.mark.parametrize("tokens", [1, 6, 150])
@pytest.mark.parametrize("d,f", [(1, 1), (9, 40), (40, 23), (61, 130), (135, 260), (258, 517)])
def test_block_outputs(tokens, d, f):
    dtype = torch.bfloat16
    s = block.make(tokens, d, f, dtype, seed=72)
    plan = GatedFfnPlan(tokens, d, f, training=True)
    sizes = dict(y=(tokens, d), g=(tokens, f), u=(tokens, f), dx=(tokens, d), dwg=(f, d), dwu=(f, d), dwd=(d, f))

    def run(out):
        plan.forward(s["x"], s["wg"], s["wu"], s["wd"], out["y"], out["g"], out["u"])
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], out["g"], out["u"], s["dy"],
                      *(out[k] for k in ("dx", "dwg", "dwu", "dwd")))
        plan.check_status()

    want = {k: torch.empty(*size, dtype=dtype, device="cuda") for k, size in sizes.items()}
    run(want)
    bufs, out = {}, {}
    for k, (rows, cols) in sizes.items():
        bufs[k], out[k] = block.guarded(rows, cols, dtype, pad_cols=behind(cols))
    run(out)
    for k, size in sizes.items():
        assert torch.equal(out[k], want[k]), k
        assert block.untouched(bufs[k], *size), k
    plan.destroy()


@pytest.mark.parametrize("f", [20, 36, 260])
def test_outputs_side_by_side_in_one_buffer(f):
    """g and u, and the gradients of both projections, as the halves of wider matrices: the second half
    starts inside the 16 bytes in which the first one ends."""
    tokens, d, dtype = 140, 44, torch.bfloat16
    s = block.make(tokens, d, f, dtype, seed=73)
    plan = GatedFfnPlan(tokens, d, f, training=True)
    y, g, u = block.run_forward(s, "silu", dtype, plan=plan)
    outs = [torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd")]
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], g, u, s["dy"], *outs)
    saved = torch.empty(tokens, 2 * f, dtype=dtype, device="cuda")
    dw = torch.empty(f, 2 * d, dtype=dtype, device="cuda")
    dx, dwd = torch.empty_like(outs[0]), torch.empty_like(outs[3])
    for _ in range(5):
        saved.fill_(5.0)
        dw.fill_(5.0)
        plan.forward(s["x"], s["wg"], s["wu"], s["wd"], y, saved[:, :f], saved[:, f:])
        assert torch.equal(saved, torch.cat((g, u), 1))
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], saved[:, :f], saved[:, f:], s["dy"], dx, dw[:, :d], dw[:, d:], dwd)
        assert torch.equal(dw, torch.cat(outs[1:3], 1))
        assert torch.equal(dx, outs[0]) and torch.equal(dwd, outs[3])
    plan.check_status()
    plan.destroy()


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("rows,cols", [(1, 5), (40, 19), (61, 90), (90, 61), (300, 130), (130, 300), (200, 201), (257, 515)])
def test_updates(batch, rows, cols):
    g = torch.randn(batch, rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(74))
    plan = OrthogonalPlan(rows, cols, batch=batch, dtype=torch.float32)
    want = torch.empty(batch, rows, cols, dtype=torch.bfloat16, device="cuda")
    plan.run(g, want)
    buf = torch.full((batch, rows + 1, cols + behind(cols)), 776.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, :rows, :cols]
    plan.run(g, out)
    plan.check_status()
    assert torch.equal(out, want)
    out.fill_(776.0)
    assert bool((buf == 776.0).all())
    plan.destroy()


@pytest.mark.parametrize("stride", [2 ** 31 + 8, 2 ** 31 + 3])
def test_row_strides_beyond_32_bits(stride):
    """Every operand and output of the block, and the matrices of an update, with rows 4 GB apart, at once
    in one buffer; on 16 bytes and not."""
    tokens, d, f, dtype = 3, 3, 2, torch.bfloat16
    s = block.make(tokens, d, f, dtype, seed=75)
    plan = GatedFfnPlan(tokens, d, f, training=True)
    y, g, u = block.run_forward(s, "silu", dtype, plan=plan)
    want = dict(y=y, g=g, u=u, **{k: torch.empty_like(s[v]) for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))})
    plan.backward(s["x"], s["wg"], s["wu"], s["wd"], g, u, s["dy"], *(want[k] for k in ("dx", "dwg", "dwu", "dwd")))
    buf = torch.empty(2 * stride + 2048, dtype=dtype, device="cuda")
    v = {}
    for i, (k, t) in enumerate({**s, **want}.items()):
        for r in range(t.shape[0]):
            buf[r * stride + 64 * i:r * stride + 64 * (i + 1)] = 776.0
        v[k] = buf[64 * i + 8:].as_strided(t.shape, (stride, 1))
    for k in s:
        v[k].copy_(s[k])
    plan.forward(v["x"], v["wg"], v["wu"], v["wd"], v["y"], v["g"], v["u"])
    plan.backward(v["x"], v["wg"], v["wu"], v["wd"], v["g"], v["u"], v["dy"], v["dx"], v["dwg"], v["dwu"], v["dwd"])
    plan.check_status()
    plan.destroy()
    for i, (k, t) in enumerate({**s, **want}.items()):
        assert torch.equal(v[k], t), k
        for r in range(t.shape[0]):
            around = buf[r * stride + 64 * i:r * stride + 64 * (i + 1)].clone()
            around[8:8 + t.shape[1]] = 776.0
            assert bool((around == 776.0).all()), k

    # updates: matrices far apart, and rows far apart with the matrices interleaved
    m = torch.randn(2, 3, 5, device="cuda").to(dtype)
    plan = OrthogonalPlan(3, 5, batch=2)
    out = torch.empty_like(m)
    plan.run(m, out)
    for strides in ((stride, 16, 1), (16, stride, 1), (13, stride, 1)):
        a, b = buf.as_strided((2, 3, 5), strides), buf[512:].as_strided((2, 3, 5), strides)
        a.copy_(m)
        b.zero_()
        plan.run(a, b)
        assert torch.equal(b, out), strides
    plan.check_status()
    plan.destroy()
