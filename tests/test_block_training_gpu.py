"""The plans as a training program uses them together: a projection through a GEMM plan, the gated
feed-forward block behind it, its backward pass, and the orthogonalised update of its weights; and
calls whose offsets pass 32 bits. Bounds as in the tests of the single operators."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan, _lib  # noqa: E402
from mlir_roller_b200.analyze import MODE_BF16  # noqa: E402
import test_ffn_gpu as block  # noqa: E402
import test_orthogonal_gpu as ortho  # noqa: E402


def test_steps_of_a_training_run():
    """x = t Wp by a GEMM plan, y = block(x), gradients, momenta, orthogonalised updates. Every stage
    is held to its bound on the inputs that the stage before it handed over; the weights move
    through two steps, so plans and workspaces are used again."""
    dtype = torch.bfloat16
    tokens, d, f = 300, 192, 328
    s = block.make(tokens, d, f, dtype, seed=31)
    gen = torch.Generator(device="cuda").manual_seed(32)
    t = torch.randn(tokens, 136, generator=gen, device="cuda").to(dtype)
    wp = (torch.randn(136, d, generator=gen, device="cuda") * 136 ** -0.5).to(dtype)
    proj = _lib.GemmPlan(_lib.find_tile(128, 128, 1), tokens, d, 136, mode=MODE_BF16, flags=_lib.FLAG_C_16BIT)
    plan = GatedFfnPlan(512, d, f, training=True)
    muon = OrthogonalPlan(f, d, batch=2, dtype=torch.float32)
    muon_down = OrthogonalPlan(d, f, dtype=torch.float32)
    # the gate's and the up projection's weights and momenta live in one buffer each
    up = torch.stack((s["wg"], s["wu"])).contiguous()
    momentum = torch.zeros(2, f, d, device="cuda")
    momentum_down = torch.zeros(d, f, device="cuda")
    wd = s["wd"].clone()
    for step in range(2):
        x = torch.empty(tokens, d, dtype=dtype, device="cuda")
        proj.run(t, wp, x)
        y = torch.empty_like(x)
        g, u = plan.new_saved(tokens)
        plan.forward(x, up[0], up[1], wd, y, g, u)
        dx, dup, dwd = torch.empty_like(x), torch.empty_like(up), torch.empty_like(wd)
        plan.backward(x, up[0], up[1], wd, g, u, s["dy"], dx, dup[0], dup[1], dwd)
        momentum.mul_(0.9).add_(dup)
        momentum_down.mul_(0.9).add_(dwd)
        update, update_down = torch.empty_like(up), torch.empty_like(wd)
        muon.run(momentum, update)
        muon_down.run(momentum_down, update_down)
        plan.check_status()
        proj.check_status()
        muon.check_status()
        muon_down.check_status()
        here = dict(x=x, wg=up[0], wu=up[1], wd=wd, g=g, u=u, dy=s["dy"])
        block.within(x, t.double() @ wp.double(),
                     (block.acc(136) + 2.0 ** -8) * (t.double().abs() @ wp.double().abs()), "x")
        for name, (want, bound) in block.forward_bounds(here, "silu", dtype).items():
            block.within(dict(y=y, g=g, u=u)[name], want, bound, name)
        for name, (want, bound) in block.backward_bounds(here, "silu", dtype).items():
            block.within(dict(dx=dx, dwg=dup[0], dwu=dup[1], dwd=dwd)[name], want, bound, name)
        ortho.check(update, momentum)
        ortho.check(update_down, momentum_down)
        up.add_(update, alpha=-0.02)
        wd.add_(update_down, alpha=-0.02)
    for p in (proj, plan, muon, muon_down):
        p.destroy()


def test_two_plans_on_two_streams():
    """Plans of different streams do not meet: the same results as one after the other."""
    dtype = torch.bfloat16
    data = [block.make(150, 256, 512, dtype, seed=40 + i) for i in range(2)]
    plans = [GatedFfnPlan(150, 256, 512) for _ in range(2)]
    want = [block.run_forward(s, "silu", dtype, plan=p) for s, p in zip(data, plans)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(s["x"]) for s in data]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, p, o, st in zip(data, plans, outs, streams):
            p.forward(s["x"], s["wg"], s["wu"], s["wd"], o, stream=st)
    torch.cuda.synchronize()
    for p, o, w in zip(plans, outs, want):
        p.check_status()
        assert torch.equal(o, w[0])
        p.destroy()


def test_block_offsets_beyond_32_bits():
    """270,000 tokens x 8192: g, u and h have 2.2e9 elements each. The last tokens are held to the
    bounds, and their gradients."""
    dtype = torch.bfloat16
    tokens, d, f, last = 270_000, 64, 8192, 40
    s = block.make(1000, d, f, dtype, seed=50)
    x, dy = (s[k].repeat(tokens // 1000, 1) for k in ("x", "dy"))
    fresh = block.make(last, d, f, dtype, seed=51)
    x[-last:], dy[-last:] = fresh["x"], fresh["dy"]
    plan = GatedFfnPlan(tokens, d, f, training=True)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    g, u = plan.new_saved(tokens)
    plan.forward(x, s["wg"], s["wu"], s["wd"], y, g, u)
    grads = [torch.empty_like(s[k]) for k in ("wg", "wu", "wd")]
    plan.backward(x, s["wg"], s["wu"], s["wd"], g, u, dy, dx, *grads)
    plan.check_status()
    tail = dict(s, x=x[-last:], dy=dy[-last:], g=g[-last:], u=u[-last:])
    for name, (want, bound) in block.forward_bounds(tail, "silu", dtype).items():
        block.within(dict(y=y, g=g, u=u)[name][-last:], want, bound, name)
    want, bound = block.backward_bounds(tail, "silu", dtype)["dx"]
    block.within(dx[-last:], want, bound, "dx")
    assert all(bool(t.isfinite().all()) for t in grads)
    plan.destroy()


def test_orthogonal_offsets_beyond_32_bits():
    """550 matrices of 65536 x 64: 2.3e9 elements. The last matrix alone gives the same result."""
    batch = 550
    g = torch.randn(65536, 64, device="cuda").to(torch.bfloat16).repeat(batch, 1, 1)
    g[-1] = ortho.make(65536, 64, "plain", seed=52)[0].to(torch.bfloat16)
    out = torch.empty_like(g)
    plan = OrthogonalPlan(65536, 64, batch=batch)
    plan.run(g, out)
    plan.check_status()
    plan.destroy()
    ortho.check(out[-1], g[-1])
    assert torch.equal(out[0], out[batch // 2])


@pytest.mark.parametrize("tokens,d,f", [(1, 512, 2048), (40, 512, 1536), (300, 264, 520), (90, 129, 257), (700, 768, 2000)])
def test_calls_in_a_row_see_what_the_calls_before_them_wrote(tokens, d, f):
    """Launches overlap (weights fetched early, independent gradient products side by side, copies of
    unaligned operands behind the first product). A chain of two blocks whose weights are rewritten
    right before every step gives the same bits with and without waiting in between."""
    dtype = torch.bfloat16
    fresh = [[block.make(tokens, d, f, dtype, seed=60 + 2 * i + j) for j in range(2)] for i in range(6)]

    def chain(wait):
        plans = [GatedFfnPlan(tokens, d, f, training=True) for _ in range(2)]
        muon = OrthogonalPlan(f, d)
        live = [{k: torch.zeros_like(v) for k, v in s.items()} for s in fresh[0]]
        seen = []

        def step():
            if wait:
                torch.cuda.synchronize()

        for data in fresh:
            for now, s in zip(live, data):
                for k in s:
                    now[k].copy_(s[k])
            step()
            x = live[0]["x"]
            saved = []
            for plan, w in zip(plans, live):
                y = torch.empty_like(x)
                g, u = plan.new_saved(tokens)
                plan.forward(x, w["wg"], w["wu"], w["wd"], y, g, u)
                step()
                saved.append((x, g, u))
                seen += [y, g, u]
                x = y
            dy = live[1]["dy"]
            for plan, w, (x, g, u) in reversed(list(zip(plans, live, saved))):
                dx, dwg, dwu, dwd = (torch.empty_like(t) for t in (x, w["wg"], w["wu"], w["wd"]))
                plan.backward(x, w["wg"], w["wu"], w["wd"], g, u, dy, dx, dwg, dwu, dwd)
                step()
                update = torch.empty_like(dwg)
                muon.run(dwg, update)
                step()
                w["wg"].add_(update, alpha=-0.1)       # the very next kernel writes a weight
                w["wd"].add_(dwd)
                step()
                seen += [dx, dwg, dwu, dwd, update]
                dy = dx
        torch.cuda.synchronize()
        for p in plans + [muon]:
            p.check_status()
            p.destroy()
        return seen

    for a, b in zip(chain(False), chain(True)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
