"""The feed-forward and orthogonalising plans among streams, graphs and other work of a program."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import GatedFfnPlan, OrthogonalPlan  # noqa: E402
import test_ffn_gpu as block  # noqa: E402


def used_memory():
    """Small pieces of device memory, filled with ones and given back: the next ones asked for hold that."""
    rt = ctypes.CDLL("libcudart.so.12")
    pieces = [ctypes.c_void_p() for _ in range(64)]
    for p in pieces:
        assert rt.cudaMalloc(ctypes.byref(p), ctypes.c_size_t(4)) == 0
        assert rt.cudaMemset(p, 255, ctypes.c_size_t(4)) == 0
    torch.cuda.synchronize()
    for p in pieces:
        assert rt.cudaFree(p) == 0


@pytest.mark.parametrize("kind", ["block", "update"])
def test_a_new_plan_is_ready_for_any_stream(kind):
    """A plan made while the default stream is busy, and used at once on a stream that does not wait for
    that one: whatever the plan sets up has to be complete."""
    s = block.make(96, 256, 512, torch.bfloat16, seed=70)
    out = torch.zeros_like(s["x"] if kind == "block" else s["wg"])

    def once(stream):
        if kind == "block":
            plan = GatedFfnPlan(96, 256, 512)
            plan.forward(s["x"], s["wg"], s["wu"], s["wd"], out, stream=stream)
        else:
            plan = OrthogonalPlan(512, 256)
            plan.run(s["wg"], out, stream=stream)
        return plan

    plan = once(None)
    plan.check_status()
    plan.destroy()
    want = out.clone()
    out.zero_()
    side = torch.cuda.Stream()
    used_memory()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)      # about a tenth of a second
    plan = once(side)
    side.synchronize()
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    plan.check_status()
    plan.destroy()


@pytest.mark.parametrize("d", [1, 2, 63, 510, 511, 512, 513, 514, 1025])
def test_rows_that_start_anywhere(d):
    """Copies of unaligned rows, around the 512 elements that a warp moves at a time: from every offset the
    same bits as from aligned rows, and nothing beside a row counts (it is NaN here)."""
    tokens, f = 37, 72
    s = block.make(tokens, d, f, torch.bfloat16, seed=71)
    plan = GatedFfnPlan(tokens, d, f)

    def view(t, lead, ld):
        buf = torch.full((t.shape[0], ld), float("nan"), dtype=t.dtype, device="cuda")
        v = buf[:, lead:lead + t.shape[1]]
        v.copy_(t)
        return v

    y, again = (torch.empty(tokens, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    aligned = (d + 7) // 8 * 8
    plan.forward(*(view(s[k], 0, aligned) for k in ("x", "wg", "wu")), s["wd"], y)
    for lead in range(8):
        for more in (0, 1, 5):
            plan.forward(*(view(s[k], lead, aligned + lead + more) for k in ("x", "wg", "wu")), s["wd"], again.zero_())
            assert torch.equal(again, y), (lead, more)
    plan.check_status()
    plan.destroy()
    assert bool(y.isfinite().all())


@pytest.mark.parametrize("d,f", [(256, 512), (130, 257)])
def test_graphs_with_copies_and_two_branches(d, f):
    """A captured step as a training program has it: inputs copied into place, forward, backward, and the two
    updates side by side in branches of the graph, behind a copy of the gradient each. (The kernels may
    start early behind one another, but not behind a copy or a join.)"""
    tokens, dtype = 200, torch.bfloat16
    plan = GatedFfnPlan(tokens, d, f, training=True)
    muon = [OrthogonalPlan(f, d), OrthogonalPlan(f, d)]
    fresh = [block.make(tokens, d, f, dtype, seed=90 + i) for i in range(4)]
    live = {k: torch.zeros_like(t) for k, t in fresh[0].items()}
    y, dx = (torch.zeros_like(live["x"]) for _ in range(2))
    g, u = plan.new_saved(tokens)
    dw = [torch.zeros_like(live[k]) for k in ("wg", "wu", "wd")]
    kept, up = ([torch.zeros_like(live["wg"]) for _ in range(2)] for _ in range(2))
    source = {k: torch.zeros_like(t) for k, t in fresh[0].items()}
    side = torch.cuda.Stream()

    def step():
        for k in live:
            live[k].copy_(source[k])
        plan.forward(live["x"], live["wg"], live["wu"], live["wd"], y, g, u)
        plan.backward(live["x"], live["wg"], live["wu"], live["wd"], g, u, live["dy"], dx, *dw)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        kept[0].copy_(dw[0])
        muon[0].run(kept[0], up[0])
        with torch.cuda.stream(side):
            kept[1].copy_(dw[1])
            muon[1].run(kept[1], up[1])
        here.wait_stream(side)
        plan.forward(dx, up[0], up[1], dw[2], y, g, u)
        return [y, g, u, dx, *dw, *up]

    want = []
    for s in fresh:
        for k in source:
            source[k].copy_(s[k])
        torch.cuda.synchronize()
        want.append([t.clone() for t in step()])
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        for s, w in zip(fresh, want):
            for k in source:
                source[k].copy_(s[k])
            graph.replay()
            for a, b in zip(outs, w):
                assert torch.equal(a, b)
    plan.check_status()
    graph.reset()
    for p in (plan, *muon):
        p.check_status()
        p.destroy()


@pytest.mark.parametrize("d,f", [(256, 512), (130, 257)])
def test_operands_that_another_stream_finishes_late(d, f):
    """Each operand is written by another stream, behind a long kernel; the plan's stream waits for its event."""
    tokens, dtype = 64, torch.bfloat16
    s = block.make(tokens, d, f, dtype, seed=95)
    plan, muon = GatedFfnPlan(tokens, d, f), OrthogonalPlan(d, f)
    y, out = torch.empty_like(s["x"]), torch.empty_like(s["wd"])
    plan.forward(s["x"], s["wg"], s["wu"], s["wd"], y)
    muon.run(s["wd"], out)
    want, want_out = y.clone(), out.clone()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    late = {k: torch.zeros_like(t) for k, t in s.items()}
    for name in ("x", "wg", "wu", "wd"):
        for k in late:
            late[k].copy_(s[k]) if k != name else late[k].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(b):
            torch.cuda._sleep(4_000_000)
            late[name].copy_(s[name])
            done = b.record_event()
        with torch.cuda.stream(a):
            plan.forward(s["x"], s["wg"], s["wu"], s["wd"], y.zero_())     # (work in front, without the operand)
            a.wait_event(done)
            plan.forward(late["x"], late["wg"], late["wu"], late["wd"], y.zero_())
            muon.run(late["wd"], out.zero_())
        a.synchronize()
        assert torch.equal(y, want) and torch.equal(out, want_out), name
    for p in (plan, muon):
        p.check_status()
        p.destroy()


def test_the_same_tensor_in_two_places():
    """One weight for both projections, one tensor as x and dy, one as g and u."""
    tokens, d, f, dtype = 150, 136, 264, torch.bfloat16
    s = block.make(tokens, d, f, dtype, seed=96)
    s["wu"], s["dy"] = s["wg"], s["x"]
    plan = GatedFfnPlan(tokens, d, f, training=True)
    y, g, u = block.run_forward(s, "silu", dtype, plan=plan)
    assert torch.equal(g, u)
    block.within(y, *block.forward_bounds(s, "silu", dtype)["y"], "y")
    s["g"] = s["u"] = g
    out = {k: torch.empty_like(s[v]) for k, v in (("dx", "x"), ("dwg", "wg"), ("dwu", "wu"), ("dwd", "wd"))}
    plan.backward(s["x"], s["wg"], s["wg"], s["wd"], g, g, s["x"], **out)
    plan.check_status()
    for name, (want, bound) in block.backward_bounds(s, "silu", dtype).items():
        block.within(out[name], want, bound, name)
    plan.destroy()


@pytest.mark.parametrize("shape", [(1, 1, 5), (3, 1, 40), (3, 40, 1), (2, 33, 70)])
def test_an_infinite_element_stays_in_its_matrix(shape):
    g = torch.randn(*shape, device="cuda")
    plan = OrthogonalPlan(*shape[1:], batch=shape[0], dtype=torch.float32)
    want, out = (torch.empty(*shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    plan.run(g, want)
    g[-1, -1, -1] = float("inf")
    plan.run(g, out)
    plan.check_status()
    plan.destroy()
    assert torch.equal(out[:-1], want[:-1])
    assert not out[-1].isfinite().all()
