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
