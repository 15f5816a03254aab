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
