"""The Newton-Schulz orthogonalisation through its public plan.

The tolerance follows the operator's own roundings. `emulated` restates the iteration in 64 bits with
exactly the documented roundings (p, q and the operand x in fp16 on the 2^10 scale, x as two fp16
numbers, the lost part of q's diagonal in the factor of x). What the kernels add to that are
fp32 sums, which move a rounding now and then, so their error is a like one: twice the emulation's,
plus the last rounding to bf16 (half a step, 2^-8), in the Frobenius norm.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from mlir_roller_b200 import _lib  # noqa: E402
from mlir_roller_b200.orthogonal import MUON_COEFFICIENTS, OrthogonalPlan  # noqa: E402

S = 1024.0


def exact(g, steps=5, coefficients=MUON_COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    if x.shape[0] > x.shape[1]:      # (the polynomial commutes with the transpose)
        return exact(g.T, steps, coefficients, eps).T
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        p = x @ x.T
        x = a * x + (b * p + c * p @ p) @ x
    return x


def emulated(g, steps=5, coefficients=MUON_COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients

    def q16(v):
        return v.to(torch.float16).double()

    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = S * x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        hi = q16(x)
        full = hi + q16(x - hi)
        p = q16(hi @ hi.T / S)
        q = b * p + c * (p @ p) / S
        lost = (q - q16(q)).diagonal() / S
        x = (a + lost)[:, None] * full + q16(q) @ hi / S
    x = x / S
    return x.T if tall else x


def make(rows, cols, kind, seed=0, batch=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(batch, *shape, generator=gen, device="cuda")

    if kind == "rank1":
        return normal(rows, 1) @ normal(1, cols)
    if kind == "decay":
        r = min(rows, cols)
        u, _ = torch.linalg.qr(normal(rows, r))
        v, _ = torch.linalg.qr(normal(cols, r))
        return u * torch.arange(1, r + 1, device="cuda").float().pow(-0.5) @ v.transpose(1, 2)
    if kind == "empty rows":
        g = normal(rows, cols)
        g[:, :rows // 2] = 0
        return g
    if kind == "outlier":
        g = normal(rows, cols)
        g[:, rows // 3, cols // 2] = 1e4
        return g
    return normal(rows, cols) * 1e-4


def check(out, g, **how):
    for o, m in zip(out.reshape(-1, *out.shape[-2:]), g.reshape(-1, *g.shape[-2:])):
        want = exact(m, **how)
        norm = want.norm()
        slack = 2 * (emulated(m, **how) - want).norm() + 2.0 ** -8 * norm
        off = (o.double() - want).norm()
        assert off <= slack, f"{off / norm:.2e} of |x|, {slack / norm:.2e} allowed"


def run(g, **how):
    batch = g.shape[0] if g.dim() == 3 else 1
    plan = OrthogonalPlan(g.shape[-2], g.shape[-1], batch=batch, dtype=g.dtype, **how)
    before = g.clone()
    out = torch.full(g.shape, 9.0, dtype=torch.bfloat16, device="cuda")
    plan.run(g, out)
    plan.check_status()
    assert torch.equal(before.view(torch.uint8), g.view(torch.uint8))   # (bits: it may hold NaN)
    plan.destroy()
    return out


SHAPES = [(1, 1), (1, 40), (40, 1), (5, 7), (64, 64), (100, 130), (129, 127), (127, 400), (300, 65), (256, 256), (257, 700),
          (700, 257), (520, 1000), (1000, 520)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_the_definition(shape, dtype):
    g = make(*shape, "plain", seed=1)[0].to(dtype)
    check(run(g), g)


@pytest.mark.parametrize("kind", ["rank1", "decay", "empty rows", "outlier"])
@pytest.mark.parametrize("shape", [(128, 320), (320, 128), (200, 200)])
def test_spectra(kind, shape):
    g = make(*shape, kind, seed=2)[0]
    check(run(g), g)


@pytest.mark.parametrize("rows,cols", [(96, 200), (200, 96), (130, 130)])
def test_batches_and_strides(rows, cols):
    for dtype in (torch.float16, torch.float32, torch.bfloat16):
        g = make(rows, cols, "decay", seed=3, batch=3).to(dtype)
        g[1] *= 3                        # every matrix has its own norm
        out = run(g)
        check(out, g)
        assert torch.equal(run(g[2].clone()), out[2])
        # views: matrices of a wider buffer, then rows of three matrices interleaved, both at an
        # odd offset; the output likewise
        for perm in (False, True):
            def view(dt):
                if perm:
                    buf = torch.full((rows, 3, cols + 3), 7.0, dtype=dt, device="cuda")
                    return buf, buf[:, :, 1:cols + 1].transpose(0, 1)
                buf = torch.full((3, rows + 2, cols + 3), 7.0, dtype=dt, device="cuda")
                return buf, buf[:, :rows, 1:cols + 1]
            _, gv = view(dtype)
            gv.copy_(g)
            buf, ov = view(torch.bfloat16)
            plan = OrthogonalPlan(rows, cols, batch=3, dtype=dtype)
            plan.run(gv, ov)
            plan.check_status()
            assert torch.equal(ov, out)
            ov.fill_(7.0)
            assert bool((buf == 7.0).all())
            plan.destroy()


def test_steps_and_coefficients():
    g = make(150, 90, "decay", seed=4)[0]
    for how in (dict(steps=1), dict(steps=8), dict(steps=12, coefficients=(1.875, -1.25, 0.375)), dict(eps=1e-2)):
        check(run(g, **how), g, **how)
    # the convergent quintic ends in an orthogonal factor
    o = run(g, steps=16, coefficients=(1.875, -1.25, 0.375)).double()
    assert (o.T @ o - torch.eye(90, device="cuda", dtype=torch.float64)).abs().max() < 0.02


def test_zero_small_and_large():
    assert bool((run(torch.zeros(70, 50, device="cuda")) == 0).all())
    g = make(70, 150, "decay", seed=5)[0]
    for scale in (1e-25, 1e-4, 1e18):
        check(run(g * scale, eps=0.0), g * scale, eps=0.0)
    # far below eps the result is g / eps, grown a-fold a step: next to nothing
    assert run(g * 1e-25).abs().max() < 1e-10


def test_norms_whose_inverse_leaves_fp32():
    # every element a normal number (subnormal ones count as zero)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for shape, size in (((5, 7), 3e-37), ((5, 7), 1.6e38), ((300, 400), 1.6e38), ((400, 300), 1.6e38)):
        signs = torch.randint(0, 2, shape, generator=gen, device="cuda") * 2 - 1
        g = signs * (1 + torch.rand(shape, generator=gen, device="cuda")) * size
        for dtype in (torch.float32, torch.bfloat16):
            check(run(g.to(dtype), eps=0.0), g.to(dtype), eps=0.0)


def test_not_finite_stays_in_its_matrix():
    g = make(64, 100, "decay", seed=6, batch=3)
    want = run(g)
    g[1, 3, 5] = float("nan")
    out = run(g)
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2]) and out[1].isnan().all()


def test_repeats_and_graph():
    g = make(300, 2000, "plain", seed=7)[0]
    plan = OrthogonalPlan(300, 2000, dtype=torch.float32)
    out = torch.empty(300, 2000, dtype=torch.bfloat16, device="cuda")
    plan.run(g, out)
    first = out.clone()
    for _ in range(10):
        plan.run(g, out.zero_())
        assert torch.equal(out, first)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        plan.run(g, out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    g.copy_(make(300, 2000, "decay", seed=8)[0])
    graph.replay()
    torch.cuda.synchronize()
    plan.check_status()
    check(out, g)
    plan.destroy()


def test_refusals():
    with pytest.raises(TypeError):
        OrthogonalPlan(4, 4, dtype=torch.float64)
    for bad in (dict(rows=0, cols=4), dict(rows=4, cols=65537), dict(rows=4, cols=4, batch=0), dict(rows=4, cols=4, steps=0),
                dict(rows=4, cols=4, steps=33), dict(rows=4, cols=4, eps=-1.0), dict(rows=4, cols=4, eps=float("nan")),
                dict(rows=4, cols=4, coefficients=(5.0, 0.0, 0.0)), dict(rows=4, cols=4, coefficients=(float("inf"), 0.0, 0.0))):
        with pytest.raises(_lib.RollerError) as e:
            OrthogonalPlan(**bad)
        assert e.value.status == _lib.ERR_INVALID, bad
    with pytest.raises(_lib.RollerError) as e:
        OrthogonalPlan(20000, 20000)
    assert e.value.status == _lib.ERR_TOO_LARGE
    plan = OrthogonalPlan(8, 12)
    g = torch.ones(8, 12, dtype=torch.bfloat16, device="cuda")
    o = torch.empty_like(g)
    for call, error in (((g.float(), o), TypeError), ((g, o.float()), TypeError), ((g.cpu(), o), ValueError),
                        ((g.T, o), ValueError), ((g[:, :11], o), ValueError), ((g.T.contiguous().T, o), ValueError),
                        ((g, g), _lib.RollerError), ((g[:1].expand(8, 12), o), _lib.RollerError),
                        ((g, o[:1].expand(8, 12)), _lib.RollerError)):
        with pytest.raises(error):
            plan.run(*call)
    plan.destroy()
    with pytest.raises(RuntimeError):
        plan.run(g, o)
