"""What is measured of the feed-forward and the orthogonalising operators, and their plain forms.

Four operators, as a training program and a server use them:

  serve     y = (act(x Wg^T) * (x Wu^T)) Wd^T, the gated feed-forward block without a backward pass
  train     the same block, handing out g = x Wg^T and u = x Wu^T for the backward pass
  backward  the gradients of x, Wg, Wu and Wd from x, the weights, the saved g and u, and dy
  ortho     the Newton-Schulz iteration that the Muon optimiser applies to the update of a weight
            matrix: x <- a x + (b x x^T + c (x x^T)^2) x, from x = update / |update|

`run` computes them in elementary torch operations (32 bits, rounded once at the end), or, where
`own` is true, with this repository's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # one token of one request, where the weights' way from memory is everything
        dict(name="serve-1", op="serve", tokens=1, d=2048, f=8192, dtype="bf16", act="silu"),
        # one token each of 48 requests
        dict(name="serve-48", op="serve", tokens=48, d=4096, f=8192, dtype="bf16", act="gelu_tanh"),
        # a short prompt through a block whose inner width is 8/3 of the outer one, an odd number
        dict(name="serve-777-odd", op="serve", tokens=777, d=2048, f=5461, dtype="fp16", act="silu"),
        # several long prompts packed
        dict(name="serve-8192", op="serve", tokens=8192, d=4096, f=8192, dtype="bf16", act="silu"),
        # the forward half of a training step
        dict(name="train-4096", op="train", tokens=4096, d=2048, f=8192, dtype="fp16", act="gelu"),
        # a small model's backward pass, a few sequences of uneven length
        dict(name="backward-200", op="backward", tokens=200, d=1024, f=2816, dtype="bf16", act="silu"),
        # the backward pass of the odd block, a ragged batch
        dict(name="backward-1999-odd", op="backward", tokens=1999, d=2048, f=5461, dtype="bf16", act="gelu_tanh"),
        # a full training batch of one GPU
        dict(name="backward-8192", op="backward", tokens=8192, d=4096, f=8192, dtype="bf16", act="silu"),
        # one small square projection's update
        dict(name="ortho-512", op="ortho", batch=1, rows=512, cols=512, dtype="bf16"),
        # the updates of three layers' odd feed-forward weights, taller than wide, kept in 32 bits
        dict(name="ortho-3x2731x1024", op="ortho", batch=3, rows=2731, cols=1024, dtype="fp32"),
        # a wide projection
        dict(name="ortho-2048x8192", op="ortho", batch=1, rows=2048, cols=8192, dtype="bf16"),
        # the largest feed-forward weight
        dict(name="ortho-8192x4096", op="ortho", batch=1, rows=8192, cols=4096, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["serve", "serve", "train", "backward", "ortho", "ortho"])
    if op == "ortho":
        while True:
            case = dict(op=op, batch=rng.choice([1, 1, 2, 3, 5, 8]), rows=_log(rng, 100, 8192),
                        cols=_log(rng, 100, 8192), dtype=rng.choice(["bf16", "bf16", "fp32", "fp16"]))
            if min(case["rows"], case["cols"]) <= 4096 and work(case)["flops"] <= work(listed()[-1])["flops"]:
                return case
    d, f = _log(rng, 256, 4096), _log(rng, 512, 8192)
    if rng.random() < 0.75:  # most models keep their widths to multiples of eight
        d, f = d // 8 * 8, f // 8 * 8
    return dict(op=op, tokens=_log(rng, 1 if op == "serve" else 64, 8192), d=d, f=f,
                dtype=rng.choice(["bf16", "bf16", "fp16"]), act=rng.choice(["silu", "gelu", "gelu_tanh"]))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale)

    dt = DTYPES[case["dtype"]]
    if case["op"] == "ortho":
        b, m, n = case["batch"], case["rows"], case["cols"]
        # a momentum: a few strong directions over a broad floor
        r = min(32, m, n)
        strong = normal(b, m, r) * torch.logspace(0, -1, r, device="cuda")
        g = strong @ normal(b, r, n, scale=r ** -0.5) + normal(b, m, n, scale=0.1)
        return {"g": (g * 1e-3).to(dt)}
    t, d, f = case["tokens"], case["d"], case["f"]
    s = {
        "x": normal(t, d).to(dt),
        "wg": normal(f, d, scale=1.5 * d ** -0.5).to(dt),
        "wu": normal(f, d, scale=d ** -0.5).to(dt),
        "wd": normal(d, f, scale=f ** -0.5).to(dt),
    }
    if case["op"] == "backward":
        s["g"] = s["x"] @ s["wg"].T
        s["u"] = s["x"] @ s["wu"].T
        s["dy"] = normal(t, d, scale=0.1).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from mlir_roller_b200 import ffn, orthogonal

        dt = DTYPES[case["dtype"]]
        if case["op"] == "ortho":
            s["plan"] = orthogonal.OrthogonalPlan(case["rows"], case["cols"], batch=case["batch"], dtype=dt,
                                                  steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
            s["out"] = torch.empty_like(s["g"], dtype=torch.bfloat16)
            return s
        s["plan"] = ffn.GatedFfnPlan(case["tokens"], case["d"], case["f"], dtype=dt, activation=case["act"],
                                     training=case["op"] == "backward")
        if case["op"] == "backward":
            s["out"] = tuple(torch.empty_like(s[k]) for k in ("x", "wg", "wu", "wd"))
        else:
            s["out"] = torch.empty_like(s["x"])
        if case["op"] == "train":
            s["saved"] = s["plan"].new_saved(case["tokens"])
    return s


def _act(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _act_slope(name, v):
    if name == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 + v * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v * v * v))
    return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)


def _run_own(s):
    case, plan = s["case"], s["plan"]
    if case["op"] == "ortho":
        plan.run(s["g"], s["out"])
        return s["out"]
    if case["op"] == "backward":
        plan.backward(s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"], s["dy"], *s["out"])
        return dict(zip(("dx", "dwg", "dwu", "dwd"), s["out"]))
    if case["op"] == "train":
        g, u = s["saved"]
        plan.forward(s["x"], s["wg"], s["wu"], s["wd"], s["out"], g, u)
        return {"y": s["out"], "g": g, "u": u}
    plan.forward(s["x"], s["wg"], s["wu"], s["wd"], s["out"])
    return s["out"]


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "ortho":
        x = s["g"].float()
        tall = case["rows"] > case["cols"]
        if tall:
            x = x.transpose(1, 2)
        a, b, c = COEFFICIENTS
        x = x / (x.square().sum(dim=(1, 2), keepdim=True, dtype=torch.float64).sqrt().float() + EPS)
        # STEPS = 5 times the same step
        x = _step(_step(_step(_step(_step(x, a, b, c), a, b, c), a, b, c), a, b, c), a, b, c)
        return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()
    x, wg, wu, wd = (s[k].float() for k in ("x", "wg", "wu", "wd"))
    act = case["act"]
    if case["op"] == "backward":
        g, u, dy = (s[k].float() for k in ("g", "u", "dy"))
        a = _act(act, g)
        dh = dy @ wd
        dg = dh * u * _act_slope(act, g)
        du = dh * a
        return {"dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.T @ x).to(dt), "dwu": (du.T @ x).to(dt),
                "dwd": (dy.T @ (a * u)).to(dt)}
    g, u = x @ wg.T, x @ wu.T
    y = ((_act(act, g) * u) @ wd.T).to(dt)
    return {"y": y, "g": g.to(dt), "u": u.to(dt)} if case["op"] == "train" else y


def _step(x, a, b, c):
    p = x @ x.transpose(1, 2)
    return a * x + (b * p + c * (p @ p)) @ x


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "ortho":
        # the same polynomial from the other side: x <- x (a + q (b + c q)) with q = x^T x, each
        # matrix by itself
        a, b, c = COEFFICIENTS
        done = []
        for x in s["g"].double():
            if case["rows"] < case["cols"]:
                x = x.T
            x = x / (torch.linalg.matrix_norm(x) + EPS)
            for _ in range(STEPS):
                q = x.T @ x
                h = c * q
                h.diagonal().add_(b)
                h = q @ h
                h.diagonal().add_(a)
                x = x @ h
            done.append((x.T if case["rows"] < case["cols"] else x).contiguous())
        return torch.stack(done)
    act = {"silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
    x, wg, wu, wd = (s[k].double() for k in ("x", "wg", "wu", "wd"))
    if case["op"] != "backward":
        g, u = torch.einsum("td,fd->tf", x, wg), torch.einsum("td,fd->tf", x, wu)
        y = torch.einsum("tf,df->td", act(g) * u, wd)
        return {"y": y, "g": g, "u": u} if case["op"] == "train" else y
    # by automatic differentiation: through the product at the saved g and u, then through the
    # two projections
    g, u = (s[k].double().requires_grad_() for k in ("g", "u"))
    wd.requires_grad_()
    dg, du, dwd = torch.autograd.grad(torch.nn.functional.linear(act(g) * u, wd), (g, u, wd), s["dy"].double())
    x, wg, wu = (v.requires_grad_() for v in (x, wg, wu))
    dx, dwg, dwu = torch.autograd.grad((torch.nn.functional.linear(x, wg), torch.nn.functional.linear(x, wu)),
                                       (x, wg, wu), (dg, du))
    return {"dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}


def work(case):
    if case["op"] == "ortho":
        b, m, n = case["batch"], *sorted((case["rows"], case["cols"]))
        size = {"fp32": 4}.get(case["dtype"], 2)
        # x x^T and its square are symmetric: half of their products are enough
        return {"bytes": b * m * n * (size + 2), "flops": STEPS * b * (m * m * n + m * m * m + 2 * m * m * n)}
    t, d, f = case["tokens"], case["d"], case["f"]
    if case["op"] == "backward":
        return {"bytes": 2 * (3 * t * d + 6 * d * f + 2 * t * f), "flops": 12 * t * d * f}
    saved = 2 * t * f if case["op"] == "train" else 0
    return {"bytes": 2 * (2 * t * d + 3 * d * f + saved), "flops": 6 * t * d * f}
