"""The gated feed-forward block on B200: forward for serving and training, and its backward pass.

    g = x Wg^T    u = x Wu^T    h = act(g) * u    y = h Wd^T

x and y are [tokens, d_model], Wg and Wu [d_ff, d_model], Wd [d_model, d_ff] (a linear layer's
weight: outputs x inputs), all bf16 or all fp16, row-major with any row stride. As with the GEMM
plans (`_lib.GemmPlan`), a plan owns the workspaces, the caller owns operands and outputs, calls only
enqueue on a stream, and calls of one plan have to be ordered on the device: use one plan per
stream, do not replay two graphs captured from one plan at the same time, and keep a plan for as
long as graphs captured from it are replayed (they use its workspaces). Sums are kept in
fp32; h and the gradients of g and u are operands of a product and hold the operand type (in fp16
with its range: over 65504 they become infinite). There is no CPU fallback.

    plan = GatedFfnPlan(4096, d_model, d_ff, activation="silu", training=True)
    g, u = plan.new_saved(x.shape[0])
    plan.forward(x, wg, wu, wd, y, g, u)                        # g, u only when a backward pass follows
    plan.backward(x, wg, wu, wd, g, u, dy, dx, dwg, dwu, dwd)   # gradients are overwritten

The reference has no counterpart: its generated kernels compute one matrix product with no
epilogue (src/roller.py:47-68).
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib

# roller_ffn_io: the number of tokens (padded to eight bytes), then bases and row strides; the forward
# pass reads the first seven matrices of twelve
_FORWARD = struct.Struct("@i4x" + 7 * "Pq")
_BACKWARD = struct.Struct("@i4x" + 12 * "Pq")

ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH}


def check_matrix(t, name: str, dtype, device, rows: int, cols: int) -> int:
    """Row stride of a 2-D tensor after checking its type, device, shape and order."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, this plan needs {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, this plan is bound to {device}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({rows}, {cols})")
    ld, step = t.stride()
    if cols > 1 and step != 1:
        raise ValueError(f"{name} needs contiguous rows, its column stride is {step}")
    if rows < 2:        # there is no second row to step to: any stride is as good
        return (cols + 7) // 8 * 8
    if ld < cols:
        raise ValueError(f"{name} has overlapping rows (row stride {ld} for {cols} columns)")
    return ld


class GatedFfnPlan:
    """The block bound to widths, type, activation and device, for up to `max_tokens` tokens."""

    def __init__(self, max_tokens: int, d_model: int, d_ff: int, *, dtype=None, activation: str = "silu",
                 training: bool = False):
        import torch
        self._h = C.c_void_p()
        self._lib = _lib.load()
        dtype = torch.bfloat16 if dtype is None else dtype
        modes = {torch.bfloat16: _lib.MODE_BF16, torch.float16: _lib.MODE_F16}
        if dtype not in modes:
            raise TypeError(f"the block exists for bf16 and fp16 operands, not {dtype}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}")
        _lib.check_ints(max_tokens=max_tokens, d_model=d_model, d_ff=d_ff)
        self.max_tokens, self.d_model, self.d_ff = max_tokens, d_model, d_ff
        self.dtype, self.activation, self.training = dtype, activation, training
        _lib.check(self._lib.roller_b200_ffn_create(max_tokens, d_model, d_ff, modes[dtype],
                                                    ACTIVATIONS[activation],
                                                    _lib.FFN_TRAINING if training else 0, C.byref(self._h)),
                   "roller_b200_ffn_create")
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._io = _lib.FfnIo()
        self._io_ref = C.byref(self._io)

    def new_saved(self, tokens: int):
        """Two tensors for g and u, with rows that start on 32 bytes (the fast layout for any d_ff)."""
        import torch
        ld = (self.d_ff + 15) // 16 * 16
        return tuple(torch.empty(tokens, ld, dtype=self.dtype, device=self.device)[:, :self.d_ff]
                     for _ in range(2))

    def _mat(self, t, name: str, rows: int, cols: int):
        """Base and row stride of one operand, checked."""
        if t.dtype is not self.dtype or t.device != self.device or t.shape != (rows, cols):
            check_matrix(t, name, self.dtype, self.device, rows, cols)      # says what is wrong
        ld, step = t.stride()
        if step != 1 or ld < cols or rows < 2:
            ld = check_matrix(t, name, self.dtype, self.device, rows, cols)
        return t.data_ptr(), ld

    def _call(self, fn, name: str, stream) -> None:
        if not self._h:
            raise RuntimeError("the plan has been destroyed")
        status = _lib.on_device(self.device, stream, fn, self._h, self._io_ref)
        if status:
            _lib.check(status, name)

    def _tokens(self, x) -> int:
        tokens = x.shape[0]
        if tokens > self.max_tokens:
            raise _lib.RollerError(_lib.ERR_TOO_LARGE, f"{tokens} tokens, the plan was made for {self.max_tokens}")
        return tokens

    def forward(self, x, wg, wu, wd, y, g=None, u=None, stream=None) -> None:
        """Writes y, and g and u when they are given (both or neither)."""
        if (g is None) != (u is None):
            raise ValueError("g and u are written together: give both or neither")
        n, d, f, mat = self._tokens(x), self.d_model, self.d_ff, self._mat
        saved = (0, 0, 0, 0) if g is None else (*mat(g, "g", n, f), *mat(u, "u", n, f))
        _FORWARD.pack_into(self._io, 0, n, *mat(x, "x", n, d), *mat(wg, "wg", f, d), *mat(wu, "wu", f, d),
                           *mat(wd, "wd", d, f), *mat(y, "y", n, d), *saved)
        self._call(self._lib.roller_b200_ffn_forward, "roller_b200_ffn_forward", stream)

    def backward(self, x, wg, wu, wd, g, u, dy, dx, dwg, dwu, dwd, stream=None) -> None:
        """Writes dx, dwg, dwu and dwd (not added to) for the gradient dy of y. g and u are what
        `forward` wrote for the same x and weights. The plan has to be made with training=True."""
        n, d, f, mat = self._tokens(x), self.d_model, self.d_ff, self._mat
        _BACKWARD.pack_into(self._io, 0, n, *mat(x, "x", n, d), *mat(wg, "wg", f, d), *mat(wu, "wu", f, d),
                            *mat(wd, "wd", d, f), 0, 0, *mat(g, "g", n, f), *mat(u, "u", n, f), *mat(dy, "dy", n, d),
                            *mat(dx, "dx", n, d), *mat(dwg, "dwg", f, d), *mat(dwu, "dwu", f, d), *mat(dwd, "dwd", d, f))
        self._call(self._lib.roller_b200_ffn_backward, "roller_b200_ffn_backward", stream)

    def check_status(self) -> None:
        """Raises RollerError(TIMEOUT) if a launch since the last check gave up on a device-side
        wait. Synchronises the plan's device."""
        _lib.check_plan_status(self.device, self._lib.roller_b200_ffn_status, self._h, "roller_b200_ffn_status")

    def destroy(self) -> None:
        if self._h:
            self._lib.roller_b200_ffn_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass
