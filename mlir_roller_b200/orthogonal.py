"""Orthogonalising the update of a weight matrix by Newton-Schulz products, as Muon does.

    x = g / (|g| + eps);  `steps` times:  x = a x + (b p + c p p) x  with  p = x x^T

drives the singular values of each matrix g of a batch towards one and leaves its singular
vectors. |g| is the Frobenius norm. Inputs are fp32, bf16 or fp16, [rows, cols] or [batch, rows, cols] with
contiguous rows and any other strides; results are bf16. The products are fp16 with fp32 sums and
x is carried with 22 bits in between, so that a matrix of low rank comes out as clean as a full
one (about 2e-3 of |x| against 64 bits, most of it the last rounding to bf16; up to 1.4e-2 with fewer
than eight rows or columns, where one singular value at a steep place of the iteration is all there
is). Where |g| is under about 1e-5 eps the result, itself close to zero, keeps only an absolute
accuracy.

A plan owns the workspaces; calls only enqueue on a stream, and calls of one plan have to be ordered
on the device. Graphs captured from a plan need it for as long as they are replayed. There is no CPU fallback. The reference has no counterpart: it multiplies two matrices
(src/roller.py:47-68).
"""
from __future__ import annotations

import ctypes as C

from . import _lib

# the quintic that Muon uses: steep at zero (weak directions grow 3.4-fold a step), and around
# one it stays between about 0.7 and 1.2
MUON_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


class OrthogonalPlan:
    """The iteration bound to a shape, input type and device."""

    def __init__(self, rows: int, cols: int, *, batch: int = 1, dtype=None, steps: int = 5,
                 coefficients=MUON_COEFFICIENTS, eps: float = 1e-7):
        import torch
        self._h = C.c_void_p()
        self._lib = _lib.load()
        dtype = torch.bfloat16 if dtype is None else dtype
        types = {torch.float32: _lib.ORTHO_IN_F32, torch.bfloat16: _lib.ORTHO_IN_BF16,
                 torch.float16: _lib.ORTHO_IN_F16}
        if dtype not in types:
            raise TypeError(f"inputs are fp32, bf16 or fp16, not {dtype}")
        _lib.check_ints(batch=batch, rows=rows, cols=cols, steps=steps)
        self.batch, self.rows, self.cols, self.dtype = batch, rows, cols, dtype
        self._out_dtype = torch.bfloat16
        a, b, c = coefficients
        _lib.check(self._lib.roller_b200_ortho_create(batch, rows, cols, types[dtype], steps, a, b, c, eps,
                                                      C.byref(self._h)), "roller_b200_ortho_create")
        self.device = torch.device("cuda", torch.cuda.current_device())

    def _strides(self, t, name: str, dtype):
        if t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, this plan needs {dtype}")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, this plan is bound to {self.device}")
        shape = tuple(t.shape)
        if shape != (self.batch, self.rows, self.cols) and not (self.batch == 1 and shape == (self.rows, self.cols)):
            raise ValueError(f"{name} has shape {shape}, expected ({self.batch}, {self.rows}, {self.cols})")
        ld, step = t.stride()[-2:]
        if self.cols > 1 and step != 1:
            raise ValueError(f"{name} needs contiguous rows, its column stride is {step}")
        zs = t.stride(0) if self.batch > 1 else 0
        return ld, zs

    def run(self, g, out, stream=None) -> None:
        """Writes the orthogonalised g into out (bf16, same shape). g is not changed."""
        if not self._h:
            raise RuntimeError("the plan has been destroyed")
        ld_g, zs_g = self._strides(g, "g", self.dtype)
        ld_o, zs_o = self._strides(out, "out", self._out_dtype)
        _lib.check(_lib.on_device(self.device, stream, self._lib.roller_b200_ortho_run, self._h, g.data_ptr(), ld_g,
                                  zs_g, out.data_ptr(), ld_o, zs_o), "roller_b200_ortho_run")

    def check_status(self) -> None:
        """Raises RollerError(TIMEOUT) if a launch since the last check gave up on a device-side
        wait. Synchronises the plan's device."""
        _lib.check_plan_status(self.device, self._lib.roller_b200_ortho_status, self._h, "roller_b200_ortho_status")

    def destroy(self) -> None:
        if self._h:
            self._lib.roller_b200_ortho_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass
