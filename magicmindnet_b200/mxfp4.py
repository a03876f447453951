"""4-bit microscaled matrices and their products (mmn_mxfp4_* in
include/mmn_optim.h): OCP Microscaling MXFP4, 32 e2m1 elements to one power-of-two
scale, multiplied on the tensor cores with fp32 accumulation.

A Linear layer of the reference (weights [out, in], crates/mmn-nn/src/lib.rs:305-307)
reads, with ``w = mxfp4_quantize(W)`` and ``wt = mxfp4_quantize(W, "cols")``:

    y  = mxfp4_linear(x, w)                        # forward
    dyq, dyt = mxfp4_quantize(dy, "both")
    dx = mxfp4_matmul(dyq, wt)                     # dy W
    mxfp4_matmul(dyt, mxfp4_quantize(x, "cols"), out=step.grad(slot))   # dW

Arrays are CUDA torch tensors of float32 or bfloat16; work is enqueued on
torch's current stream of their GPU.
"""
from __future__ import annotations

import ctypes

from . import _native as N
from .norm import _dtype, _gpu_of, _on_gpu, _rows_view, _stream, _torch


class Mxfp4Matrix:
    """rows x cols values in MXFP4 on one GPU, blocks of 32 along the columns.
    `codes` and `scales` are views of its buffer in the layout the C header
    gives."""

    __slots__ = ("shape", "device", "_buf", "_code_bytes", "_c", "_index", "__weakref__")

    def __init__(self, rows: int, cols: int, device):
        torch = _torch()
        # the sizes of mmn_mxfp4_size, without the call
        code_bytes = rows * ((cols + 31) // 32 * 16)
        total = code_bytes + ((rows + 127) // 128 * ((cols + 255) // 256) * 1024)
        self.shape = (rows, cols)
        self._buf = buf = torch.empty(total, dtype=torch.uint8, device=device)
        self.device = buf.device
        self._index = buf.get_device()
        self._code_bytes = code_bytes
        ptr = buf.data_ptr()
        self._c = N.Mxfp4C(ptr, ptr + code_bytes, rows, cols)

    @property
    def codes(self):
        """uint8 [rows, ceil(cols / 32) * 16], two elements to a byte."""
        return self._buf[:self._code_bytes].view(self.shape[0], (self.shape[1] + 31) // 32 * 16)

    @property
    def scales(self):
        """uint8 scale bytes in blocks of 512 (128 rows x 4 blocks)."""
        return self._buf[self._code_bytes:]

    def dequantize(self, dtype=None, out=None):
        """The values, as float32 (default) or bfloat16; both hold them exactly."""
        if out is None:
            torch = _torch()
            out = torch.empty(*self.shape, dtype=dtype or torch.float32, device=self.device)
            ld = self.shape[1]
        else:
            ld = _out_pitch(out, self.shape, dtype, self._index)
        N.check(N.lib().mmn_mxfp4_dequantize(self._c, out.data_ptr(), ld, _dtype(out, "out"),
                                             self._index, _stream(self._index)))
        return out


def _out_pitch(out, shape, dtype, index: int) -> int:
    _on_gpu(out, "out", index)
    if out.shape != shape or (dtype is not None and out.dtype != dtype):
        raise N.ShapeError(N.MMN_E_SHAPE, f"out must be a {tuple(shape)} matrix"
                           + (f" of {dtype}" if dtype is not None else ""))
    return _rows_view(out, "out")[2]


def _mx(m, what: str, index=None) -> Mxfp4Matrix:
    if not isinstance(m, Mxfp4Matrix):
        raise TypeError(f"{what}: expected an Mxfp4Matrix")
    if index is not None and m._index != index:
        raise ValueError(f"{what} is on {m.device}, expected cuda:{index}")
    return m


def mxfp4_quantize(x, along: str = "rows", out=None):
    """x [rows, cols] to 4 bits. along="rows": the matrix itself (blocks along its
    rows); "cols": its transpose [cols, rows] (blocks down x's columns); "both": the
    pair, from one read of x. `out` (an Mxfp4Matrix, a pair for "both") is refilled
    in place, for weights whose copies keep their place from step to step."""
    if along not in ("rows", "cols", "both"):
        raise ValueError(f'along must be "rows", "cols" or "both", got {along!r}')
    index = _gpu_of(x, "x")
    if x.dim() != 2:
        raise ValueError("x: expected a matrix")
    rows, cols, ld = _rows_view(x, "x")
    xd = _dtype(x, "x")
    if out is None:
        dev = x.device
        q = Mxfp4Matrix(rows, cols, dev) if along != "cols" else None
        qt = Mxfp4Matrix(cols, rows, dev) if along != "rows" else None
    else:
        q, qt = {"rows": (out, None), "cols": (None, out)}[along] if along != "both" else out
        q = None if q is None else _mx(q, "out", index)
        qt = None if qt is None else _mx(qt, "out", index)
    N.check(N.lib().mmn_mxfp4_quantize(
        x.data_ptr(), ld, xd, rows, cols, None if q is None else q._c,
        None if qt is None else qt._c, index, _stream(index)))
    return (q, qt) if along == "both" else (q if q is not None else qt)


def mxfp4_matmul(a, b, out=None, out_dtype=None, accumulate: bool = False):
    """A B^T of two 4-bit matrices [m, k] and [n, k]: fp32 accumulation, the result
    bfloat16 (default) or float32, or in `out` (overwritten, or with
    accumulate=True added to)."""
    index = _mx(a, "a")._index
    _mx(b, "b", index)
    shape = (a.shape[0], b.shape[0])
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs an out to add to")
        torch = _torch()
        out = torch.empty(*shape, dtype=out_dtype or torch.bfloat16, device=a.device)
        ld = shape[1]
    else:
        ld = _out_pitch(out, shape, out_dtype, index)
    N.check(N.lib().mmn_mxfp4_matmul(a._c, b._c, out.data_ptr(), ld, _dtype(out, "out"),
                                     bool(accumulate), index, _stream(index)))
    return out


def mxfp4_linear(x, w, out=None, out_dtype=None):
    """x W^T with x [..., in] rounded to 4 bits on the way and w an Mxfp4Matrix
    [out, in]: the forward pass of a Linear layer. The result [..., out] has x's
    dtype, out_dtype, or goes to `out`."""
    index = _gpu_of(x, "x")
    _mx(w, "w", index)
    rows, cols, ld = _rows_view(x, "x")
    if cols != w.shape[1]:
        raise N.ShapeError(N.MMN_E_SHAPE, f"x has {cols} columns, w {w.shape[1]}")
    shape = (*x.shape[:-1], w.shape[0])
    if out is None:
        out = _torch().empty(*shape, dtype=out_dtype or x.dtype, device=x.device)
        old = shape[-1]
    else:
        old = _out_pitch(out, shape, out_dtype, index)
    xq = None if rows <= N.MXFP4_DIRECT_ROWS else Mxfp4Matrix(rows, cols, x.device)
    N.check(N.lib().mmn_mxfp4_linear(x.data_ptr(), ld, _dtype(x, "x"), rows, w._c,
                                     None if xq is None else xq._c, out.data_ptr(), old,
                                     _dtype(out, "out"), index, _stream(index)))
    return out


def kernel_status(device: int = 0) -> None:
    """Waits for torch's current stream of the GPU and raises KernelTimeoutError
    when a kernel of these operators on it gave up a bounded wait since the last
    such report. OptimizerStep.sync and .step_host raise it too, each step for itself."""
    _torch()
    N.check(N.lib().mmn_kernel_status(device, _stream(device)))
