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
from .norm import _cuda_tensor, _dtype, _rows_view, _stream


class Mxfp4Matrix:
    """rows x cols values in MXFP4 on one GPU, blocks of 32 along the columns.
    `codes` and `scales` are views of its buffer in the layout the C header
    gives."""

    def __init__(self, rows: int, cols: int, device):
        import torch

        cb, sb = ctypes.c_int64(), ctypes.c_int64()
        N.check(N.lib().mmn_mxfp4_size(rows, cols, ctypes.byref(cb), ctypes.byref(sb)))
        self.shape = (rows, cols)
        self.device = torch.device(device)
        self._buf = torch.empty(cb.value + sb.value, dtype=torch.uint8, device=self.device)
        self._code_bytes = cb.value
        ptr = self._buf.data_ptr()
        self._c = N.Mxfp4C(ptr, ptr + cb.value, rows, cols)

    @property
    def codes(self):
        """uint8 [rows, ceil(cols / 32) * 16], two elements to a byte."""
        return self._buf[:self._code_bytes].view(self.shape[0], -1) if self._code_bytes else \
            self._buf[:0].view(self.shape[0], 0)

    @property
    def scales(self):
        """uint8 scale bytes in blocks of 512 (128 rows x 4 blocks)."""
        return self._buf[self._code_bytes:]

    def dequantize(self, dtype=None, out=None):
        """The values, as float32 (default) or bfloat16; both hold them exactly."""
        import torch

        if out is None:
            out = torch.empty(self.shape, dtype=dtype or torch.float32, device=self.device)
            ld = self.shape[1]
        else:
            ld = _out_pitch(out, self.shape, dtype, self.device)
        N.check(N.lib().mmn_mxfp4_dequantize(ctypes.byref(self._c), out.data_ptr(), ld,
                                             _dtype(out, "out"), self.device.index,
                                             _stream(self.device)))
        return out


def _matrix(t, what: str):
    _cuda_tensor(t, what)
    if t.dim() != 2:
        raise ValueError(f"{what}: expected a matrix")
    return _rows_view(t, what)


def _out_pitch(out, shape, dtype, device) -> int:
    _cuda_tensor(out, "out", device)
    if tuple(out.shape) != tuple(shape) or (dtype is not None and out.dtype != dtype):
        raise N.ShapeError(N.MMN_E_SHAPE, f"out must be a {tuple(shape)} matrix"
                           + (f" of {dtype}" if dtype is not None else ""))
    return _rows_view(out, "out")[2]


def _mx(m, what: str, device=None) -> Mxfp4Matrix:
    if not isinstance(m, Mxfp4Matrix):
        raise TypeError(f"{what}: expected an Mxfp4Matrix")
    if device is not None and m.device != device:
        raise ValueError(f"{what} is on {m.device}, expected {device}")
    return m


def mxfp4_quantize(x, along: str = "rows", out=None):
    """x [rows, cols] to 4 bits. along="rows": the matrix itself (blocks along its
    rows); "cols": its transpose [cols, rows] (blocks down x's columns); "both": the
    pair, from one read of x. `out` (an Mxfp4Matrix, a pair for "both") is refilled
    in place, for weights whose copies keep their place from step to step."""
    if along not in ("rows", "cols", "both"):
        raise ValueError(f'along must be "rows", "cols" or "both", got {along!r}')
    rows, cols, ld = _matrix(x, "x")
    xd, dev = _dtype(x, "x"), x.device
    if out is None:
        q = Mxfp4Matrix(rows, cols, dev) if along != "cols" else None
        qt = Mxfp4Matrix(cols, rows, dev) if along != "rows" else None
    else:
        q, qt = {"rows": (out, None), "cols": (None, out)}[along] if along != "both" else out
        q = None if q is None else _mx(q, "out", dev)
        qt = None if qt is None else _mx(qt, "out", dev)
    N.check(N.lib().mmn_mxfp4_quantize(
        x.data_ptr(), ld, xd, rows, cols, None if q is None else ctypes.byref(q._c),
        None if qt is None else ctypes.byref(qt._c), dev.index, _stream(dev)))
    return (q, qt) if along == "both" else (q if q is not None else qt)


def mxfp4_matmul(a, b, out=None, out_dtype=None, accumulate: bool = False):
    """A B^T of two 4-bit matrices [m, k] and [n, k]: fp32 accumulation, the result
    bfloat16 (default) or float32, or in `out` (overwritten, or with
    accumulate=True added to)."""
    import torch

    _mx(a, "a")
    _mx(b, "b", a.device)
    shape = (a.shape[0], b.shape[0])
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs an out to add to")
        out = torch.empty(shape, dtype=out_dtype or torch.bfloat16, device=a.device)
        ld = shape[1]
    else:
        ld = _out_pitch(out, shape, out_dtype, a.device)
    N.check(N.lib().mmn_mxfp4_matmul(ctypes.byref(a._c), ctypes.byref(b._c), out.data_ptr(), ld,
                                     _dtype(out, "out"), int(bool(accumulate)), a.device.index,
                                     _stream(a.device)))
    return out


def mxfp4_linear(x, w, out=None, out_dtype=None):
    """x W^T with x [..., in] rounded to 4 bits on the way and w an Mxfp4Matrix
    [out, in]: the forward pass of a Linear layer. The result [..., out] has x's
    dtype, out_dtype, or goes to `out`."""
    import torch

    _cuda_tensor(x, "x")
    dev = x.device
    _mx(w, "w", dev)
    rows, cols, ld = _rows_view(x, "x")
    if cols != w.shape[1]:
        raise N.ShapeError(N.MMN_E_SHAPE, f"x has {cols} columns, w {w.shape[1]}")
    shape = tuple(x.shape[:-1]) + (w.shape[0],)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or x.dtype, device=dev)
        old = shape[-1]
    else:
        old = _out_pitch(out, shape, out_dtype, dev)
    xq = None if rows <= N.MXFP4_DIRECT_ROWS else Mxfp4Matrix(rows, cols, dev)
    N.check(N.lib().mmn_mxfp4_linear(x.data_ptr(), ld, _dtype(x, "x"), rows, ctypes.byref(w._c),
                                     None if xq is None else ctypes.byref(xq._c), out.data_ptr(),
                                     old, _dtype(out, "out"), dev.index, _stream(dev)))
    return out


def kernel_status(device: int = 0) -> None:
    """Waits for torch's current stream of the GPU and raises KernelTimeoutError
    when a product's kernel on it gave up a bounded wait."""
    import torch

    N.check(N.lib().mmn_kernel_status(device, _stream(torch.device("cuda", device))))
