"""Layer norm beside the optimizer step (mmn_layer_norm* in include/mmn_optim.h):
the LayerNorm layer of crates/mmn-nn/src/lib.rs, whose gamma and beta grads
crates/mmn-models/src/chatbot.rs:118-206 hands to AdamW.

Arrays are CUDA torch tensors of float32 or bfloat16; work is enqueued on
torch's current stream of their GPU. One token's call is bound by the host, so
the checks here take no detours: 22 us a call with a stream object, a device
object and a shape tuple for every tensor, about half without.
"""
from __future__ import annotations

import ctypes
import functools

from . import _native as N
from .optim import _CUDA_STREAM_LEGACY

_t = None          # torch, once a call needs it
_dtypes = {}       # torch dtype -> MMN_DTYPE_*
_raw_stream = None


def _torch():
    """torch and the tables that need it, on first use."""
    global _t, _raw_stream
    if _t is None:
        import torch

        _dtypes[torch.float32] = N.DTYPE_F32
        _dtypes[torch.bfloat16] = N.DTYPE_BF16
        # the stream handle without a Stream object around it, where torch has it
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _t = torch
    return _t


def _stream(index: int) -> int:
    """torch's current stream of a GPU; its default stream goes as cudaStreamLegacy."""
    return _raw_stream(index) or _CUDA_STREAM_LEGACY


def _dtype(t, what: str) -> int:
    d = _dtypes.get(t.dtype)
    if d is None:
        raise TypeError(f"{what}: expected a float32 or bfloat16 tensor, got {t.dtype}")
    return d


def _gpu_of(t, what: str) -> int:
    """The GPU of a CUDA tensor."""
    if not isinstance(t, (_t or _torch()).Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: expected a CUDA tensor")
    return t.get_device()


def _on_gpu(t, what: str, index: int) -> None:
    if _gpu_of(t, what) != index:
        raise ValueError(f"{what} is on {t.device}, expected cuda:{index}")


def _rows_view(t, what: str):
    """(rows, cols, distance between rows) of a tensor taken as the matrix of its
    last axis: that axis contiguous, the leading ones evenly spaced."""
    shape = t.shape
    if not shape:
        raise ValueError(f"{what}: expected at least one axis")
    cols = shape[-1]
    if cols and t.is_contiguous():
        return t.numel() // cols, cols, cols
    rows = 1
    for n in shape[:-1]:
        rows *= n
    if t.is_contiguous():
        return rows, cols, cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    seen, ld = 1, None
    for n, s in zip(reversed(shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != ld * seen:
            raise ValueError(f"{what}: the rows must be evenly spaced")
        seen *= n
    if ld is None:
        return rows, cols, cols
    if ld < cols:
        raise ValueError(f"{what}: rows that share memory (an expanded tensor); pass a copy")
    return rows, cols, ld


def _vector(t, n: int, what: str, index: int) -> int:
    """dtype of a contiguous vector of n elements on a GPU."""
    if isinstance(t, _t.Tensor) and t.get_device() == index and t.dim() == 1 \
            and t.numel() == n and t.is_contiguous():
        return _dtypes.get(t.dtype) or _dtype(t, what)
    _on_gpu(t, what, index)
    raise ValueError(f"{what}: expected a contiguous vector of {n} elements")


def layer_norm(x, gamma, beta, eps: float = 1e-5, out_dtype=None, out=None):
    """(y, mean, rstd) of a layer norm over the last axis: y = (x - mean) * rstd *
    gamma + beta with rstd = 1 / sqrt(var + eps). y has out_dtype (x's dtype by
    default) or goes to `out`, which may be x; mean and rstd are float32 with
    x's leading shape, for layer_norm_backward."""
    index = _gpu_of(x, "x")
    rows, cols, ld = _rows_view(x, "x")
    xd = _dtype(x, "x")
    pd = _vector(gamma, cols, "gamma", index)
    if _vector(beta, cols, "beta", index) != pd:
        raise TypeError("gamma and beta must have one dtype")
    if out is None:
        if ld == cols:
            out = _t.empty_like(x, dtype=out_dtype)
        else:
            out = _t.empty(*x.shape, dtype=out_dtype or x.dtype, device=x.device)
        old = cols
    else:
        _on_gpu(out, "out", index)
        if out.shape != x.shape or (out_dtype is not None and out.dtype != out_dtype):
            raise N.ShapeError(N.MMN_E_SHAPE, "out must have x's shape (and out_dtype)")
        old = _rows_view(out, "out")[2]
    dev = x.device
    if x.dim() == 2:
        mean = _t.empty(rows, dtype=_t.float32, device=dev)
        rstd = _t.empty(rows, dtype=_t.float32, device=dev)
    else:
        mean = _t.empty(x.shape[:-1], dtype=_t.float32, device=dev)
        rstd = _t.empty(x.shape[:-1], dtype=_t.float32, device=dev)
    if cols == 0:
        mean.zero_()
        rstd.fill_(float("inf") if eps == 0 else eps ** -0.5)
    N.check(N.lib().mmn_layer_norm(
        x.data_ptr(), ld, xd, gamma.data_ptr(), beta.data_ptr(), pd, eps, rows, cols,
        out.data_ptr(), old, _dtype(out, "out"), mean.data_ptr(), rstd.data_ptr(), index,
        _stream(index)))
    return out, mean, rstd


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows: int, cols: int, index: int) -> int:
    """mmn_layer_norm_backward_workspace, which depends on nothing else."""
    need = ctypes.c_int64()
    N.check(N.lib().mmn_layer_norm_backward_workspace(rows, cols, index, need))
    return need.value


def layer_norm_backward(dy, x, gamma, mean, rstd, dgamma=None, dbeta=None,
                        accumulate: bool = False, out=None):
    """(dx, dgamma, dbeta) of layer_norm from dy and the forward pass's x, gamma,
    mean and rstd. dgamma and dbeta are new float32 vectors, or the ones given
    (float32 or bfloat16, such as OptimizerStep.grad views), which are
    overwritten, or with accumulate=True added to. dx has x's dtype or goes to
    `out`, which may be dy or x."""
    index = _gpu_of(x, "x")
    _on_gpu(dy, "dy", index)
    rows, cols, ld = _rows_view(x, "x")
    if dy.shape != x.shape:
        raise N.ShapeError(N.MMN_E_SHAPE, "dy and x must have one shape")
    dld = _rows_view(dy, "dy")[2]
    xd, dd = _dtype(x, "x"), _dtype(dy, "dy")
    pd = _vector(gamma, cols, "gamma", index)
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        _on_gpu(t, what, index)
        if t.dtype != _t.float32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{what}: expected {rows} contiguous float32 values")
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate=True needs dgamma and dbeta to add to")
    dev = x.device
    if dgamma is None and dbeta is None:
        dgamma = _t.empty(cols, dtype=_t.float32, device=dev)
        dbeta = _t.empty(cols, dtype=_t.float32, device=dev)
        gd = N.DTYPE_F32
    else:
        if dgamma is None:
            dgamma = _t.empty(cols, dtype=dbeta.dtype, device=dev)
        elif dbeta is None:
            dbeta = _t.empty(cols, dtype=dgamma.dtype, device=dev)
        gd = _vector(dgamma, cols, "dgamma", index)
        if _vector(dbeta, cols, "dbeta", index) != gd:
            raise TypeError("dgamma and dbeta must have one dtype")
    if out is None:
        out = _t.empty_like(x) if ld == cols else _t.empty(*x.shape, dtype=x.dtype, device=dev)
        old = cols
    else:
        _on_gpu(out, "out", index)
        if out.shape != x.shape or out.dtype != x.dtype:
            raise N.ShapeError(N.MMN_E_SHAPE, "out must have x's shape and dtype")
        old = _rows_view(out, "out")[2]
    need = _workspace_bytes(rows, cols, index)
    ws = _t.empty(need, dtype=_t.uint8, device=dev)
    N.check(N.lib().mmn_layer_norm_backward(
        dy.data_ptr(), dld, dd, x.data_ptr(), ld, xd, gamma.data_ptr(), pd, mean.data_ptr(),
        rstd.data_ptr(), rows, cols, out.data_ptr(), old, dgamma.data_ptr(), dbeta.data_ptr(), gd,
        bool(accumulate), ws.data_ptr(), need, index, _stream(index)))
    return out, dgamma, dbeta
