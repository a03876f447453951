"""Layer norm beside the optimizer step (mmn_layer_norm* in include/mmn_optim.h):
the LayerNorm layer of crates/mmn-nn/src/lib.rs, whose gamma and beta grads
crates/mmn-models/src/chatbot.rs:118-206 hands to AdamW.

Arrays are CUDA torch tensors of float32 or bfloat16; work is enqueued on
torch's current stream of their GPU.
"""
from __future__ import annotations

import ctypes

from . import _native as N
from .optim import _CUDA_STREAM_LEGACY


def _dtype(t, what: str) -> int:
    import torch

    if t.dtype == torch.float32:
        return N.DTYPE_F32
    if t.dtype == torch.bfloat16:
        return N.DTYPE_BF16
    raise TypeError(f"{what}: expected a float32 or bfloat16 tensor, got {t.dtype}")


def _cuda_tensor(t, what: str, device=None):
    """A CUDA tensor (of `device` when one is given), else an error."""
    import torch

    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: expected a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, expected {device}")


def _rows_view(t, what: str):
    """(rows, cols, distance between rows) of a tensor taken as the matrix of its
    last axis: that axis contiguous, the leading ones evenly spaced."""
    if t.dim() == 0:
        raise ValueError(f"{what}: expected at least one axis")
    cols = t.shape[-1]
    if t.is_contiguous():
        return _lead(t), cols, cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    rows, ld = 1, None
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if ld is None:
            ld = s
        elif s != ld * rows:
            raise ValueError(f"{what}: the rows must be evenly spaced")
        rows *= n
    if ld is None:
        return rows, cols, cols
    if ld < cols:
        raise ValueError(f"{what}: rows that share memory (an expanded tensor); pass a copy")
    return rows, cols, ld


def _lead(t) -> int:
    n = 1
    for s in t.shape[:-1]:
        n *= s
    return n


def _vector(t, n: int, what: str, device) -> int:
    """dtype of a contiguous 1-D tensor of n elements on `device`."""
    _cuda_tensor(t, what, device)
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous vector of {n} elements")
    return _dtype(t, what)


def _stream(device) -> int:
    """torch's current stream of a device; its default stream goes as cudaStreamLegacy."""
    import torch

    return torch.cuda.current_stream(device).cuda_stream or _CUDA_STREAM_LEGACY


def layer_norm(x, gamma, beta, eps: float = 1e-5, out_dtype=None, out=None):
    """(y, mean, rstd) of a layer norm over the last axis: y = (x - mean) * rstd *
    gamma + beta with rstd = 1 / sqrt(var + eps). y has out_dtype (x's dtype by
    default) or goes to `out`, which may be x; mean and rstd are float32 with
    x's leading shape, for layer_norm_backward."""
    import torch

    _cuda_tensor(x, "x")
    dev = x.device
    rows, cols, ld = _rows_view(x, "x")
    xd = _dtype(x, "x")
    pd = _vector(gamma, cols, "gamma", dev)
    if _vector(beta, cols, "beta", dev) != pd:
        raise TypeError("gamma and beta must have one dtype")
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=dev)
        old = cols
    else:
        _cuda_tensor(out, "out", dev)
        if out.shape != x.shape or (out_dtype is not None and out.dtype != out_dtype):
            raise N.ShapeError(N.MMN_E_SHAPE, "out must have x's shape (and out_dtype)")
        old = _rows_view(out, "out")[2]
    stats = torch.empty((2,) + tuple(x.shape[:-1]), dtype=torch.float32, device=dev)
    mean, rstd = stats[0], stats[1]
    if cols == 0:
        mean.zero_()
        rstd.fill_(float("inf") if eps == 0 else eps ** -0.5)
    N.check(N.lib().mmn_layer_norm(
        x.data_ptr(), ld, xd, gamma.data_ptr(), beta.data_ptr(), pd, eps, rows, cols,
        out.data_ptr(), old, _dtype(out, "out"), mean.data_ptr(), rstd.data_ptr(), dev.index,
        _stream(dev)))
    return out, mean, rstd


def layer_norm_backward(dy, x, gamma, mean, rstd, dgamma=None, dbeta=None,
                        accumulate: bool = False, out=None):
    """(dx, dgamma, dbeta) of layer_norm from dy and the forward pass's x, gamma,
    mean and rstd. dgamma and dbeta are new float32 vectors, or the ones given
    (float32 or bfloat16, such as OptimizerStep.grad views), which are
    overwritten, or with accumulate=True added to. dx has x's dtype or goes to
    `out`, which may be dy or x."""
    import torch

    _cuda_tensor(x, "x")
    dev = x.device
    _cuda_tensor(dy, "dy", dev)
    rows, cols, ld = _rows_view(x, "x")
    if dy.shape != x.shape:
        raise N.ShapeError(N.MMN_E_SHAPE, "dy and x must have one shape")
    dld = _rows_view(dy, "dy")[2]
    xd, dd = _dtype(x, "x"), _dtype(dy, "dy")
    pd = _vector(gamma, cols, "gamma", dev)
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        _cuda_tensor(t, what, dev)
        if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{what}: expected {rows} contiguous float32 values")
    if accumulate and (dgamma is None or dbeta is None):
        raise ValueError("accumulate=True needs dgamma and dbeta to add to")
    if dgamma is None:
        dgamma = torch.empty(cols, dtype=torch.float32 if dbeta is None else dbeta.dtype,
                             device=dev)
    if dbeta is None:
        dbeta = torch.empty(cols, dtype=dgamma.dtype, device=dev)
    gd = _vector(dgamma, cols, "dgamma", dev)
    if _vector(dbeta, cols, "dbeta", dev) != gd:
        raise TypeError("dgamma and dbeta must have one dtype")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
        old = cols
    else:
        _cuda_tensor(out, "out", dev)
        if out.shape != x.shape or out.dtype != x.dtype:
            raise N.ShapeError(N.MMN_E_SHAPE, "out must have x's shape and dtype")
        old = _rows_view(out, "out")[2]
    L = N.lib()
    need = ctypes.c_int64()
    N.check(L.mmn_layer_norm_backward_workspace(rows, cols, dev.index, ctypes.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
    N.check(L.mmn_layer_norm_backward(
        dy.data_ptr(), dld, dd, x.data_ptr(), ld, xd, gamma.data_ptr(), pd, mean.data_ptr(),
        rstd.data_ptr(), rows, cols, out.data_ptr(), old, dgamma.data_ptr(), dbeta.data_ptr(), gd,
        int(bool(accumulate)), ws.data_ptr(), need.value, dev.index, _stream(dev)))
    return out, dgamma, dbeta
