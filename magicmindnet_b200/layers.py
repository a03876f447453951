"""Layers whose weights are slots of an OptimizerStep: LayerNorm and a Linear
that multiplies in 4 bits (crates/mmn-nn/src/lib.rs LayerNorm and Linear; the
slots are those of ``chatbot_param_order``: ln1/ln2 gamma and beta, and the q, k,
v, out, ffn, ffn2 matrices).

``forward`` keeps what ``backward`` needs; ``backward`` returns the input's
gradient and writes the weights' gradients into the step's grad slots, where
``OptimizerStep.step`` reads them. ``accumulate=True`` adds to the slots instead
(the second and later micro-batches of a step). A layer holds one forward pass
at a time: the next one before its ``backward`` (or ``discard``) is refused.
``training=False`` holds nothing. Work is enqueued on torch's current stream,
which must be the one the step was made on (or ordered with it), as for
``OptimizerStep.param`` and ``.grad`` views. After the step is closed a layer
refuses its calls: the slots are gone.
"""
from __future__ import annotations

from . import _native as N
from .mxfp4 import Mxfp4Matrix, mxfp4_linear, mxfp4_matmul, mxfp4_quantize
from .norm import layer_norm, layer_norm_backward


class _Layer:
    """What a forward pass leaves for its backward pass."""

    _saved = None

    def _open(self) -> None:
        if not self.step._h:
            raise N.MmnError(N.MMN_E_STATE, "the step is closed, its slots are gone")

    def _hold(self, saved) -> None:
        self._saved = saved

    def _free(self) -> None:
        if self._saved is not None:
            raise N.MmnError(N.MMN_E_STATE, "a forward pass still waits for its backward pass "
                                            "(discard() drops it)")

    def _held(self):
        if self._saved is None:
            raise N.MmnError(N.MMN_E_STATE, "backward without a forward pass")
        return self._saved

    def discard(self) -> None:
        """Drops the forward pass that waits for its backward pass, if any."""
        self._saved = None


class LayerNorm(_Layer):
    """Layer norm with the gain in `gamma_slot` and the shift in `beta_slot`."""

    def __init__(self, step, gamma_slot: int, beta_slot: int, eps: float = 1e-5):
        gs, bs = step.shapes[gamma_slot], step.shapes[beta_slot]
        if len(gs) != 1 or gs != bs:
            raise N.ShapeError(N.MMN_E_SHAPE, f"gamma {gs} and beta {bs} must be equal vectors")
        self.step, self.gamma_slot, self.beta_slot, self.eps = step, gamma_slot, beta_slot, eps
        self._gamma, self._beta = step.forward_param(gamma_slot), step.forward_param(beta_slot)
        self._dgamma, self._dbeta = step.grad(gamma_slot), step.grad(beta_slot)

    def forward(self, x, training: bool = True, out_dtype=None):
        """The norm of x [..., d]; x itself is kept for backward and must not change
        before it."""
        self._open()
        if training:
            self._free()
        y, mean, rstd = layer_norm(x, self._gamma, self._beta, self.eps, out_dtype)
        if training:
            self._hold((x, mean, rstd))
        return y

    def backward(self, dy, accumulate: bool = False):
        self._open()
        x, mean, rstd = self._held()
        dx, _, _ = layer_norm_backward(dy, x, self._gamma, mean, rstd, self._dgamma, self._dbeta,
                                       accumulate)
        self._saved = None
        return dx


class Linear(_Layer):
    """y = x W^T with W [out, in] in `slot`. The forward pass and both gradient
    products run on 4-bit operands; the weight's 4-bit copies (W for the forward
    pass, W transposed for the input's gradient) are made by ``refresh``, which
    is called once here and again after every ``OptimizerStep.step``,
    ``step_host`` or ``set_param``: ``forward`` refuses copies that are older. (What
    is written straight into an ``OptimizerStep.param`` view it cannot see.)"""

    def __init__(self, step, slot: int):
        shape = step.shapes[slot]
        if len(shape) != 2:
            raise N.ShapeError(N.MMN_E_SHAPE, f"slot {slot} is {shape}, not a matrix")
        import torch

        self.step, self.slot = step, slot
        self._param, self._grad = step.forward_param(slot), step.grad(slot)
        dev = torch.device("cuda", step.device)
        self.w = Mxfp4Matrix(shape[0], shape[1], dev)
        self.wt = Mxfp4Matrix(shape[1], shape[0], dev)
        self.refresh()

    def refresh(self) -> None:
        """Both 4-bit copies from the slot's present values, in place (one read). On
        several ranks: after the fence that ends the step's parameter exchange."""
        self._open()
        version = self.step.param_version
        mxfp4_quantize(self._param, "both", out=(self.w, self.wt))
        self._version = version

    def forward(self, x, training: bool = True, out_dtype=None):
        """x [..., in] -> [..., out]; training=False keeps nothing for backward."""
        self._open()
        if self._version != self.step.param_version:
            raise N.MmnError(N.MMN_E_STATE, "the parameters have changed since the weight's 4-bit "
                                            "copies were made (refresh() renews them)")
        if not training:
            return mxfp4_linear(x, self.w, out_dtype=out_dtype)
        if x.shape[-1] != self.w.shape[1]:
            raise N.ShapeError(N.MMN_E_SHAPE,
                               f"x has {x.shape[-1]} columns, the weight {self.w.shape[1]}")
        self._free()
        xq, xt = mxfp4_quantize(_as_matrix(x), "both")
        y = mxfp4_matmul(xq, self.w, out_dtype=out_dtype or x.dtype)
        self._hold((xt, x.dtype, x.shape))
        return y.view(tuple(x.shape[:-1]) + (self.w.shape[0],))

    def backward(self, dy, accumulate: bool = False):
        self._open()
        xt, dtype, shape = self._held()
        want = tuple(shape[:-1]) + (self.w.shape[0],)
        if tuple(dy.shape) != want:
            raise N.ShapeError(N.MMN_E_SHAPE, f"dy is {tuple(dy.shape)}, expected {want}")
        dyq, dyt = mxfp4_quantize(_as_matrix(dy), "both")
        # dx first: its room may be missing, and a backward pass that failed leaves the
        # slot as it was, so that it can be called again
        dx = mxfp4_matmul(dyq, self.wt, out_dtype=dtype)
        mxfp4_matmul(dyt, xt, out=self._grad, accumulate=accumulate)
        self._saved = None
        return dx.view(shape)


def _as_matrix(t):
    """[..., n] as [rows, n]; a view where the strides allow one."""
    rows = 1
    for n in t.shape[:-1]:
        rows *= n
    return t.reshape(rows, t.shape[-1])
