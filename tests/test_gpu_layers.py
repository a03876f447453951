"""LayerNorm and Linear bound to OptimizerStep slots: forward, backward, the step
and the refreshed copies, together as a training loop runs them."""
import pytest

from test_gpu_layer_norm import check_backward, check_forward
from test_gpu_mxfp4 import check_product, data, plain_values

pytestmark = pytest.mark.gpu

D, FFN, TOKENS = 192, 520, 75
NAMES = [("ffn2", (D, FFN)), ("ffn", (FFN, D)), ("ln2.gamma", (D,)), ("ln2.beta", (D,))]


def make_step(mmn, **kw):
    import torch

    cfg = mmn.StepConfig(adamw=mmn.AdamWConfig(lr=1e-2), muon=mmn.MuonConfig(), **kw)
    step = mmn.OptimizerStep([(k, s) for k, (_, s) in enumerate(NAMES)], cfg)
    gen = torch.Generator(device="cuda").manual_seed(0)
    for k, (name, s) in enumerate(NAMES):
        v = 0.05 * torch.randn(s, device="cuda", generator=gen)
        if name.endswith("gamma"):
            v += 1
        step.set_param(k, v.cpu().numpy())
    return step


@pytest.mark.parametrize("grad_dtype", ["f32", "bf16"])
def test_block_trains_through_the_step(mmn, grad_dtype):
    """x -> layer norm -> ffn -> ffn2, two micro-batches accumulated into the slots,
    the step, the refreshed copies: every stage against its 64-bit form on the
    values that entered it, for two steps."""
    import torch

    step = make_step(mmn, grad_dtype=grad_dtype)
    ln, ffn, ffn2 = mmn.LayerNorm(step, 2, 3), mmn.Linear(step, 1), mmn.Linear(step, 0)
    for it in range(2):
        grads = None
        for mb in range(2):
            x = data(TOKENS, D, "bf16", 10 * it + mb, 0.3)
            dy = data(TOKENS, D, "bf16", 100 + 10 * it + mb, 0.3)
            y = ln.forward(x)
            _, mean, rstd = ln._saved
            check_forward(y, mean, rstd, x, step.param(2), step.param(3), 1e-5)
            z = ffn.forward(y.view(3, 25, D))
            assert z.shape == (3, 25, FFN) and z.dtype == torch.bfloat16
            z = z.view(TOKENS, FFN)
            check_product(z, plain_values(y), plain_values(step.param(1)))
            out = ffn2.forward(z)
            check_product(out, plain_values(z), plain_values(step.param(0)))
            assert torch.equal(out, ffn2.forward(z, training=False))
            base = [step.grad(k).clone() for k in range(4)] if mb else [None] * 4
            dz = ffn2.backward(dy, accumulate=mb > 0)
            check_product(step.grad(0), plain_values(dy.t()), plain_values(z.t()), base[0])
            check_product(dz, plain_values(dy), plain_values(step.param(0).t()))
            dyn = ffn.backward(dz.view(3, 25, FFN), accumulate=mb > 0)
            assert dyn.shape == (3, 25, D)
            dyn = dyn.view(TOKENS, D)
            check_product(step.grad(1), plain_values(dz.t()), plain_values(y.t()), base[1])
            check_product(dyn, plain_values(dz), plain_values(step.param(1).t()))
            dx = ln.backward(dyn, accumulate=mb > 0)
            check_backward(dx, step.grad(2), step.grad(3), dyn, x, step.param(2), mean, rstd,
                           base[2:] if mb else None)
        before = [step.param(k).clone() for k in range(4)]
        step.step(grad_divisor=2.0)
        step.sync()
        for k in range(4):
            assert not torch.equal(step.param(k), before[k])
        for layer in (ffn, ffn2):
            layer.refresh()
            p = step.param(layer.slot)
            assert torch.equal(layer.w.dequantize().double(), plain_values(p))
            assert torch.equal(layer.wt.dequantize().double(), plain_values(p.t()))
    mmn.kernel_status()
    step.close()


def test_non_finite_activation_skips_the_step(mmn):
    """An Inf that enters the 4-bit product reaches the grad slots as NaN, so the
    loss-scaled step sees it and skips."""
    import torch

    step = make_step(mmn, loss_scaling=True, loss_scale_init=1.0)
    lin = mmn.Linear(step, 1)
    for k in (0, 2, 3):
        step.grad(k).zero_()
    x, dy = data(TOKENS, D, "bf16", 1, 0.3), data(TOKENS, FFN, "bf16", 2, 0.3)
    before = step.param(1).clone()
    dy[5, 7] = float("inf")
    lin.forward(x)
    lin.backward(dy)
    assert torch.isnan(step.grad(1)).any()
    step.step()
    step.sync()
    assert step.loss_scale() == (0.5, 1) and torch.equal(step.param(1), before)
    step.close()


def test_linear_gradients_against_differences(mmn):
    """On values that 4 bits hold exactly (whole blocks with a 6 or -6 along both
    axes) the layer is linear: changing one weight by d changes sum(dy * y) by
    d dW, exactly, and one input by d dx."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(3)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                        device="cuda")
    exact = lambda r, c: _with_sixes(grid[torch.randint(16, (r, c), device="cuda", generator=gen)])
    out, inn, rows = 96, 64, 160
    step = mmn.OptimizerStep([(0, (out, inn))], mmn.StepConfig())
    w, x, dy = exact(out, inn), exact(rows, inn), exact(rows, out)
    f = lambda: (dy.double() * lin.forward(x, training=False).double()).sum()
    step.set_param(0, w.cpu().numpy())
    lin = mmn.Linear(step, 0)
    lin.forward(x)
    dx = lin.backward(dy).double()
    dw = step.grad(0).double()
    y0 = f()
    for r, c, v in ((5, 7, 2.0), (95, 63, -0.5), (40, 33, 1.5)):
        w2 = w.clone()
        w2[r, c] = v
        step.set_param(0, w2.cpu().numpy())
        lin.refresh()
        assert f() - y0 == (v - w[r, c].double()) * dw[r, c]
    step.set_param(0, w.cpu().numpy())
    lin.refresh()
    for r, c, v in ((3, 9, 3.0), (159, 60, -1.0)):
        old = x[r, c].item()
        x[r, c] = v
        assert f() - y0 == (v - old) * dx[r, c]
        x[r, c] = old
    step.close()


def _with_sixes(t):
    """Every 32 x 1 and 1 x 32 block holds a 6, away from the places that the test
    changes (those have (row - column) % 32 other than 0)."""
    n = min(t.shape)
    for i in range(t.shape[0]):
        for j in range(i % 32, t.shape[1], 32):
            t[i, j] = 6.0
    assert n >= 32
    return t


def test_state_and_shape_errors(mmn):
    import torch

    step = make_step(mmn)
    with pytest.raises(mmn.ShapeError):
        mmn.Linear(step, 2)
    with pytest.raises(mmn.ShapeError):
        mmn.LayerNorm(step, 0, 1)
    lin, ln = mmn.Linear(step, 1), mmn.LayerNorm(step, 2, 3)
    for layer in (lin, ln):
        with pytest.raises(mmn.MmnError):
            layer.backward(torch.zeros(4, D, device="cuda"))
    with pytest.raises(mmn.ShapeError):
        lin.forward(torch.zeros(4, D + 1, device="cuda"))
    x = torch.zeros(4, D, device="cuda")
    for layer in (lin, ln):
        layer.forward(x)
        layer.forward(x, training=False)  # holds nothing
        with pytest.raises(mmn.MmnError):  # the first pass still waits
            layer.forward(x)
    with pytest.raises(mmn.ShapeError):
        lin.backward(x)
    lin.discard()
    lin.forward(x)
    lin.backward(torch.zeros(4, FFN, device="cuda"))
    with pytest.raises(mmn.MmnError):  # held once, used once
        lin.backward(torch.zeros(4, FFN, device="cuda"))
    with pytest.raises(TypeError):
        lin.forward(torch.zeros(4, D))  # host memory
    step.close()


FIRST_CALLS = """
import sys
sys.path.insert(0, %r)
import torch
import magicmindnet_b200 as mmn
x = torch.randn(300, 512, device="cuda").bfloat16()
dy = torch.randn(300, 512, device="cuda").bfloat16()
g, w = torch.ones(512, device="cuda"), torch.randn(512, 512, device="cuda")

def block():
    y, mean, rstd = mmn.layer_norm(x, g, g)
    q, qt = mmn.mxfp4_quantize(w, "both")
    z = mmn.mxfp4_linear(y, q)
    z1 = mmn.mxfp4_linear(y[:1], q)
    dq, dt = mmn.mxfp4_quantize(dy, "both")
    dz = mmn.mxfp4_matmul(dq, qt)
    dw = mmn.mxfp4_matmul(dt, mmn.mxfp4_quantize(y, "cols"), out_dtype=torch.float32)
    return (z, z1, dw, q.dequantize()) + mmn.layer_norm_backward(dz, x, g, mean, rstd)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # the very first calls of this process
    got = block()
for it in range(3):
    x.copy_(torch.randn_like(x)); dy.copy_(torch.randn_like(dy))
    graph.replay()
    for a, b in zip(got, block()):
        assert torch.equal(a, b)
mmn.kernel_status()
print("captured")
"""


def test_first_calls_inside_a_capture():
    """A process whose first calls are being captured: nothing is allocated or set
    up in a way that a capture forbids."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS % root], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_two_graphs_at_once(mmn):
    """Two captured passes over different data, replayed together on two streams:
    each keeps its own workspaces."""
    import torch

    w = data(512, 384, "f32", 1, 0.5)
    q, qt = mmn.mxfp4_quantize(w, "both")
    g = torch.ones(384, device="cuda")

    def passes(x, dy):
        y, mean, rstd = mmn.layer_norm(x, g, g)
        dq, dt = mmn.mxfp4_quantize(dy, "both")
        dz = mmn.mxfp4_matmul(dq, qt)
        dw = mmn.mxfp4_matmul(dt, mmn.mxfp4_quantize(y, "cols"), out_dtype=torch.float32)
        return (mmn.mxfp4_linear(y, q), dw) + mmn.layer_norm_backward(dz, x, g, mean, rstd)

    runs = []
    for s in (1, 2):
        x, dy = data(2000, 384, "bf16", s, 0.3), data(2000, 512, "bf16", s + 5, 0.3)
        want = passes(x, dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = passes(x, dy)
        # (x and dy stay: a graph keeps the addresses of its inputs, not the tensors)
        runs.append((graph, got, want, torch.cuda.Stream(), x, dy))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, s, _, _ in runs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _, _ in runs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    mmn.kernel_status()


def test_backward_that_failed_can_be_called_again(mmn, monkeypatch):
    """No room for dx: the grad slot keeps what it held, and the second call adds the
    weight's gradient once."""
    import torch

    from magicmindnet_b200 import layers

    step = make_step(mmn)
    lin = mmn.Linear(step, 1)
    x, dy = data(TOKENS, D, "bf16", 1, 0.3), data(TOKENS, FFN, "bf16", 2, 0.3)
    base = torch.randn(FFN, D, device="cuda")
    step.grad(1).copy_(base)
    lin.forward(x)
    real = layers.mxfp4_matmul

    def no_room(a, b, out=None, **kw):
        if out is None:
            raise torch.cuda.OutOfMemoryError("no room for dx")
        return real(a, b, out=out, **kw)

    monkeypatch.setattr(layers, "mxfp4_matmul", no_room)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        lin.backward(dy, accumulate=True)
    monkeypatch.undo()
    assert torch.equal(step.grad(1), base)
    dx = lin.backward(dy, accumulate=True)
    check_product(step.grad(1), plain_values(dy.t()), plain_values(x.t()), base)
    check_product(dx, plain_values(dy), plain_values(step.param(1).t()))
    step.close()


def test_linear_refuses_copies_older_than_the_weight(mmn):
    """After anything that changes the parameters, until refresh. A forward pass that
    came before still gets its backward pass."""
    import numpy as np
    import torch

    step = make_step(mmn)
    lin, other = mmn.Linear(step, 1), mmn.Linear(step, 0)
    x, dy = data(TOKENS, D, "bf16", 1, 0.3), data(TOKENS, FFN, "bf16", 2, 0.3)
    n = len(NAMES)
    for k in range(n):
        step.grad(k).normal_()
    changes = (step.step, lambda: step.step_host([None] * n, [None] * n),
               lambda: step.set_param(1, np.full((FFN, D), 0.25, np.float32)))
    for change in changes:
        lin.forward(x)
        change()
        step.sync()
        lin.backward(dy)
        for training in (True, False):
            with pytest.raises(mmn.MmnError, match="refresh"):
                lin.forward(x, training=training)
        with pytest.raises(mmn.MmnError, match="refresh"):
            other.forward(data(3, FFN, "bf16", 3), training=False)
        lin.refresh()
        other.refresh()
        y = lin.forward(x, training=False)
        check_product(y, plain_values(x), plain_values(step.param(1)))
    assert torch.equal(step.param(1), torch.full((FFN, D), 0.25, device="cuda"))
    step.sync()  # nothing here changes a parameter
    step.set_grad(1, np.zeros((FFN, D), np.float32))
    step.get_param(1)
    lin.forward(x, training=False)
    step.close()


def test_layers_of_a_closed_step_refuse(mmn):
    step = make_step(mmn)
    lin, ln = mmn.Linear(step, 1), mmn.LayerNorm(step, 2, 3)
    x = data(TOKENS, D, "bf16", 1, 0.3)
    dy = [lin.forward(x), ln.forward(x)]
    step.close()
    for layer, g in zip((lin, ln), dy):
        layer_calls = [lambda: layer.forward(x), lambda: layer.forward(x, training=False),
                       lambda: layer.backward(g)]
        for call in layer_calls + ([lin.refresh] if layer is lin else []):
            with pytest.raises(mmn.MmnError, match="closed"):
                call()
    with pytest.raises(mmn.MmnError):
        mmn.Linear(step, 1)
