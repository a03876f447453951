"""Workloads of the layer operators that stand next to the optimizer step: layer
norm (forward, backward with the weights' gradients) and 4-bit microscaled
floating point (quantisation along either axis, the linear product with its
gradients). With ``own`` false ``run`` computes them from elementary torch
operations; with ``own`` true it calls the package.
"""
import math

import torch

own = False

F32, BF16 = "f32", "bf16"
_DTYPES = {F32: torch.float32, BF16: torch.bfloat16}
_EPS = 1e-5
_BLOCK = 32  # elements that share one scale


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one token of the d_model 2048 decoder being served: pure latency
        dict(name="ln_token", op="ln", rows=1, cols=2048, x=BF16, y=BF16),
        # a training micro-batch, fp32 residual stream into bf16 activations
        dict(name="ln_train", op="ln", rows=16384, cols=2048, x=F32, y=BF16),
        # a ragged batch at a width no vector divides
        dict(name="ln_odd", op="ln", rows=3001, cols=1013, x=F32, y=F32),
        # the d_model 64 Chatbot on a few hundred tokens: smallest training call
        dict(name="ln_grad_chat", op="ln_grad", rows=512, cols=64, x=F32, y=F32),
        # a training micro-batch of the d_model 4096 decoder
        dict(name="ln_grad_train", op="ln_grad", rows=16384, cols=4096, x=BF16, y=BF16),
        # activations quantised for the product and, transposed, for its weight gradient
        dict(name="quant_act", op="quant", rows=8192, cols=4096, x=BF16),
        # a ragged batch, fp32, neither axis a multiple of the block
        dict(name="quant_odd", op="quant", rows=1999, cols=1030, x=F32),
        # one token through an FFN matrix of the d_model 2048 decoder
        dict(name="linear_token", op="linear", rows=1, cols=2048, out=8192, x=BF16),
        # a few sequences decoded together, d_model 4096
        dict(name="linear_batch", op="linear", rows=48, cols=4096, out=4096, x=BF16),
        # a prompt through the FFN of the d_model 4096 decoder
        dict(name="linear_prompt", op="linear", rows=4096, cols=4096, out=14336, x=BF16),
        # backward of an FFN matrix of the d_model 2048 decoder over a micro-batch
        dict(name="linear_grad_train", op="linear_grad", rows=4096, cols=2048, out=8192, x=BF16),
        # backward over a ragged handful of tokens with odd widths, fp32
        dict(name="linear_grad_odd", op="linear_grad", rows=333, cols=1030, out=517, x=F32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Spread over the logarithm; half of them whole multiples of 64 as widths are."""
    n = _log(rng, lo, hi)
    return n if n < 64 or rng.random() < 0.5 else n // 64 * 64


def draw(rng):
    op = rng.choice(["ln", "ln_grad", "quant", "linear", "linear_grad"])
    dtype = rng.choice([F32, BF16])
    case = dict(op=op, x=dtype)
    if op in ("ln", "ln_grad"):
        cols = _size(rng, 8, 16384)
        case.update(rows=_log(rng, 1, min(32768, (16384 * 4096) // cols)), cols=cols,
                    y=rng.choice([dtype, BF16]))
    elif op == "quant":
        cols = _size(rng, 8, 16384)
        case.update(rows=_log(rng, 1, min(16384, (8192 * 4096) // cols)), cols=cols)
    else:
        cols, out = _size(rng, 32, 8192), _size(rng, 32, 14336)
        top = 4096 * 4096 * 14336 if op == "linear" else 4096 * 2048 * 8192
        case.update(rows=_log(rng, 1, max(1, min(4096, top // (cols * out)))), cols=cols, out=out)
    return case


# --------------------------------------------------------------------- inputs
def _normal(shape, gen):
    return torch.randn(shape, device="cuda", generator=gen)


def _stream(rows, cols, gen):
    """A residual stream: rows of their own size and mean, a few loud channels."""
    x = _normal((rows, cols), gen) * (0.5 + torch.rand((rows, 1), device="cuda", generator=gen))
    loud = 1.0 + 7.0 * (torch.rand((1, cols), device="cuda", generator=gen) < 0.01).float()
    return x * loud + 0.25 * _normal((rows, 1), gen)


def _inputs(case, seed):
    """The floating-point inputs of a case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, dtype = case["rows"], case["cols"], _DTYPES[case["x"]]
    s = {}
    if case["op"] in ("ln", "ln_grad"):
        s["x"] = _stream(rows, cols, gen).to(dtype)
        s["gamma"] = 1.0 + 0.1 * _normal((cols,), gen)
        s["beta"] = 0.1 * _normal((cols,), gen)
        if case["op"] == "ln_grad":
            s["dy"] = (1e-2 * _normal((rows, cols), gen)).to(_DTYPES[case["y"]])
            x = s["x"].double()
            mean = x.mean(1)
            var = (x - mean[:, None]).square_().mean(1)
            s["mean"], s["rstd"] = mean.float(), (var + _EPS).rsqrt().float()
    elif case["op"] == "quant":
        s["x"] = _stream(rows, cols, gen).to(dtype)
    else:
        s["x"] = _stream(rows, cols, gen).to(dtype)
        s["w"] = 0.02 * _normal((case["out"], cols), gen)
        if case["op"] == "linear_grad":
            s["dy"] = (1e-2 * _normal((rows, case["out"]), gen)).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "linear":
        # the weight is held in 4 bits, blocks along the axis that is summed
        s["w4"] = _pack(s.pop("w"), "rows")
    elif case["op"] == "linear_grad":
        # the transposed weight, and the activations that the forward pass saved
        s["w4t"] = _pack(s.pop("w"), "cols")
        s["x4t"] = _pack(s.pop("x"), "cols")
    return s


def _pack(x, along):
    if own:
        import magicmindnet_b200 as mmn

        return mmn.mxfp4_quantize(x, along=along)
    return _mx_values((x if along == "rows" else x.t()).float())


# ---------------------------------------------------------------- plain forms
def _mx_values(x):
    """fp32 [R, K] -> the values its 4-bit form stands for, blocks along K."""
    rows, k = x.shape
    pad = -k % _BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, _BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    # amax = m * 2^e with m in [1/2, 1): floor(log2 amax) = e - 1; 6 = 1.5 * 2^2 is the top element
    shared = (torch.frexp(amax).exponent - 3).clamp_(min=-127)
    v = torch.ldexp(b, -shared)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp_(max=6.0)
    out = torch.ldexp(torch.copysign(q, v), shared)
    out = torch.where(torch.isfinite(amax), out, torch.nan)
    return out.view(rows, k + pad)[:, :k]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "ln":
        x = s["x"].float()
        mean = x.mean(1)
        xc = x - mean[:, None]
        rstd = (xc.square().mean(1) + _EPS).rsqrt()
        y = xc * rstd[:, None] * s["gamma"] + s["beta"]
        return y.to(_DTYPES[case["y"]]), mean, rstd
    if op == "ln_grad":
        x, dy = s["x"].float(), s["dy"].float()
        h = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["gamma"]
        c1 = g.mean(1, keepdim=True)
        c2 = (g * h).mean(1, keepdim=True)
        dx = (g - c1 - h * c2) * s["rstd"][:, None]
        dgamma = (dy * h).sum(0, dtype=torch.float64).float()
        dbeta = dy.sum(0, dtype=torch.float64).float()
        return dx.to(s["x"].dtype), dgamma, dbeta
    if op == "quant":
        x = s["x"].float()
        return (_mx_values(x).to(s["x"].dtype),
                _mx_values(x.t().contiguous()).to(s["x"].dtype))
    if op == "linear":
        y = _mx_values(s["x"].float()) @ s["w4"].t()
        return y.to(s["x"].dtype)
    dy = s["dy"].float()
    dx = _mx_values(dy) @ s["w4t"].t()
    dw = _mx_values(dy.t().contiguous()) @ s["x4t"].t()
    return dx.to(s["dy"].dtype), dw


# ------------------------------------------------------------ the package's own
def _run_own(s):
    import magicmindnet_b200 as mmn

    case = s["case"]
    op = case["op"]
    if op == "ln":
        return mmn.layer_norm(s["x"], s["gamma"], s["beta"], _EPS, out_dtype=_DTYPES[case["y"]])
    if op == "ln_grad":
        return mmn.layer_norm_backward(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"])
    if op == "quant":
        q, qt = mmn.mxfp4_quantize(s["x"], along="both")
        return q.dequantize(s["x"].dtype), qt.dequantize(s["x"].dtype)
    if op == "linear":
        return mmn.mxfp4_linear(s["x"], s["w4"])
    q, qt = mmn.mxfp4_quantize(s["dy"], along="both")
    return (mmn.mxfp4_matmul(q, s["w4t"], out_dtype=s["dy"].dtype),
            mmn.mxfp4_matmul(qt, s["x4t"], out_dtype=torch.float32))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------- work
def work(case):
    rows, cols, e = case["rows"], case["cols"], _DTYPES[case["x"]].itemsize
    n = rows * cols
    mx = lambda r, k: r * (math.ceil(k / _BLOCK) * 17)  # 16 bytes of elements, 1 of scale a block
    if case["op"] == "ln":
        return dict(bytes=n * (e + _DTYPES[case["y"]].itemsize) + 8 * rows + 8 * cols, flops=8 * n)
    if case["op"] == "ln_grad":
        return dict(bytes=n * (2 * e + _DTYPES[case["y"]].itemsize) + 8 * rows + 12 * cols,
                    flops=15 * n)
    if case["op"] == "quant":
        # the 4-bit forms are written once and read once for the values
        return dict(bytes=n * 3 * e + 2 * (mx(rows, cols) + mx(cols, rows)), flops=8 * n)
    out = case["out"]
    if case["op"] == "linear":
        return dict(bytes=n * e + mx(out, cols) + rows * out * e, flops=2 * n * out)
    return dict(bytes=rows * out * e + mx(cols, out) + mx(cols, rows) + n * e + 4 * out * cols,
                flops=4 * n * out)


# ---------------------------------------------------------------------- exact
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_values(x):
    """The 4-bit form's values in 64 bits: every element goes to the grid point that
    its place among the midpoints names (a midpoint belongs to its even neighbour)."""
    x = x.double()
    rows, k = x.shape
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(x)
    for k0 in range(0, k, _BLOCK):
        b = x[:, k0:k0 + _BLOCK]
        amax = b.abs().amax(1)
        e = torch.floor(torch.log2(amax))
        # log2 may round across a power of two
        e = torch.where(torch.exp2(e) > amax, e - 1, e)
        e = torch.where(torch.exp2(e + 1) <= amax, e + 1, e)
        scale = torch.exp2(torch.clamp(torch.where(amax > 0, e, -200.0) - 2, min=-127))
        a = (b.abs() / scale[:, None]).contiguous()
        up = torch.bucketize(a, mid, right=True)   # a midpoint goes up
        down = torch.bucketize(a, mid)             # a midpoint goes down
        q = grid[torch.where(up % 2 == 0, up, down)]
        v = torch.sign(b) * q * scale[:, None]
        out[:, k0:k0 + _BLOCK] = torch.where(torch.isfinite(amax)[:, None], v, torch.nan)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("ln", "ln_grad"):
        x, gamma = s["x"].double(), s["gamma"].double()
        n = x.shape[1]
        if op == "ln":
            mean = x.sum(1) / n
            d = x - mean[:, None]
            rstd = 1.0 / torch.sqrt((d * d).sum(1) / n + _EPS)
            return d * rstd[:, None] * gamma + s["beta"].double(), mean, rstd
        dy, r = s["dy"].double(), s["rstd"].double()[:, None]
        h = (x - s["mean"].double()[:, None]) * r
        dgamma, dbeta = (dy * h).sum(0), dy.sum(0)
        dy.mul_(gamma)
        dx = dy - dy.sum(1, keepdim=True) / n
        return (dx - h * ((dy * h).sum(1, keepdim=True) / n)) * r, dgamma, dbeta
    if op == "quant":
        return _exact_values(s["x"]), _exact_values(s["x"].t())
    if op == "linear":
        return _exact_values(s["x"]) @ _exact_values(s["w"]).t()
    dy = s["dy"]
    return (_exact_values(dy) @ _exact_values(s["w"].t()).t(),
            _exact_values(dy.t()) @ _exact_values(s["x"].t()).t())
