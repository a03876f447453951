"""Layer norm and its gradients against a plain 64-bit form.

Tolerances, per element, with u = 2^-24 (half a step of fp32) and H the half
step of the output's type (2^-24 fp32, 2^-8 bf16 relative to the value):
  mean     a sum of n terms in which each passes through at most D additions
           (32 in a thread, 5 + 5 across lanes and warps, n / 512 more for the
           looping kernel): D u mean|x|, and the division u|mean|
  h        (x - mean) r: r (D u mean|x| + u |x - mean|) + |h| (D + 6) u, the second
           term for the variance's sum, its division, square root and reciprocal
  y        |gamma| err(h) + 3 u (|h gamma| + |beta|) + H |y|
  dx       r [3u|g| + (D + 4) u mean|g| + |h| ((D + 4) u mean|g h| + mean(|g| err h))
              + |c2| err(h) + 4u (|g| + |c1| + |h c2|)] + H |dx|
  dgamma   a sum over rows in which each passes through at most R additions (the
           rows of one block, its 32 row groups, a part of the blocks' sums, the
           parts): (R + 3) u sum|dy h| + sum |dy| err(h) + H |dgamma|
  dbeta    R u sum|dy| + H |dbeta|
The backward pass takes mean and rstd as inputs: there err(h) is
r u |x - mean| + 2 u |h|.
"""
import itertools

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": "float32", "bf16": "bfloat16"}


def half(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def depth(cols):
    return 32 + 10 + cols / 512


def row_depth(rows):
    return 32 + rows / 64 + 592 / 8 + 8


def plain(x, gamma, beta, eps):
    x, gamma, beta = x.double(), gamma.double(), beta.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1.0 / (var + eps).sqrt()
    h = (x - mean) * rstd
    return h * gamma + beta, mean, rstd, h


def check(got, want, tol, what):
    import torch

    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, bad.nonzero()[0].tolist(),
                           (got.double() - want).abs().max().item())
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all()


def check_forward(y, mean, rstd, x, gamma, beta, eps):
    wy, wm, wr, h = plain(x, gamma, beta, eps)
    D = depth(x.shape[-1])
    xd = x.double()
    mabs = xd.abs().mean(-1, keepdim=True)
    merr = D * U * mabs + U * wm.abs()
    check(mean, wm[..., 0], merr[..., 0] + 1e-45, "mean")
    check(rstd, wr[..., 0], (wr * (D + 6) * U + wr ** 3 * merr ** 2)[..., 0], "rstd")
    herr = wr * (D * U * mabs + U * (xd - wm).abs()) + h.abs() * (D + 6) * U
    g = gamma.double().abs()
    tol = g * herr + 3 * U * ((h * gamma.double()).abs() + beta.double().abs())
    check(y, wy, tol * 1.01 + half(y.dtype) * wy.abs() + 1e-44, "y")


def check_backward(dx, dgamma, dbeta, dy, x, gamma, mean, rstd, base=None):
    dyd, xd, g64 = dy.double(), x.double(), gamma.double()
    rows, cols = xd.shape
    r, m = rstd.double().view(-1, 1), mean.double().view(-1, 1)
    h = (xd - m) * r
    g = dyd * g64
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    want = r * (g - c1 - h * c2)
    D = depth(cols)
    herr = r * U * (xd - m).abs() + 2 * U * h.abs()
    tol = r * (3 * U * g.abs() + (D + 4) * U * g.abs().mean(1, keepdim=True)
               + h.abs() * ((D + 4) * U * (g * h).abs().mean(1, keepdim=True)
                            + (g.abs() * herr).mean(1, keepdim=True))
               + c2.abs() * herr + 4 * U * (g.abs() + c1.abs() + (h * c2).abs()))
    check(dx, want, tol * 1.01 + half(dx.dtype) * want.abs() + 1e-44, "dx")
    R = row_depth(rows)
    wg, wb = (dyd * h).sum(0), dyd.sum(0)
    tg = (R + 3) * U * (dyd * h).abs().sum(0) + (dyd.abs() * herr).sum(0)
    tb = R * U * dyd.abs().sum(0)
    if base is not None:
        wg, wb = wg + base[0].double(), wb + base[1].double()
    check(dgamma, wg, tg * 1.01 + (half(dgamma.dtype) + U) * wg.abs() + 1e-44, "dgamma")
    check(dbeta, wb, tb * 1.01 + (half(dbeta.dtype) + U) * wb.abs() + 1e-44, "dbeta")


def make(rows, cols, xd, yd, pd="f32", seed=0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, device="cuda", generator=gen)
    x = (n(rows, cols) * (0.1 + n(rows, 1).abs()) + 2 * n(rows, 1)).to(getattr(torch, DT[xd]))
    gamma = (1 + 0.2 * n(cols)).to(getattr(torch, DT[pd]))
    beta = (0.3 * n(cols)).to(getattr(torch, DT[pd]))
    dy = (0.1 * n(rows, cols)).to(getattr(torch, DT[yd]))
    return x, gamma, beta, dy


# every width class (8, 32, 128, 256, 512 threads a row; looping), its edges, odd widths
WIDTHS = [1, 2, 7, 8, 63, 64, 65, 256, 260, 512, 520, 1013, 1024, 1032, 2048, 2056, 4096, 4100,
          8192, 8200, 16384, 16392, 20001]


@pytest.mark.parametrize("xd,yd", list(itertools.product(("f32", "bf16"), repeat=2)))
@pytest.mark.parametrize("cols", WIDTHS)
def test_forward_and_backward_over_widths(mmn, cols, xd, yd):
    import torch

    rows = 37
    x, gamma, beta, dy = make(rows, cols, xd, yd, seed=cols)
    y, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5, out_dtype=dy.dtype)
    assert y.dtype == dy.dtype and mean.shape == rstd.shape == (rows,)
    check_forward(y, mean, rstd, x, gamma, beta, 1e-5)
    out = mmn.layer_norm_backward(dy, x, gamma, mean, rstd)
    assert out[0].dtype == x.dtype and out[1].dtype == torch.float32
    check_backward(*out, dy, x, gamma, mean, rstd)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 148, 1000, 5000])
@pytest.mark.parametrize("cols,xd,yd", [(64, "f32", "f32"), (200, "bf16", "bf16"),
                                        (1030, "f32", "bf16"), (9000, "bf16", "f32")])
def test_row_counts(mmn, rows, cols, xd, yd):
    x, gamma, beta, dy = make(rows, cols, xd, yd, seed=rows)
    y, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5, out_dtype=dy.dtype)
    check_forward(y, mean, rstd, x, gamma, beta, 1e-5)
    check_backward(*mmn.layer_norm_backward(dy, x, gamma, mean, rstd), dy, x, gamma, mean, rstd)


@pytest.mark.parametrize("gd", ["f32", "bf16"])
@pytest.mark.parametrize("pd", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 1013, 2048, 8200])
def test_param_and_grad_types_and_accumulation(mmn, cols, pd, gd):
    """gamma and beta in either type; gradients into given buffers, overwritten and
    then added to."""
    import torch

    x, gamma, beta, dy = make(150, cols, "f32", "bf16", pd, seed=5)
    y, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5)
    check_forward(y, mean, rstd, x, gamma, beta, 1e-5)
    t = getattr(torch, DT[gd])
    dg = torch.full((cols,), float("nan"), device="cuda", dtype=t)
    db = dg.clone()
    dx, a, b = mmn.layer_norm_backward(dy, x, gamma, mean, rstd, dg, db)
    assert a is dg and b is db
    check_backward(dx, dg, db, dy, x, gamma, mean, rstd)
    base = (dg.clone(), db.clone())
    out = mmn.layer_norm_backward(dy, x, gamma, mean, rstd, dg, db, accumulate=True)
    check_backward(*out, dy, x, gamma, mean, rstd, base)


def test_rows_where_statistics_are_hard(mmn):
    """Constant rows (variance zero), a mean of 2000 deviations, one loud element,
    the largest magnitudes whose squares still sum, subnormal values."""
    import torch

    cols = 1000
    x, gamma, beta, dy = make(6, cols, "f32", "f32", seed=3)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = 1000.0 + 0.5 * torch.randn(cols, device="cuda")
    x[3, 17] = 1e4
    x[4] = 1e15 * torch.randn(cols, device="cuda")
    x[5] = 1e-40
    for eps in (1e-5, 1e-12):
        y, mean, rstd = mmn.layer_norm(x, gamma, beta, eps)
        check_forward(y, mean, rstd, x, gamma, beta, eps)
        check_backward(*mmn.layer_norm_backward(dy, x, gamma, mean, rstd), dy, x, gamma, mean,
                       rstd)


def test_non_finite_values_stay_in_their_row(mmn):
    import torch

    x, gamma, beta, dy = make(40, 300, "f32", "f32", seed=4)
    x[7, 11], x[20, 299] = float("nan"), float("inf")
    y, mean, rstd = mmn.layer_norm(x, gamma, beta)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 20]] = True
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()
    dx, dg, db = mmn.layer_norm_backward(dy, x, gamma, mean, rstd)
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    assert torch.isnan(dg).all() and torch.isfinite(db).all()


def test_empty(mmn):
    import torch

    g = torch.ones(16, device="cuda")
    x = torch.zeros(0, 16, device="cuda")
    y, mean, rstd = mmn.layer_norm(x, g, g)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dg = torch.full((16,), 5.0, device="cuda")
    db = dg.clone()
    mmn.layer_norm_backward(x, x, g, mean, rstd, dg, db, accumulate=True)
    assert (dg == 5).all() and (db == 5).all()
    dx, a, b = mmn.layer_norm_backward(x, x, g, mean, rstd, dg, db)
    assert dx.shape == (0, 16) and not dg.any() and not db.any()
    e = torch.zeros(5, 0, device="cuda")
    y, mean, rstd = mmn.layer_norm(e, g[:0], g[:0])
    assert y.shape == (5, 0) and mean.shape == (5,)


@pytest.mark.parametrize("cols", [96, 101, 2048, 9000])
def test_strided_unaligned_and_in_place(mmn, cols):
    """Column slices of wider buffers at odd offsets, three leading axes, outputs
    in place; elements outside the slices are left as they were."""
    import torch

    rows = 30
    wide = torch.randn(2, 15, 3 * cols + 5, device="cuda")
    keep = wide.clone()
    x = wide[..., 3:3 + cols]
    y = wide[..., 4 + cols:4 + 2 * cols]
    gbuf = torch.randn(cols + 1, device="cuda")
    gamma, beta = gbuf[1:], gbuf[:-1]
    x0 = x.clone()
    out, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5, out=y)
    assert out is y and mean.shape == (2, 15)
    check_forward(y.reshape(rows, cols), mean.view(-1), rstd.view(-1), x0.view(rows, cols), gamma,
                  beta, 1e-5)
    same = torch.ones_like(wide, dtype=torch.bool)
    same[..., 4 + cols:4 + 2 * cols] = False
    assert torch.equal(wide[same], keep[same])
    # forward in place, backward in place of dy and of x
    z = x0.clone()
    z2, m2, r2 = mmn.layer_norm(z, gamma, beta, 1e-5, out=z)
    # bit for bit what the same layout gives out of place; against the slices' result, which
    # another kernel sums in another order, within the bounds
    for a, b in zip((z, m2, r2), mmn.layer_norm(x0, gamma, beta, 1e-5)):
        assert torch.equal(a, b)
    check_forward(z.view(rows, cols), m2.view(-1), r2.view(-1), x0.view(rows, cols), gamma, beta,
                  1e-5)
    dy = torch.randn(2, 15, cols, device="cuda")
    want = mmn.layer_norm_backward(dy, x0, gamma, mean, rstd)
    for which in (0, 1):
        args = [dy.clone(), x0.clone()]
        got = mmn.layer_norm_backward(*args, gamma, mean, rstd, out=args[which])
        assert got[0] is args[which]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("xd,yd", list(itertools.product(("f32", "bf16"), repeat=2)))
@pytest.mark.parametrize("cols,ld,rows", [(66, 67, 5), (130, 133, 2500), (509, 509, 1300),
                                          (1021, 1024, 40), (2043, 2043, 700), (4095, 4097, 19),
                                          (8185, 8185, 9), (8200, 8201, 170), (16377, 16377, 3),
                                          (16383, 16383, 3), (600, 601, 1300), (1013, 1015, 1250),
                                          (1500, 1501, 2400), (4051, 4051, 1201), (6002, 6003, 1190),
                                          (9001, 9001, 1200)])
def test_rows_that_start_anywhere(mmn, cols, ld, rows, xd, yd):
    """Slices at offsets from an aligned address, x, dy and the outputs alike and not
    alike: the bounds hold, NaN around the inputs is not read into the results, and what
    lies around the outputs stays."""
    import torch

    x, gamma, beta, dy = make(rows, cols, xd, yd, seed=cols)

    def place(t, off, fill):
        buf = torch.full((rows * ld + 32,), fill, dtype=t.dtype, device="cuda")
        v = buf[off:off + rows * ld].view(rows, ld)[:, :cols]
        v.copy_(t)
        return buf, v

    nan = float("nan")
    for off, out_off in ((0, 0), (1, 1), (3, 3), (7, 7), (2, 5)):
        _, xv = place(x, off, nan)
        ybuf, yv = place(torch.zeros_like(dy), out_off, 7.0)
        _, mean, rstd = mmn.layer_norm(xv, gamma, beta, 1e-5, out=yv)
        check_forward(yv, mean, rstd, x, gamma, beta, 1e-5)
        yv.fill_(7.0)
        assert (ybuf == 7.0).all(), off
        _, dyv = place(dy, off, nan)
        dbuf, dxv = place(torch.zeros_like(x), out_off, 7.0)
        _, dgamma, dbeta = mmn.layer_norm_backward(dyv, xv, gamma, mean, rstd, out=dxv)
        check_backward(dxv, dgamma, dbeta, dy, x, gamma, mean, rstd)
        dxv.fill_(7.0)
        assert (dbuf == 7.0).all(), off


def test_one_row_as_a_vector(mmn):
    import torch

    x, gamma, beta, dy = make(1, 200, "f32", "f32", seed=3)
    y, mean, rstd = mmn.layer_norm(x[0], gamma, beta)
    assert y.shape == (200,) and mean.shape == rstd.shape == ()
    check_forward(y[None], mean[None], rstd[None], x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = mmn.layer_norm_backward(dy[0], x[0], gamma, mean, rstd)
    assert dx.shape == (200,)
    check_backward(dx[None], dgamma, dbeta, dy, x, gamma, mean, rstd)


@pytest.mark.parametrize("rows,cols", [(270000, 8192), (70000, 32768)])
def test_offsets_beyond_32_bits(mmn, rows, cols):
    """More than 2^31 elements: the last rows, and the sums over all of them."""
    import torch

    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    tail, gamma, beta, dyt = make(5, cols, "bf16", "bf16", seed=8)
    x[-5:] = tail
    y, mean, rstd = mmn.layer_norm(x, gamma, beta)
    check_forward(y[-5:], mean[-5:], rstd[-5:], tail, gamma, beta, 1e-5)
    assert torch.equal(y[0], beta.bfloat16()) and torch.equal(y[rows // 2], beta.bfloat16())
    y.zero_()
    y[-5:] = dyt  # now dy: nothing but in the last rows
    out = mmn.layer_norm_backward(y, x, gamma, mean, rstd)
    check_backward(out[0][-5:], out[1], out[2], dyt, tail, gamma, mean[-5:], rstd[-5:])
    assert not out[0][:-5].any()


def test_gradients_against_differences(mmn):
    """The directional derivative of sum(dy * layer_norm(x)) in 64 bits, central
    differences of step 1e-6 (their own error is about 1e-10), against the
    kernel's gradients."""
    import torch

    x, gamma, beta, dy = make(11, 130, "f32", "f32", seed=9)
    _, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5)
    dx, dg, db = mmn.layer_norm_backward(dy, x, gamma, mean, rstd)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(5):
        v = [torch.randn(t.shape, device="cuda", generator=gen, dtype=torch.float64)
             for t in (x, gamma, beta)]
        f = lambda s: (dy.double() * plain(x.double() + s * v[0], gamma.double() + s * v[1],
                                           beta.double() + s * v[2], 1e-5)[0]).sum()
        num = (f(1e-6) - f(-1e-6)) / 2e-6
        ours = [(a.double() * b).sum() for a, b in zip((dx, dg, db), v)]
        mag = sum((a.double() * b).abs().sum() for a, b in zip((dx, dg, db), v))
        # the kernels' own error is below 200 u of the terms' magnitude
        assert abs(num - sum(ours)) <= 200 * U * mag * max(1.0, float(rstd.max())) + 1e-6


def test_same_result_every_run(mmn):
    import torch

    x, gamma, beta, dy = make(3000, 777, "bf16", "bf16", seed=2)
    _, mean, rstd = mmn.layer_norm(x, gamma, beta)
    first = mmn.layer_norm_backward(dy, x, gamma, mean, rstd)
    for _ in range(5):
        for a, b in zip(mmn.layer_norm_backward(dy, x, gamma, mean, rstd), first):
            assert torch.equal(a, b)


def test_streams_and_graph(mmn):
    """On a side stream, and captured once and replayed on new inputs."""
    import torch

    x, gamma, beta, dy = make(64, 512, "f32", "bf16", seed=6)
    y0, m0, r0 = mmn.layer_norm(x, gamma, beta, out_dtype=torch.bfloat16)
    b0 = mmn.layer_norm_backward(dy, x, gamma, m0, r0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y1, m1, r1 = mmn.layer_norm(x, gamma, beta, out_dtype=torch.bfloat16)
        b1 = mmn.layer_norm_backward(dy, x, gamma, m1, r1)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip((y1, m1, r1) + b1, (y0, m0, r0) + b0):
        assert torch.equal(a, b)
    sx, sdy = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gm, gr = mmn.layer_norm(sx, gamma, beta, out_dtype=torch.bfloat16)
        gb = mmn.layer_norm_backward(sdy, sx, gamma, gm, gr)
    x2, _, _, dy2 = make(64, 512, "f32", "bf16", seed=7)
    for nx, ndy in ((x, dy), (x2, dy2)):
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        wy, wm, wr = mmn.layer_norm(nx, gamma, beta, out_dtype=torch.bfloat16)
        wb = mmn.layer_norm_backward(ndy, nx, gamma, wm, wr)
        for a, b in zip((gy, gm, gr) + gb, (wy, wm, wr) + wb):
            assert torch.equal(a, b)


def test_refusals(mmn):
    import torch

    x = torch.zeros(4, 8, device="cuda")
    g = torch.zeros(8, device="cuda")
    with pytest.raises(ValueError):
        mmn.layer_norm(x, g[:7], g)
    with pytest.raises(TypeError):
        mmn.layer_norm(x, g, g.bfloat16())
    with pytest.raises(TypeError):
        mmn.layer_norm(x.half(), g, g)
    with pytest.raises(ValueError):
        mmn.layer_norm(x.t(), g[:4], g[:4])
    with pytest.raises(mmn.ShapeError):
        mmn.layer_norm(x, g, g, out=torch.zeros(4, 9, device="cuda"))
    with pytest.raises(mmn.MmnError):
        mmn.layer_norm(x, g, g, eps=-1.0)
    _, m, r = mmn.layer_norm(x, g, g)
    with pytest.raises(mmn.ShapeError):
        mmn.layer_norm_backward(x[:3], x, g, m, r)
    with pytest.raises(ValueError):
        mmn.layer_norm_backward(x, x, g, m[:3], r)
    with pytest.raises(ValueError):
        mmn.layer_norm_backward(x, x, g, m, r, accumulate=True)
    with pytest.raises(ValueError):
        mmn.layer_norm_backward(x[0].expand(4, 8), x, g, m, r)
    with pytest.raises(mmn.MmnError):  # dx would overwrite half of x's rows
        buf = torch.zeros(8, 8, device="cuda")
        mmn.layer_norm_backward(x, buf[:4], g, m, r, out=buf[2:6])
    # host memory where device memory is needed, seen before any launch
    from magicmindnet_b200 import _native as N

    h = torch.zeros(4, 8)
    rc = N.lib().mmn_layer_norm(h.data_ptr(), 8, 0, g.data_ptr(), g.data_ptr(), 0, 1e-5, 4, 8,
                                x.data_ptr(), 8, 0, None, None, 0, None)
    assert rc == N.MMN_E_INVALID
    ws = torch.zeros(16, device="cuda")
    rc = N.lib().mmn_layer_norm_backward(
        x.data_ptr(), 8, 0, x.data_ptr(), 8, 0, g.data_ptr(), 0, m.data_ptr(), r.data_ptr(), 4, 8,
        torch.zeros_like(x).data_ptr(), 8, ws.data_ptr(), ws[8:].data_ptr(), 0, 0, ws.data_ptr(), 4,
        0, None)
    assert rc == N.MMN_E_INVALID  # workspace too small
    big = torch.zeros(1 << 16, device="cuda")
    rc = N.lib().mmn_layer_norm_backward(
        x.data_ptr(), 8, 0, x.data_ptr(), 8, 0, g.data_ptr(), 0, m.data_ptr(), r.data_ptr(), 4, 8,
        torch.zeros_like(x).data_ptr(), 8, big.data_ptr(), ws.data_ptr(), 0, 0, big.data_ptr(),
        big.numel() * 4, 0, None)
    assert rc == N.MMN_E_INVALID  # the workspace is also dgamma


# Dense aligned rows, enough that every row group of the walking kernels takes several
# and goes round its ring: each width class of the forward kernel (32 threads a row in
# both depths, 64, 128, 256, 512) and of the backward one (32, 64, 128, 256, 512), few more
# rows than the forward's threshold, and counts that divide into no grid.
@pytest.mark.parametrize("xd,yd", list(itertools.product(("f32", "bf16"), repeat=2)))
@pytest.mark.parametrize("cols,rows", [(72, 1185), (72, 20011), (256, 12007), (384, 1185),
                                       (384, 12007), (768, 1185), (768, 5003), (1024, 2500),
                                       (1024, 12007), (2048, 1185), (2048, 2500), (2048, 5003),
                                       (4096, 1185), (4096, 5003), (8192, 1185), (8192, 2500),
                                       (16384, 1187)])
def test_many_aligned_rows(mmn, cols, rows, xd, yd):
    x, gamma, beta, dy = make(rows, cols, xd, yd, seed=rows + cols)
    y, mean, rstd = mmn.layer_norm(x, gamma, beta, 1e-5, out_dtype=dy.dtype)
    check_forward(y, mean, rstd, x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = mmn.layer_norm_backward(dy, x, gamma, mean, rstd)
    check_backward(dx, dgamma, dbeta, dy, x, gamma, mean, rstd)
    # in place too: a row is read before its place is written
    z = x.clone() if x.dtype == y.dtype else None
    if z is not None:
        mmn.layer_norm(z, gamma, beta, 1e-5, out=z)
        check_forward(z, mean, rstd, x, gamma, beta, 1e-5)
    base = (dgamma.clone(), dbeta.clone())
    args = [dy.clone(), x]
    out = args[0] if dy.dtype == x.dtype else None
    dx, _, _ = mmn.layer_norm_backward(*args, gamma, mean, rstd, dgamma, dbeta, accumulate=True,
                                       out=out)
    check_backward(dx, dgamma, dbeta, dy, x, gamma, mean, rstd, base)
