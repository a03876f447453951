"""4-bit microscaled matrices and their products against a plain 64-bit form.

The quantised values are whole multiples of a power of two chosen by comparisons,
so they have to be equal to the plain form's. A product's terms are exact in
fp32 (9-bit integers times powers of two); what is lost are the additions. Per
element, with S = sum |a b|: every MMA step (64 terms) may lose one unit of the
running sum's last place, 2^-23 S at most, so (K / 64 + 2) 2^-23 S, the output's
rounding H |out| (H = 2^-24 fp32, 2^-8 bf16), and with accumulation 2^-24 |sum|.
Non-finite values: the NaN pattern of the plain form.
"""
import itertools

import pytest

pytestmark = pytest.mark.gpu


def T(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def plain_values(x):
    """[R, K] -> the values of its 4-bit form, in 64 bits, blocks of 32 along K."""
    import torch

    x = x.double()
    rows, k = x.shape
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64,
                        device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    pad = -k % 32
    b = torch.nn.functional.pad(x, (0, pad)).reshape(rows, (k + pad) // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(finite, amax, torch.ones_like(amax)))
    e = torch.where(amax > 0, e - 1, torch.full_like(e, -1000))
    scale = torch.exp2(torch.clamp(e.double() - 2, min=-127.0))
    a = (b.abs() / scale).contiguous()
    up, down = torch.bucketize(a, mid, right=True), torch.bucketize(a, mid)
    q = grid[torch.where(up % 2 == 0, up, down)]
    v = torch.where(finite, torch.sign(b) * q * scale, torch.full_like(b, float("nan")))
    return v.reshape(rows, k + pad)[:, :k]


def same(got, want, what=""):
    import torch

    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    ok = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert ok.all(), (what, (~ok).nonzero()[0].tolist())


def data(rows, cols, dtype, seed=0, spread=3.0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda: torch.randn((rows, cols), device="cuda", generator=gen)
    return (n() * torch.exp(spread * n())).to(T(dtype))


def check_product(out, a, b, base=None):
    """a, b: 64-bit values [m, k], [n, k]."""
    import torch

    want, mag = a @ b.t(), a.abs() @ b.abs().t()
    k = a.shape[1]
    tol = (k / 64 + 2) * 2.0 ** -23 * mag
    if base is not None:
        want = want + base.double()
        tol = tol + 2.0 ** -24 * want.abs()
    tol = tol + torch.finfo(out.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + 1e-44
    bad = ~((out.double() - want).abs() <= tol)
    assert out.shape == want.shape
    assert not bad.any(), (bad.nonzero()[0].tolist(), (out.double() - want).abs().max().item())


SHAPES = [(1, 1), (1, 32), (2, 33), (31, 31), (32, 64), (33, 95), (127, 129), (128, 128),
          (129, 257), (256, 512), (300, 520), (1000, 1030), (1, 5000), (5000, 1), (70, 2048),
          # more tiles than the GPU takes at once, an odd and an even number each way
          (2890, 2888), (3000, 3208), (100000, 72), (5, 100000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_both_ways(mmn, rows, cols, dtype):
    import torch

    x = data(rows, cols, dtype, seed=rows + cols)
    q, qt = mmn.mxfp4_quantize(x, "both")
    want, want_t = plain_values(x), plain_values(x.t())
    for out in (torch.float32, torch.bfloat16):
        same(q.dequantize(out), want, "rows")
        same(qt.dequantize(out), want_t, "cols")
    for along, both in (("rows", q), ("cols", qt)):
        one = mmn.mxfp4_quantize(x, along)
        assert one.shape == both.shape
        assert torch.equal(one.codes, both.codes) and torch.equal(one.scales, both.scales)


def test_layout_of_codes_and_scales(mmn):
    """The documented bytes: even column in the low half, blocks filled with zeros,
    a scale byte at its place and zeros in a row's unused blocks."""
    import torch

    rows, cols = 130, 70
    x = data(rows, cols, "f32", seed=3, spread=1.0)
    q = mmn.mxfp4_quantize(x)
    assert q.codes.shape == (rows, 48) and q.scales.numel() == 2 * 2 * 512
    low, high = q.codes & 15, q.codes >> 4
    code = torch.stack((low, high), -1).view(rows, 96)
    assert not code[:, cols:].any()
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                        device="cuda", dtype=torch.float64)
    s = q.scales.view(2, 2, 32, 4, 4)  # row tile, column block, row % 32, row / 32, block % 4
    r = torch.arange(rows, device="cuda")
    got = torch.stack([s[r // 128, 0, r % 32, r // 32 % 4, k] for k in range(3)], -1)
    val = grid[code[:, :cols].long()].view(rows, cols) * torch.exp2(
        got.double() - 127)[:, torch.arange(cols, device="cuda") // 32]
    same(val, plain_values(x))
    assert not s[:, 1].any() and not s[0, 0, :, :, 3].any()


def test_rounding_of_every_midpoint(mmn):
    """Every grid point, midpoint and its fp32 neighbours, both signs, at scales
    from the smallest to the largest."""
    import torch

    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    pts = torch.cat((grid, (grid[1:] + grid[:-1]) / 2, torch.tensor([7.0, 7.999])))
    pts = torch.cat((pts, torch.nextafter(pts, torch.tensor(0.0)),
                     torch.nextafter(pts, torch.tensor(9.0))))
    pts = pts[(pts >= 0) & (pts < 8)].tolist()
    rows = []
    for i in range(0, len(pts), 15):
        part = pts[i:i + 15]
        row = part + [-p for p in part]
        rows.append([6.0] + row + [0.0] * (31 - len(row)))  # 6 fixes the scale at 1
    x = torch.tensor(rows, device="cuda")
    for e in (-125, -60, -1, 0, 1, 60, 124):
        y = x * 2.0 ** e
        same(mmn.mxfp4_quantize(y).dequantize(), plain_values(y), e)
        yt = y.t().contiguous()
        same(mmn.mxfp4_quantize(yt, "cols").dequantize(), plain_values(y), e)


def test_non_finite_and_strided_in_many_tiles(mmn):
    """The walk over many tiles: a slice of a wider buffer, Inf and NaN in its
    corners and edges."""
    import torch

    buf = data(2900, 3100, "bf16", 4, 1.0)
    x = buf[10:2890, 16:3072]
    x[0, 0], x[-1, -1], x[128, 127], x[1500, 3055] = (float("nan"), float("inf"), -float("inf"),
                                                      float("nan"))
    q, qt = mmn.mxfp4_quantize(x, "both")
    same(q.dequantize(), plain_values(x))
    same(qt.dequantize(torch.bfloat16), plain_values(x.t()))


def test_smallest_and_largest_magnitudes(mmn):
    import torch

    rows = []
    for m in (1e-45, 1e-42, 1.1754944e-38, 2.0 ** -125, 2.0 ** -124, 3e38, 3.4028235e38, 1.0):
        rows.append([m] + [m * f for f in (-1.0, 0.5, -0.25, 0.75, 0.1, 1e-3)] + [0.0] * 25)
    x = torch.tensor(rows, device="cuda", dtype=torch.float64).float()
    same(mmn.mxfp4_quantize(x).dequantize(), plain_values(x))
    same(mmn.mxfp4_quantize(x.t().contiguous(), "cols").dequantize(torch.bfloat16),
         plain_values(x))
    z = torch.zeros(3, 70, device="cuda")
    q = mmn.mxfp4_quantize(z)
    assert not q.dequantize().any() and not q.codes.any() and not q.scales.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_non_finite_blocks(mmn, dtype):
    """Inf or NaN anywhere in a block makes that block NaN and no other, and the
    product's sums over it NaN, against zeros too."""
    import torch

    a, b = data(200, 520, dtype, 1, 1.0), data(140, 520, dtype, 2, 1.0)
    a[3, 40], a[150, 519], a[7, 0] = float("nan"), float("inf"), -float("inf")
    b[9, 100] = float("nan")
    b[20] = 0
    qa, qat = mmn.mxfp4_quantize(a, "both")
    va, vb = plain_values(a), plain_values(b)
    same(qa.dequantize(), va)
    same(qat.dequantize(torch.bfloat16), plain_values(a.t()))
    for m in (200, 20):  # both orientations of the product
        out = mmn.mxfp4_matmul(mmn.mxfp4_quantize(a[:m]), mmn.mxfp4_quantize(b),
                               out_dtype=torch.float32)
        nan = torch.isnan(va[:m] @ vb.t())
        assert torch.equal(torch.isnan(out), nan) and nan.any() and not nan.all()
        assert torch.isnan(out[3, 20])


# few and many rows on either side, sums shorter and longer than a block, a stage
# (256) and the pipeline, ragged everywhere
PRODUCTS = [(1, 1, 1), (1, 128, 256), (3, 300, 100), (16, 129, 64), (17, 517, 1030),
            (32, 128, 2048), (33, 1000, 96), (64, 77, 4096), (100, 640, 333), (128, 128, 256),
            (129, 1, 512), (200, 300, 31), (256, 256, 1024), (300, 513, 2500), (513, 257, 4128),
            (1000, 31, 700), (2048, 16, 8192), (5, 2000, 14336), (777, 1030, 1999),
            (512, 512, 256), (520, 264, 1000), (2304, 2560, 300),
            # wide tiles of either width, one and several a CTA pair
            (2304, 2048, 700), (2100, 2001, 520), (4100, 2000, 1000), (5000, 3001, 300)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(mmn, m, n, k, out):
    import torch

    a, b = data(m, k, "f32", m, 1.0), data(n, k, "bf16", n + 1, 1.0)
    qa, qb = mmn.mxfp4_quantize(a), mmn.mxfp4_quantize(b)
    va, vb = plain_values(a), plain_values(b)
    check_product(mmn.mxfp4_matmul(qa, qb, out_dtype=T(out)), va, vb)
    # added to what an aligned buffer holds
    base = torch.randn(m, n, device="cuda").to(T(out))
    got = mmn.mxfp4_matmul(qa, qb, out=base.clone(), accumulate=True)
    check_product(got, va, vb, base)
    # into a slice of a wider buffer at an odd place, then added to it
    buf = torch.full((m, n + 11), 7.0, device="cuda", dtype=T(out))
    view = buf[:, 3:3 + n]
    assert mmn.mxfp4_matmul(qa, qb, out=view) is view
    check_product(view, va, vb)
    base = view.clone()
    mmn.mxfp4_matmul(qa, qb, out=view, accumulate=True)
    check_product(view, va, vb, base)
    assert (buf[:, :3] == 7).all() and (buf[:, 3 + n:] == 7).all()


@pytest.mark.parametrize("dtype,out", list(itertools.product(["f32", "bf16"], repeat=2)))
@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (1, 8192, 2048), (7, 100, 70), (48, 513, 1056),
                                   (100, 77, 512), (300, 520, 1030), (640, 1024, 2048),
                                   (16, 200, 9000), (17, 130, 33000), (33, 128, 17000),
                                   (64, 19200, 2500), (20, 19001, 5000)])
def test_linear(mmn, m, n, k, dtype, out):
    import torch

    x, w = data(m, k, dtype, 5, 1.0), data(n, k, "f32", 6, 0.5)
    q = mmn.mxfp4_quantize(w)
    vx, vw = plain_values(x), plain_values(w)
    y = mmn.mxfp4_linear(x, q, out_dtype=T(out))
    check_product(y, vx, vw)
    # equal to quantising first: one arithmetic behind both calls
    assert torch.equal(y, mmn.mxfp4_matmul(mmn.mxfp4_quantize(x), q, out_dtype=T(out)))
    # rows of a wider buffer, three axes
    wide = torch.randn(2, m, k + 3, device="cuda").to(T(dtype))
    wide[1, :, 1:1 + k] = x
    y3 = mmn.mxfp4_linear(wide[:, :, 1:1 + k], q, out_dtype=T(out))
    assert y3.shape == (2, m, n)
    check_product(y3[1], vx, vw)


def test_linear_keeps_non_finite_values(mmn):
    import torch

    x, w = data(5, 300, "bf16", 5, 1.0), data(200, 300, "f32", 6, 0.5)
    x[2, 299] = float("inf")
    x[4, 0] = float("nan")
    y = mmn.mxfp4_linear(x, mmn.mxfp4_quantize(w))
    assert torch.isnan(y[[2, 4]]).all() and torch.isfinite(y[[0, 1, 3]]).all()


def test_strided_and_unaligned_inputs(mmn):
    import torch

    buf = data(400, 600, "bf16", 8, 1.0)
    for x in (buf[::2, 3:400], buf[5:100, 8:8 + 256], buf[:, 1:2], buf[:1, 7:71]):
        q, qt = mmn.mxfp4_quantize(x, "both")
        same(q.dequantize(), plain_values(x))
        same(qt.dequantize(), plain_values(x.t()))
        out = torch.zeros(x.shape[0], x.shape[1] + 5, device="cuda", dtype=torch.bfloat16)
        view = out[:, 2:2 + x.shape[1]]
        assert q.dequantize(out=view) is view
        same(view, plain_values(x))
        assert not out[:, :2].any() and not out[:, 2 + x.shape[1]:].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols,ld", [(1, 3), (33, 41), (130, 133), (300, 301), (520, 552), (1029, 1029)])
def test_rows_that_start_anywhere(mmn, cols, ld, dtype):
    """A slice at every offset from an aligned address gives what a copy of it gives, reads
    nothing around it (NaN) and writes nothing around it."""
    import torch

    rows = 141
    for off in range(17):
        buf = torch.full((rows * ld + 32,), float("nan"), dtype=T(dtype), device="cuda")
        x = buf[off:off + rows * ld].view(rows, ld)[:, :cols]
        x.copy_(data(rows, cols, dtype, seed=cols + off))
        want, want_t = mmn.mxfp4_quantize(x.clone(), "both")
        q, qt = mmn.mxfp4_quantize(x, "both")
        for got, ref in ((q, want), (qt, want_t), (mmn.mxfp4_quantize(x), want),
                         (mmn.mxfp4_quantize(x, "cols"), want_t)):
            assert torch.equal(got.codes, ref.codes) and torch.equal(got.scales, ref.scales), off
        same(q.dequantize(), plain_values(x), off)
        out = torch.full_like(buf, 7.0)
        view = out[off:off + rows * ld].view(rows, ld)[:, :cols]
        q.dequantize(out=view)
        assert torch.equal(view, want.dequantize(T(dtype))), off
        view.fill_(7.0)
        assert (out == 7.0).all(), off


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("m,n,k", [(700, 1112, 512), (2000, 1304, 300), (40, 264, 512)])
def test_aligned_slices_leave_their_neighbours(mmn, m, n, k, accumulate, out):
    """Aligned column slices of a wider buffer (the widest stores) whose last tile
    ends inside the slice: rows and columns around it stay as they were."""
    import torch

    a, b = data(m, k, "f32", 1, 1.0), data(n, k, "f32", 2, 1.0)
    buf = torch.randn(m + 2, n + 24, device="cuda").to(T(out))
    keep = buf.clone()
    view = buf[1:1 + m, 8:8 + n]
    mmn.mxfp4_matmul(mmn.mxfp4_quantize(a), mmn.mxfp4_quantize(b), out=view, accumulate=accumulate)
    check_product(view, plain_values(a), plain_values(b),
                  keep[1:1 + m, 8:8 + n] if accumulate else None)
    outside = torch.ones_like(buf, dtype=torch.bool)
    outside[1:1 + m, 8:8 + n] = False
    assert torch.equal(buf[outside], keep[outside])


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("m,n,k", [(700, 1111, 512), (1999, 1301, 300), (515, 1030, 130), (40, 263, 512)])
def test_unaligned_slices_leave_their_neighbours(mmn, m, n, k, accumulate, out):
    """The same with rows that start anywhere, at even and odd pitches and offsets."""
    import torch

    a, b = data(m, k, "f32", 3, 1.0), data(n, k, "f32", 4, 1.0)
    qa, qb = mmn.mxfp4_quantize(a), mmn.mxfp4_quantize(b)
    for pad, off in ((9, 1), (10, 2), (13, 7), (16, 3)):
        buf = torch.randn(m + 2, n + pad, device="cuda").to(T(out))
        keep = buf.clone()
        view = buf[1:1 + m, off:off + n]
        mmn.mxfp4_matmul(qa, qb, out=view, accumulate=accumulate)
        check_product(view, plain_values(a), plain_values(b),
                      keep[1:1 + m, off:off + n] if accumulate else None)
        outside = torch.ones_like(buf, dtype=torch.bool)
        outside[1:1 + m, off:off + n] = False
        assert torch.equal(buf[outside], keep[outside])


@pytest.mark.parametrize("m", [3, 200])
def test_linear_within_one_buffer(mmn, m):
    """x and the result as column slices of one buffer; slices that meet are refused."""
    import torch

    w = data(96, 64, "f32", 6, 0.5)
    q = mmn.mxfp4_quantize(w)
    buf = data(m, 200, "bf16", 3, 1.0)
    x, out = buf[:, :64], buf[:, 100:196]
    want = mmn.mxfp4_linear(x.clone(), q)
    assert mmn.mxfp4_linear(x, q, out=out) is out
    assert torch.equal(out, want)
    with pytest.raises(mmn.MmnError):
        mmn.mxfp4_linear(x, q, out=buf[:, 63:159])


def test_refill_in_place(mmn):
    import torch

    x, y = data(130, 300, "f32", 1), data(130, 300, "f32", 2)
    pair = mmn.mxfp4_quantize(x, "both")
    ptrs = [m.codes.data_ptr() for m in pair]
    again = mmn.mxfp4_quantize(y, "both", out=pair)
    assert again[0] is pair[0] and again[1] is pair[1]
    assert [m.codes.data_ptr() for m in pair] == ptrs
    same(pair[0].dequantize(), plain_values(y))
    same(pair[1].dequantize(), plain_values(y.t()))
    with pytest.raises(mmn.ShapeError):
        mmn.mxfp4_quantize(data(130, 301, "f32"), "both", out=pair)


def test_empty(mmn):
    import torch

    for shape in ((0, 64), (64, 0), (0, 0)):
        x = torch.zeros(shape, device="cuda")
        q, qt = mmn.mxfp4_quantize(x, "both")
        assert q.dequantize().shape == shape and qt.dequantize().shape == shape[::-1]
    a, b = (mmn.mxfp4_quantize(torch.zeros(n, 0, device="cuda")) for n in (5, 300))
    out = torch.full((5, 300), 3.0, device="cuda")
    mmn.mxfp4_matmul(a, b, out=out, accumulate=True)
    assert (out == 3).all()
    mmn.mxfp4_matmul(a, b, out=out)
    assert not out.any()
    w = mmn.mxfp4_quantize(torch.ones(7, 64, device="cuda"))
    assert mmn.mxfp4_linear(torch.zeros(0, 64, device="cuda"), w).shape == (0, 7)
    assert mmn.mxfp4_linear(torch.zeros(2, 0, 64, device="cuda"), w).shape == (2, 0, 7)


def test_same_result_every_run(mmn):
    import torch

    for m, n, k in ((1, 8192, 2048), (48, 4096, 4096), (1000, 1030, 4096)):
        qa, qb = mmn.mxfp4_quantize(data(m, k, "f32", 1)), mmn.mxfp4_quantize(data(n, k, "f32", 2))
        first = mmn.mxfp4_matmul(qa, qb, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(mmn.mxfp4_matmul(qa, qb, out_dtype=torch.float32), first)
    mmn.kernel_status()


def test_streams_and_graph(mmn):
    """Two products at once on two streams, and a captured forward and backward
    replayed on new inputs."""
    import torch

    w = data(1000, 700, "f32", 1, 0.5)
    q, qt = mmn.mxfp4_quantize(w, "both")
    xs = [data(300, 700, "bf16", s, 1.0) for s in (2, 3)]
    want = [mmn.mxfp4_linear(x, q) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([mmn.mxfp4_linear(x, q) for _ in range(3)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g, y in zip(got, want):
        for t in g:
            assert torch.equal(t, y)
    sx, sdy = xs[0].clone(), data(300, 1000, "bf16", 4, 1.0)
    for warm in range(1):
        mmn.mxfp4_quantize(sx, "both")
    graph = torch.cuda.CUDAGraph()
    grad = torch.zeros(1000, 700, device="cuda")
    with torch.cuda.graph(graph):
        gy = mmn.mxfp4_linear(sx, q)
        dq, dt = mmn.mxfp4_quantize(sdy, "both")
        gx = mmn.mxfp4_matmul(dq, qt)
        mmn.mxfp4_matmul(dt, mmn.mxfp4_quantize(sx, "cols"), out=grad)
    for x, dy in ((xs[0], sdy.clone()), (xs[1], data(300, 1000, "bf16", 9, 1.0))):
        sx.copy_(x)
        sdy.copy_(dy)
        graph.replay()
        assert torch.equal(gy, mmn.mxfp4_linear(x, q))
        dq2, dt2 = mmn.mxfp4_quantize(dy, "both")
        assert torch.equal(gx, mmn.mxfp4_matmul(dq2, qt))
        assert torch.equal(grad, mmn.mxfp4_matmul(dt2, mmn.mxfp4_quantize(x, "cols"),
                                                  out_dtype=torch.float32))


def test_offsets_beyond_32_bits(mmn):
    """More than 2^31 elements of input, codes and output positions behind it."""
    import torch

    rows, cols = 70000, 32768  # 2.3e9 bf16 elements
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[-3:] = data(3, cols, "bf16", 1, 1.0)
    q, qt = mmn.mxfp4_quantize(x, "both")
    want = plain_values(x[-3:])
    v = q.dequantize(torch.bfloat16)
    same(v[-3:], want)
    assert not v[:3].any()
    del v
    vt = qt.dequantize(torch.bfloat16)
    same(vt[-5:, -32:], plain_values(x[-32:, -5:].t()))
    del vt, qt, x
    b = data(40000, cols, "bf16", 2, 1.0)
    qb = mmn.mxfp4_quantize(b)
    out = mmn.mxfp4_matmul(q, qb)  # 70000 x 40000 outputs
    check_product(out[-3:, -200:], want, plain_values(b[-200:]))
    assert not out[:3].any()
    mmn.kernel_status()


def test_refusals(mmn):
    import torch

    x = torch.zeros(4, 64, device="cuda")
    q = mmn.mxfp4_quantize(x)
    with pytest.raises(TypeError):
        mmn.mxfp4_quantize(x.half())
    with pytest.raises(ValueError):
        mmn.mxfp4_quantize(x[0])
    with pytest.raises(ValueError):
        mmn.mxfp4_quantize(x.t())
    with pytest.raises(ValueError):
        mmn.mxfp4_quantize(x[0].expand(3, 64))
    with pytest.raises(mmn.ShapeError):
        mmn.mxfp4_matmul(q, mmn.mxfp4_quantize(torch.zeros(4, 65, device="cuda")))
    with pytest.raises(mmn.ShapeError):
        mmn.mxfp4_matmul(q, q, out=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(TypeError):
        mmn.mxfp4_matmul(q, q, out=torch.zeros(4, 4, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        mmn.mxfp4_matmul(q, q, accumulate=True)
    with pytest.raises(mmn.ShapeError):
        mmn.mxfp4_linear(x[:, :32], q)
    from magicmindnet_b200 import _native as N

    import ctypes

    h = torch.zeros(4, 64)  # host memory
    assert N.lib().mmn_mxfp4_quantize(h.data_ptr(), 64, 0, 4, 64, ctypes.byref(q._c), None, 0,
                                      None) == N.MMN_E_INVALID
    c = N.Mxfp4C(q._c.codes, h.data_ptr() // 16 * 16, 4, 64)
    assert N.lib().mmn_mxfp4_matmul(ctypes.byref(c), ctypes.byref(q._c), x.data_ptr(), 4, 0, 0, 0,
                                    None) == N.MMN_E_INVALID


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("m,n,k", [(700, 1111, 512), (2304, 2049, 64), (2465, 939, 300), (300, 2050, 96),
                                   (90, 1111, 64), (1030, 1036, 64)])
def test_aligned_rows_that_end_anywhere_leave_their_neighbours(mmn, m, n, k, accumulate, out):
    """Rows that start on 16 bytes and end inside 16: what follows each, the last one
    too, stays bit for bit (NaN and subnormal patterns among it)."""
    import torch

    a, b = data(m, k, "f32", 1, 1.0), data(n, k, "f32", 2, 1.0)
    qa, qb = mmn.mxfp4_quantize(a), mmn.mxfp4_quantize(b)
    bits = {"f32": torch.int32, "bf16": torch.int16}[out]
    for pad in (8 - n % 8, 16 - n % 8):
        ld = n + pad
        for off in (0, 8):
            buf = torch.randint(-2 ** 15, 2 ** 15, (off + m * ld + 8,), device="cuda").to(bits)
            raw = buf.clone()
            # numbers in the slice itself
            view = buf.view(T(out))[off:off + m * ld].view(m, ld)[:, :n]
            view.copy_(torch.randn(m, n, device="cuda"))
            base = view.clone()
            mmn.mxfp4_matmul(qa, qb, out=view, accumulate=accumulate)
            check_product(view, plain_values(a), plain_values(b), base if accumulate else None)
            outside = torch.ones_like(buf, dtype=torch.bool)
            outside[off:off + m * ld].view(m, ld)[:, :n] = False
            assert torch.equal(buf[outside], raw[outside]), (pad, off)
