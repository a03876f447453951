"""The mmn_mxfp4_* calls refuse bad arguments before any device is touched. No GPU."""
import ctypes

import pytest

vp = ctypes.c_void_p
F32, BF16 = 0, 1


@pytest.fixture(scope="module")
def N():
    from magicmindnet_b200 import _native

    return _native


def mx(N, rows, cols, base):
    """A made-up matrix: codes at base, scales 16 MB further."""
    return N.Mxfp4C(base, base + (1 << 24), rows, cols)


def ref(m):
    return None if m is None else ctypes.byref(m)


def gate(N):
    return N.MMN_E_INVALID if N.lib().mmn_cuda_is_available() else N.MMN_E_NO_DEVICE


def test_sizes(N):
    """17 bytes per block of 32, rows of codes in 16-byte units, scales in 512-byte
    blocks of 128 x 128, an even number of them per 128 rows."""
    c, s = ctypes.c_int64(), ctypes.c_int64()
    f = lambda r, k: (N.lib().mmn_mxfp4_size(r, k, ctypes.byref(c), ctypes.byref(s)), c.value,
                      s.value)
    assert f(1, 1) == (0, 16, 1024)
    assert f(128, 256) == (0, 128 * 128, 1024)
    assert f(129, 257) == (0, 129 * 144, 2 * 4 * 512)
    assert f(4096, 14336) == (0, 4096 * 7168, 32 * 112 * 512)
    assert f(0, 64) == (0, 0, 0) and f(5, 0) == (0, 0, 0)
    big = 1 << 30
    assert f(big, big) == (0, big * big // 2, big // 128 * (big // 128) * 512)
    assert f(big + 1, 1)[0] == N.MMN_E_SHAPE and f(-1, 1)[0] == N.MMN_E_INVALID
    assert N.lib().mmn_mxfp4_size(1, 1, None, ctypes.byref(s)) == N.MMN_E_INVALID


def test_python_matrix_has_the_c_sizes(N):
    import magicmindnet_b200 as mmn

    c, s = ctypes.c_int64(), ctypes.c_int64()
    for r, k in ((1, 1), (5, 33), (128, 256), (129, 257), (300, 1030), (0, 64), (7, 0)):
        N.check(N.lib().mmn_mxfp4_size(r, k, ctypes.byref(c), ctypes.byref(s)))
        m = mmn.Mxfp4Matrix(r, k, "cpu")
        assert m.codes.numel() == c.value and m.scales.numel() == s.value
        assert m.codes.shape == (r, (k + 31) // 32 * 16)


def quant(N, x=vp(0x7000000000), ld=64, dt=F32, rows=4, cols=64, q="q", qt="qt"):
    q = mx(N, 4, 64, 0x1000000000) if q == "q" else q
    qt = mx(N, 64, 4, 0x2000000000) if qt == "qt" else qt
    return N.lib().mmn_mxfp4_quantize(x, ld, dt, rows, cols, ref(q), ref(qt), 0, None)


def test_quantize_refusals(N):
    bad = N.MMN_E_INVALID
    assert quant(N) == gate(N)
    assert quant(N, q=None) == gate(N) and quant(N, qt=None) == gate(N)
    assert quant(N, q=None, qt=None) == bad
    assert quant(N, dt=2) == bad
    assert quant(N, rows=-4) == bad
    assert quant(N, x=None) == bad
    assert quant(N, ld=63) == bad
    assert quant(N, q=mx(N, 4, 65, 0x1000000000)) == N.MMN_E_SHAPE
    assert quant(N, qt=mx(N, 4, 64, 0x1000000000)) == N.MMN_E_SHAPE
    assert quant(N, q=mx(N, 4, 64, 0x1000000008)) == bad           # alignment
    assert quant(N, q=N.Mxfp4C(None, 0x1000000000, 4, 64)) == bad  # null codes
    assert quant(N, q=mx(N, 4, 64, 0x7000000000)) == bad           # over x
    assert quant(N, qt=mx(N, 64, 4, 0x1000000000)) == bad          # over q
    assert quant(N, q=N.Mxfp4C(0x1000000000, 0x1000000010, 4, 64)) == bad  # scales over codes
    assert N.lib().mmn_last_error()


def test_dequantize_refusals(N):
    bad = N.MMN_E_INVALID
    f = N.lib().mmn_mxfp4_dequantize
    q, out = mx(N, 4, 64, 0x1000000000), vp(0x3000000000)
    assert f(ref(q), out, 64, F32, 0, None) == gate(N)
    assert f(None, out, 64, F32, 0, None) == bad
    assert f(ref(q), None, 64, F32, 0, None) == bad
    assert f(ref(q), out, 63, F32, 0, None) == bad
    assert f(ref(q), out, 64, 5, 0, None) == bad
    assert f(ref(q), vp(0x1000000010), 64, F32, 0, None) == bad
    assert f(ref(mx(N, 4, -64, 0x1000000000)), out, 64, F32, 0, None) == bad
    assert f(ref(mx(N, 4, (1 << 30) + 1, 0x1000000000)), out, 1 << 31, F32, 0, None) == N.MMN_E_SHAPE


def test_matmul_refusals(N):
    bad = N.MMN_E_INVALID

    def f(a=mx(N, 4, 64, 0x1000000000), b=mx(N, 8, 64, 0x2000000000), out=vp(0x3000000000), ld=8,
          dt=BF16):
        return N.lib().mmn_mxfp4_matmul(ref(a), ref(b), out, ld, dt, 0, 0, None)

    assert f() == gate(N)
    assert f(b=mx(N, 4, 64, 0x1000000000), ld=4) == gate(N)  # A A^T is allowed
    assert f(a=None) == bad and f(b=None) == bad
    assert f(b=mx(N, 8, 96, 0x2000000000)) == N.MMN_E_SHAPE
    assert f(out=None) == bad and f(ld=7) == bad and f(dt=3) == bad
    assert f(out=vp(0x1000000000)) == bad and f(out=vp(0x2000000000 + (1 << 24))) == bad
    assert f(a=N.Mxfp4C(0x1000000000, None, 4, 64)) == bad


def test_linear_refusals(N):
    bad = N.MMN_E_INVALID

    def f(x=vp(0x7000000000), ld=64, xd=BF16, rows=4, w=mx(N, 8, 64, 0x2000000000),
          xq=mx(N, 4, 64, 0x1000000000), out=vp(0x3000000000), old=8, od=BF16):
        return N.lib().mmn_mxfp4_linear(x, ld, xd, rows, ref(w), ref(xq), out, old, od, 0, None)

    assert f() == gate(N)
    assert f(x=None) == bad and f(ld=63) == bad and f(xd=4) == bad and f(od=4) == bad
    assert f(w=None) == bad and f(out=None) == bad and f(old=7) == bad
    few = N.MXFP4_DIRECT_ROWS
    assert f(xq=None) == gate(N)  # few rows need no room
    assert f(rows=few, xq=None) == gate(N) and f(rows=few + 1, xq=None) == bad
    assert f(rows=5) == N.MMN_E_SHAPE
    assert f(xq=mx(N, 4, 96, 0x1000000000)) == N.MMN_E_SHAPE
    assert f(xq=mx(N, 4, 64, 0x2000000000)) == bad  # the room lies over the weight
    assert f(xq=mx(N, 4, 64, 0x7000000000)) == bad  # ... over x
    assert f(out=vp(0x7000000000)) == bad           # out over x


def test_direct_rows_constant_agrees(N):
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "mmn_optim.h")).read()
    assert re.findall(r"#define MMN_MXFP4_DIRECT_ROWS (\d+)", text) == [str(N.MXFP4_DIRECT_ROWS)]


def test_wrappers_refuse_what_is_not_theirs():
    import torch

    import magicmindnet_b200 as mmn

    x = torch.zeros(4, 64)
    with pytest.raises(TypeError):
        mmn.mxfp4_quantize(x)
    with pytest.raises(ValueError):
        mmn.mxfp4_quantize(x, "diagonal")
    with pytest.raises(TypeError):
        mmn.mxfp4_matmul(x, x)
    with pytest.raises(TypeError):
        mmn.mxfp4_linear(x, x)
