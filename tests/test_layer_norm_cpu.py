"""mmn_layer_norm and mmn_layer_norm_backward refuse bad arguments before any
device is touched; the wrappers refuse tensors that are not theirs. No GPU."""
import ctypes

import pytest

vp = ctypes.c_void_p
F32, BF16 = 0, 1
X, Y, G, B, M, R = (vp(0x100000 * k) for k in range(1, 7))


@pytest.fixture(scope="module")
def N():
    from magicmindnet_b200 import _native

    return _native


def fwd(N, x=X, x_ld=64, xd=F32, gamma=G, beta=B, pd=F32, eps=1e-5, rows=4, cols=64, y=Y, y_ld=64,
        yd=F32, mean=M, rstd=R, device=0):
    return N.lib().mmn_layer_norm(x, x_ld, xd, gamma, beta, pd, eps, rows, cols, y, y_ld, yd, mean,
                                  rstd, device, None)


def bwd(N, dy=Y, dy_ld=64, dd=F32, x=X, x_ld=64, xd=F32, gamma=G, pd=F32, mean=M, rstd=R, rows=4,
        cols=64, dx=vp(0x900000), dx_ld=64, dgamma=vp(0xA00000), dbeta=vp(0xB00000), gd=F32, acc=0,
        ws=vp(0xC00000), wsb=1 << 40):
    return N.lib().mmn_layer_norm_backward(dy, dy_ld, dd, x, x_ld, xd, gamma, pd, mean, rstd, rows,
                                           cols, dx, dx_ld, dgamma, dbeta, gd, acc, ws, wsb, 0,
                                           None)


def gate(N):
    """What a well-formed call on made-up addresses gives: no GPU, or with one a
    refusal of the addresses before any launch."""
    return N.MMN_E_INVALID if N.lib().mmn_cuda_is_available() else N.MMN_E_NO_DEVICE


@pytest.mark.parametrize("kw", [
    dict(xd=2), dict(yd=-1), dict(pd=7), dict(eps=-1e-5), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(rows=-1), dict(cols=-1), dict(x=None), dict(y=None),
    dict(gamma=None), dict(beta=None), dict(x_ld=63), dict(y_ld=63), dict(x_ld=0),
    dict(y=vp(0x100000 + 4)),               # shifted by one element
    dict(y=X, yd=BF16),                     # in place, but of another element size
    dict(y=X, y_ld=128, x_ld=64),           # in place, but of another pitch
    dict(x_ld=100, y_ld=100, y=vp(0x100000 + 4 * 63)),  # slices that share a column
    dict(mean=R), dict(mean=vp(0x600000 + 12)), dict(rstd=vp(0x200000 + 64)), dict(mean=X),
])
def test_forward_refusals(N, kw):
    assert fwd(N, **kw) == N.MMN_E_INVALID
    assert N.lib().mmn_last_error()


def test_forward_too_large_is_a_shape_error(N):
    assert fwd(N, rows=1 << 31) == N.MMN_E_SHAPE
    assert fwd(N, cols=1 << 31, x_ld=1 << 31, y_ld=1 << 31) == N.MMN_E_SHAPE


@pytest.mark.parametrize("kw", [
    dict(), dict(y=X), dict(x_ld=128, y_ld=128, y=vp(0x100000 + 4 * 64)),  # slices side by side
    dict(rows=1, x_ld=0, y_ld=-5),  # the pitch of a single row is not read
    dict(mean=None), dict(rstd=None), dict(mean=None, rstd=None), dict(mean=vp(0x600000 + 16)),
])
def test_forward_allowed_up_to_the_device(N, kw):
    assert fwd(N, **kw) == gate(N)


@pytest.mark.parametrize("kw", [
    dict(xd=2), dict(dd=2), dict(pd=2), dict(gd=2), dict(rows=-1), dict(cols=-1), dict(dy=None),
    dict(x=None), dict(gamma=None), dict(mean=None), dict(rstd=None), dict(dx=None),
    dict(dgamma=None), dict(dbeta=None), dict(ws=None), dict(ws=vp(0xC00004)), dict(x_ld=63),
    dict(dy_ld=63), dict(dx_ld=63), dict(dgamma=vp(0xB00000)),
    dict(dx=vp(0x100000 + 4)), dict(dx=Y, dd=BF16),
    dict(dgamma=vp(0xB00000 + 4 * 63)), dict(dbeta=vp(0x900000 + 8)), dict(dgamma=vp(0x900000)),
])
def test_backward_refusals(N, kw):
    assert bwd(N, **kw) == N.MMN_E_INVALID
    assert N.lib().mmn_last_error()


@pytest.mark.parametrize("kw", [dict(), dict(dx=X), dict(dx=Y), dict(acc=1)])
def test_backward_allowed_up_to_the_device(N, kw):
    assert bwd(N, **kw) == gate(N)


# gamma, beta, mean and rstd lie at G, B, M, R; x at X, and dy (backward) or y at Y.
# An output that a block writes while another still reads it as an input is refused.
@pytest.mark.parametrize("kw", [
    dict(y=G), dict(y=B), dict(y=vp(0x300000 - 4 * 255)),  # y's last element is gamma's first
    dict(mean=G), dict(rstd=G), dict(mean=vp(0x400000 + 4 * 63)), dict(rstd=vp(0x400000 - 12)),
    dict(y=vp(0x300000 - 2 * 64), yd=BF16), dict(beta=vp(0x200000), pd=BF16),
])
def test_forward_refuses_outputs_over_the_parameters(N, kw):
    assert fwd(N, **kw) == N.MMN_E_INVALID
    assert b"overlap" in N.lib().mmn_last_error()


@pytest.mark.parametrize("kw", [dict(dx=a) for a in (G, M, R)] + [
    dict(dx=vp(0x300000 + 4 * 63)), dict(dx=vp(0x500000 - 4 * 255)), dict(mean=vp(0x900010)),
] + [{d: a} for d in ("dgamma", "dbeta") for a in (X, Y, G, M, R)] + [
    dict(dgamma=vp(0x500000 - 4 * 63)), dict(dbeta=vp(0x300000 + 2 * 63), pd=BF16, gd=BF16),
])
def test_backward_refuses_outputs_over_the_inputs(N, kw):
    assert bwd(N, **kw) == N.MMN_E_INVALID
    assert b"overlap" in N.lib().mmn_last_error()


@pytest.mark.parametrize("kw", [
    dict(y=vp(0x300000 - 4 * 256)), dict(mean=vp(0x300000 - 16)), dict(rstd=vp(0x400000 + 4 * 64)),
    # gamma in the gap between the rows of y
    dict(y_ld=256, y=vp(0x300000 - 4 * 64)),
])
def test_forward_allows_neighbours_of_the_parameters(N, kw):
    assert fwd(N, **kw) == gate(N)


@pytest.mark.parametrize("kw", [
    dict(dx=vp(0x300000 - 4 * 256)), dict(dgamma=vp(0x500000 + 16)), dict(dbeta=vp(0x300000 - 256)),
    dict(dx_ld=256, dx=vp(0x300000 - 4 * 64)),
])
def test_backward_allows_neighbours_of_the_inputs(N, kw):
    assert bwd(N, **kw) == gate(N)


def test_workspace_arguments(N):
    n = ctypes.c_int64()
    f = N.lib().mmn_layer_norm_backward_workspace
    assert f(4, 64, 0, None) == N.MMN_E_INVALID
    assert f(-1, 64, 0, ctypes.byref(n)) == N.MMN_E_INVALID
    assert f(1 << 31, 64, 0, ctypes.byref(n)) == N.MMN_E_SHAPE


def test_wrappers_refuse_host_tensors():
    import torch

    import magicmindnet_b200 as mmn

    x, g = torch.zeros(4, 8), torch.zeros(8)
    with pytest.raises(TypeError):
        mmn.layer_norm(x, g, g)
    with pytest.raises(TypeError):
        mmn.layer_norm_backward(x, x, g, g, g)


def test_rows_of_strided_tensors():
    """What counts as a matrix of rows, without a device."""
    import torch

    from magicmindnet_b200.norm import _rows_view

    t = torch.zeros(6, 4, 10)
    assert _rows_view(t, "t") == (24, 10, 10)
    assert _rows_view(t[..., 2:8], "t") == (24, 6, 10)
    assert _rows_view(t[::2, 0], "t") == (3, 10, 80)
    assert _rows_view(t[0, 0], "t") == (1, 10, 10)
    assert _rows_view(t[:, :0], "t") == (0, 10, 10)
    assert _rows_view(t[..., :0], "t") == (24, 0, 0)
    assert _rows_view(t[..., :1], "t") == (24, 1, 10)
    for bad in (t.transpose(1, 2), t[:, ::3, :][:, :, ::2], t[:, :3], t[0, 0].expand(5, 10)):
        with pytest.raises(ValueError):
            _rows_view(bad, "t")
    with pytest.raises(ValueError):
        _rows_view(torch.zeros(()), "t")


def test_layer_wait_selftest_arguments(N):
    f = N.lib().mmn_selftest_layer_wait
    assert f(0, 0, None) == N.MMN_E_INVALID and f(0, 2_000_000_001, None) == N.MMN_E_INVALID
    if not N.lib().mmn_cuda_is_available():
        assert f(0, 1000, None) == N.MMN_E_NO_DEVICE
