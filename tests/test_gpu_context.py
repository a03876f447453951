"""A thread that holds a context of its own on the GPU: the library works in the
primary context, where its handles, kernels and torch's tensors are."""
import ctypes
import threading

import pytest

pytestmark = pytest.mark.gpu


def _run(fn):
    """fn in a thread of its own, its exception raised here."""
    failed = []

    def body():
        try:
            fn()
        except BaseException as e:  # noqa: BLE001 (handed to the test)
            failed.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    if failed:
        raise failed[0]


def test_calls_leave_a_foreign_context(mmn):
    import torch

    from magicmindnet_b200 import _native as N

    x = torch.randn(5, 64, device="cuda")
    g, b = torch.randn(64, device="cuda"), torch.randn(64, device="cuda")
    want = mmn.layer_norm(x, g, b)[0]
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    host = torch.zeros(5, 64)
    cu = ctypes.CDLL("libcuda.so.1")
    vp = ctypes.c_void_p

    def check(rc):
        assert rc == 0, rc

    def call(src):
        return N.lib().mmn_layer_norm(src.data_ptr(), 64, 0, g.data_ptr(), b.data_ptr(), 0, 1e-5, 5,
                                      64, y.data_ptr(), 64, 0, None, None, 0, None)

    def current():
        c = vp()
        check(cu.cuCtxGetCurrent(ctypes.byref(c)))
        return c.value

    def body():
        dev, primary, own = ctypes.c_int(), vp(), vp()
        check(cu.cuInit(0))
        check(cu.cuDeviceGet(ctypes.byref(dev), 0))
        check(cu.cuDevicePrimaryCtxRetain(ctypes.byref(primary), dev))
        check(cu.cuCtxCreate_v2(ctypes.byref(own), 0, dev))
        try:
            assert current() == own.value != primary.value
            # a call that is refused behind the change of the context, before any launch
            assert call(host) == N.MMN_E_INVALID
            assert current() == primary.value
            # and one that runs
            check(cu.cuCtxSetCurrent(own))
            N.check(call(x))
            assert current() == primary.value
            N.check(N.lib().mmn_kernel_status(0, None))
        finally:
            check(cu.cuCtxDestroy_v2(own))
            check(cu.cuDevicePrimaryCtxRelease_v2(dev))

    _run(body)
    assert torch.equal(y, want)
