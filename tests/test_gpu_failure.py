"""Failure detection on the device without a fault: the bounded wait that every
pipelined kernel uses gives up after its limit, reports MMN_E_TIMEOUT through
the status word, and leaves the context usable."""
import time

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_bounded_wait_times_out_and_reports(mmn):
    from magicmindnet_b200 import _native as N

    t0 = time.monotonic()
    rc = N.lib().mmn_selftest_bounded_wait(0, 200_000_000)  # 200 ms
    dt = time.monotonic() - t0
    assert rc == N.MMN_E_TIMEOUT, N.lib().mmn_last_error()
    assert 0.2 <= dt < 5.0
    assert b"gave up" in N.lib().mmn_last_error()
    # the device is still usable afterwards
    g = np.random.default_rng(0).normal(0, 1e-2, (64, 96)).astype(np.float32)
    out = mmn.newton_schulz5(g)
    assert np.isfinite(out).all()
    assert N.lib().mmn_selftest_bounded_wait(0, 0) == N.MMN_E_INVALID


def test_layer_wait_is_reported_by_every_observer(mmn):
    """A layer operator's kernel that gives up: the status call and every step on the
    device say so, once each, and the work goes on."""
    import torch

    from magicmindnet_b200 import _native as N

    steps = [mmn.OptimizerStep([(0, (64, 96)), (1, (64,))], mmn.StepConfig()) for _ in range(3)]
    mmn.kernel_status()
    for s in steps:
        s.step()
        s.sync()
    side = torch.cuda.Stream()
    assert N.lib().mmn_selftest_layer_wait(0, 0, None) == N.MMN_E_INVALID
    assert N.lib().mmn_selftest_layer_wait(0, 3_000_000_000, None) == N.MMN_E_INVALID
    # nothing below depends on torch's or the step's stream being this one
    N.check(N.lib().mmn_selftest_layer_wait(0, 50_000_000, side.cuda_stream))
    side.synchronize()
    steps[0].step()
    with pytest.raises(mmn.KernelTimeoutError, match="layer operator"):
        steps[0].sync()
    steps[0].sync()  # reported once
    with pytest.raises(mmn.KernelTimeoutError):
        steps[1].step_host([None, None], [None, None])
    steps[1].step_host([None, None], [None, None])
    with pytest.raises(mmn.KernelTimeoutError):
        mmn.kernel_status()
    mmn.kernel_status()
    # a step made afterwards has nothing to report; one that never asked still has
    late = mmn.OptimizerStep([(0, (64, 96))], mmn.StepConfig())
    late.step()
    late.sync()
    N.check(N.lib().mmn_selftest_layer_wait(0, 50_000_000, None))
    for observe in (late.sync, mmn.kernel_status, steps[2].sync, steps[1].sync, steps[0].sync):
        with pytest.raises(mmn.KernelTimeoutError):
            observe()
        observe()
    x = torch.randn(5, 64, device="cuda")
    y = mmn.layer_norm(x, torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"))[0]
    assert torch.isfinite(y).all()
    for s in steps + [late]:
        s.close()
