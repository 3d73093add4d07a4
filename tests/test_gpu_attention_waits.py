"""The attention kernels' waits end by the clock, whatever one try takes, and waits that share a limit end together."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("limit_ms,waits", [(100, 1), (100, 12), (250, 5)])
def test_waits_give_up_in_time(jx, dev, limit_ms, waits):
    jx.device_status()
    given_up, waited = C.c_int(0), C.c_float(0)
    jx.call("jx_selftest_wait_timeout", limit_ms, waits, C.byref(given_up), C.byref(waited))
    assert given_up.value == waits
    # 64 tries without the clock at each wait besides the limit: a few ms each at the most
    assert limit_ms <= waited.value <= limit_ms + 100 * waits
    assert jx.device_status() == jx.DEVERR_TIMEOUT
    assert jx.device_status() == 0


@pytest.mark.parametrize("limit_ms,waits", [(0, 1), (1001, 1), (10, 0), (10, 65)])
def test_limits_are_checked(jx, dev, limit_ms, waits):
    given_up, waited = C.c_int(0), C.c_float(0)
    with pytest.raises(jx.JaxRsError):
        jx.call("jx_selftest_wait_timeout", limit_ms, waits, C.byref(given_up), C.byref(waited))
