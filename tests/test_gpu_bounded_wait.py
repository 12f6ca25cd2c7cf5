"""A device wait that nothing ends gives up by itself in about a second."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu


def test_wait_gives_up():
    import whirlwind_trt_plugins_b200 as ww
    ns = ctypes.c_ulonglong(0)
    assert ww.lib().ww_selftest_bounded_wait(ctypes.byref(ns)) == 0
    assert 0.1 < ns.value * 1e-9 < 4.0
