"""Amplitudes and epsilons that are finite as given but not as the 32-bit numbers
the kernels take: refused, before any device is touched."""
import ctypes

import pytest

from tests import capi_rotary as capi
from tests.test_rotary_cpu import _args


@pytest.mark.parametrize("kw", [dict(amplitude=1e39), dict(amplitude=-1e300), dict(eps=1e39)])
def test_beyond_32_bits(kw):
    L, a = capi.lib(), _args(**kw)
    assert L.vlak_qk_norm_rotary_fwd(ctypes.byref(a), None) == 1
    assert b"finite" in L.vlak_last_error_message()
    assert L.vlak_qk_norm_rotary_bwd(ctypes.byref(a), 0x1000, 1 << 40, None) == 1
    if "amplitude" in kw:
        assert L.vlak_rotary(ctypes.byref(a), None) == 1
