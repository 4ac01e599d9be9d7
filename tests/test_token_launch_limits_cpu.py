"""What no launch can hold and no GPU's memory either is refused before anything touches the device."""
import ctypes

import pytest


@pytest.mark.parametrize("entry,lists", [("sdk_adamw_step", 4), ("sdk_adamw_step_8bit", 6)])
def test_tensors_of_2_to_36_values_are_refused(entry, lists):
    from _spherical_distortion_ext import _capi
    lib = _capi.load()
    lib.sdk_last_error.restype = ctypes.c_char_p
    one, sizes = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(1 << 36)
    assert getattr(lib, entry)(*([one] * lists), sizes, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 0, None) == -1
    assert "too large" in lib.sdk_last_error().decode()
