"""More calls that ltxattn_rotary_embed refuses, all before any device work."""
import ctypes

import pytest

from ltxattn import _lib
from test_rotary_ffn_abi import rotary_args


@pytest.mark.parametrize("kw", [
    {"q_out.stride_t": 32}, {"q_out.stride_h": 63}, {"q_out.stride_b": 8},  # less than a row of 64 apart
    {"k_out.stride_t": 32}, {"k_out.stride_b": 63},
])
def test_outputs_whose_rows_overlap(kw):
    rc = _lib.load().ltxattn_rotary_embed(ctypes.byref(rotary_args(**kw)), None)
    assert rc == _lib.ERR_SHAPE, (rc, _lib.last_error())
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("magnitude", [float("inf"), float("-inf"), float("nan"), 1e39])
def test_magnitudes_that_are_not_finite(magnitude):
    # 1e39 is infinite in the call's fp32
    a = rotary_args(magnitude=magnitude)
    assert _lib.load().ltxattn_rotary_embed(ctypes.byref(a), None) == _lib.ERR_ARG
    assert "magnitude" in _lib.last_error()
