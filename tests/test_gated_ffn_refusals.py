"""More calls that the feed-forward entry points refuse, all before any device work."""
import ctypes

import pytest

from ltxattn import _lib
from test_rotary_ffn_abi import bwd_args, ffn_args


@pytest.mark.parametrize("kw", [
    dict(hidden=2 ** 26 + 8, x_stride=2 ** 27, w_gate_stride=2 ** 27, w_up_stride=2 ** 27),
    dict(inner=2 ** 26 + 8, w_down_stride=2 ** 27),
    dict(out_dim=2 ** 26 + 8, out_stride=2 ** 27),
])
def test_products_too_long_for_a_bounded_wait(kw):
    # an epilogue waits for its tile's whole sum, 2 s at most; at 0.33 us for 64 products those are 3.9e8 products, of
    # which dx takes two for a step of inner
    rc = _lib.load().ltxattn_gated_ffn(ctypes.byref(ffn_args(**kw)), None)
    assert rc == _lib.ERR_UNSUPPORTED, (rc, _lib.last_error())


@pytest.mark.parametrize("only", ["dw_gate", "dw_up", "dw_down"])
def test_weight_gradients_of_too_many_tokens(only):
    L = _lib.load()
    none = dict(dx=None, dw_gate=None, dw_up=None, dw_down=None)
    one = {**none, only: 4096 * 9, "workspace_bytes": 0}
    rc = L.ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(m=2 ** 27 + 1, **one)), None)
    assert rc == _lib.ERR_UNSUPPORTED, (rc, _lib.last_error())
    # the most that are taken, and dx of more, get as far as their workspace
    rc = L.ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(m=2 ** 27, **one)), None)
    assert rc == _lib.ERR_WORKSPACE, (rc, _lib.last_error())
    rc = L.ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(m=2 ** 27 + 1, **{**none, "dx": 4096 * 8, "workspace_bytes": 0})), None)
    assert rc == _lib.ERR_WORKSPACE, (rc, _lib.last_error())
