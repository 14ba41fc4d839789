"""More calls that the feed-forward entry points refuse, all before any device work."""
import ctypes

import pytest
import torch

from ltxattn import Failure, _lib, gated_ffn_backward, gated_ffn_plan
from ltxattn.ffn import _output, _pack
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


def test_sizes_past_32_bits_are_failures_of_the_call():
    # a batch of 2^31 tokens fits on the GPU at a small width
    many = [_lib.BF16, 0, 2 ** 31, 8, 8, 8] + 7 * [4096, 8] + [4096, 0]
    with pytest.raises(Failure) as e:
        _pack(_lib.GATED_FFN_ARGS, *many)
    assert e.value.kind == "arg" and e.value.status == _lib.ERR_ARG
    with pytest.raises(Failure) as e:
        gated_ffn_plan(2 ** 32 + 1, 64, 64, 64)  # as an int32, one token
    assert e.value.kind == "shape"


@pytest.mark.parametrize("name,kw", [("dx", dict(need_dx=False)), ("dw_gate", dict(need_dw=False)),
                                     ("dw_up", dict(need_dw=False)), ("dw_down", dict(need_dw=False))])
def test_outputs_of_gradients_that_are_not_needed(name, kw):
    # they would come back as they were
    t = torch.zeros(8, 8, dtype=torch.bfloat16)
    with pytest.raises(Failure, match=f"{name} is given") as e:
        gated_ffn_backward(t, t, t, t, t, t, t, **kw, **{name: t})
    assert e.value.kind == "arg"


def test_outputs_that_are_no_tensors():
    with pytest.raises(Failure, match="out must be a CUDA tensor"):
        _output("out", [0.0], (1,), torch.zeros(1))
