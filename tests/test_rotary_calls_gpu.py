"""Calls of the rotary entry points on a B200 that their documentation allows, or that they must refuse."""
import pytest
import torch

from ltxattn import Failure, rotary_embed, rotary_embed_backward, rotary_frequencies

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(offset=2 ** 63), dict(offset=-2 ** 63 - 1), dict(offset=1.5), dict(offset="1"),
                                dict(magnitude=1e39), dict(magnitude=None)])
@pytest.mark.parametrize("call", [rotary_embed, rotary_embed_backward])
def test_numbers_that_the_call_cannot_take(call, kw):
    freq, _ = rotary_frequencies(64)
    q = torch.zeros(1, 2, 3, 64, device="cuda")
    with pytest.raises(Failure) as e:
        call(q, freq, **kw)
    assert e.value.kind == "arg"


def test_a_graph_that_kept_what_is_turned_in_place_says_so():
    freq, _ = rotary_frequencies(64)
    leaf = torch.randn(1, 2, 3, 64, device="cuda", requires_grad=True)
    q, k = leaf * 2, leaf * 3
    loss = (q * q * k).sum()  # keeps q and k
    before = q._version, k._version
    rotary_embed(q, freq, k=k, out_q=q, out_k=k)
    assert q._version > before[0] and k._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # outputs of the call's own, and inputs, count as they did
    before = q._version
    assert not rotary_embed(q, freq).requires_grad and q._version == before
    with torch.inference_mode():
        t = torch.zeros(1, 2, 3, 64, device="cuda")
        rotary_embed(t, freq, out_q=t)
