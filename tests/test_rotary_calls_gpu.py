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
