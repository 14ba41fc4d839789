"""Calls of the rotary entry points on a B200 that their documentation allows, or that they must refuse."""
import math

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


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_stay_in_their_pair(layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(41)
    x = torch.randn((2, 3, 7, 64), generator=g, device="cuda").to(dtype)
    freq, _ = rotary_frequencies(48)
    y = rotary_embed(x, freq, layout=layout, offset=3)
    a, b = (5, 5 + 24) if layout == "half" else (10, 11)
    x[0, 1, 4, a], x[1, 2, 6, 60] = float("inf"), float("-inf")  # one that is turned and one that is copied
    z = rotary_embed(x, freq, layout=layout, offset=3)
    same = torch.ones_like(x, dtype=torch.bool)
    same[0, 1, 4, a] = same[0, 1, 4, b] = same[1, 2, 6, 60] = False
    assert torch.equal(z[same], y[same])
    angle = 7 * freq[5].cpu()
    assert z[0, 1, 4, a].item() == math.copysign(math.inf, angle.cos().item())
    assert z[0, 1, 4, b].item() == math.copysign(math.inf, angle.sin().item())
    assert z[1, 2, 6, 60].item() == -math.inf


def test_turned_keys_feed_the_next_call():
    # calls in a row on one stream, each reading what the one before wrote: n turns by 1 are one by n
    g = torch.Generator(device="cuda").manual_seed(42)
    x = torch.randn((1, 8, 500, 128), generator=g, device="cuda")
    freq, _ = rotary_frequencies(128)
    ones = torch.ones(500, dtype=torch.int64, device="cuda")
    y = x
    for _ in range(20):
        y = rotary_embed(y, freq, positions=ones)
    want = rotary_embed(x, freq, positions=20 * ones)
    # each of 21 turns is off by under 2^-21 + 2^-24 of the pair's size, and a pair keeps its size
    size = x[..., :64].hypot(x[..., 64:]).repeat(1, 1, 1, 2)
    assert bool(((y - want).abs() <= 21 * 1.5 * (2.0 ** -21 + 2.0 ** -24) * size).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads", [3, 40])  # a thread through all heads of a token, and tokens with their own CTAs
@pytest.mark.parametrize("call,sign", [(rotary_embed, 1.0), (rotary_embed_backward, -1.0)])
def test_turns_to_the_accuracy_of_fp32(call, sign, layout, heads):
    # The bound from what the kernel computes, u = 2^-24.  Angles up to 1e6 radians are off by under 2^-31 in fp64, here
    # and in the kernel; the remainder, under pi / 4, is rounded to fp32: u / 2.  The sine's series leaves 2^-29; its last
    # sum rounds by u / 2, and its term x^3 ps, under 0.081, is off by 5 u of itself: 0.95 u + 2^-29 together.  The cosine's
    # x^2 pc, under 0.31, is off by 2.5 u of itself, and its sum rounds by u / 2: 1.3 u + 2^-32.  So (cos, sin) are off by
    # 1.8 u and 1.5 u; b sin is rounded by u, and the sum once, relative to it: 2.5 u (|a| + |b|) + u |out| holds both.
    g = torch.Generator(device="cuda").manual_seed(43)
    D, T = 128, 25000 if heads == 3 else 900
    x = torch.randn((1, heads, T, D), generator=g, device="cuda")
    place = torch.randint(0, 1000000, (T,), generator=g, device="cuda")
    freq, _ = rotary_frequencies(D)
    got = call(x, freq, positions=place, layout=layout).double()
    angle = sign * place.double()[:, None] * freq
    cos, sin = angle.cos(), angle.sin()
    pair = (lambda t: (t[..., :D // 2], t[..., D // 2:])) if layout == "half" else (lambda t: (t[..., 0::2], t[..., 1::2]))
    a, b = pair(x.double())
    u = 2.0 ** -24
    for out, want in zip(pair(got), (a * cos - b * sin, b * cos + a * sin)):
        assert bool(((out - want).abs() <= 2.5 * u * (a.abs() + b.abs()) + u * want.abs()).all())
