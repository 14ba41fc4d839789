"""ltxattn_rotary_embed on a B200 against the rotation in 64 bits.

Tolerance, per element of the pair (a, b): the angle's remainder is rounded to
fp32 (2^-28 of a turn, 2^-25 radians), sincospif is off by a few units of 2^-24,
the magnitude, the two products and their sum round once each: together under
2^-21 magnitude (|a| + |b|).  The store rounds once more, by half a step of the
type relative to the value.  Elements that are not turned are copied: no error.
"""
import math

import pytest
import torch

from ltxattn import AttentionBackend, rotary_embed, rotary_embed_backward, rotary_frequencies

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def plain(x, freq, place, layout, magnitude=1.0, inverse=False):
    """(out, |a| + |b| per element, 0 where copied) in float64; place [B, T]."""
    n = freq.numel()
    angle = place.double()[:, None, :, None] * freq * (-1.0 if inverse else 1.0)
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude
    out = x.double().clone(memory_format=torch.contiguous_format)
    size = torch.zeros_like(out)
    first = slice(0, n) if layout == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if layout == "half" else slice(1, 2 * n, 2)
    a, b = out[..., first].clone(), out[..., second].clone()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(magnitude)
    return out, size


def check(got, x, freq, place, layout, magnitude=1.0, inverse=False):
    want, size = plain(x, freq, place, layout, magnitude, inverse)
    assert got.dtype == x.dtype and got.shape == x.shape
    err = (got.double() - want).abs()
    tol = 2.0 ** -21 * size + HALF_STEP[x.dtype] * want.abs() * (size > 0) + 2.0 ** -20 * HALF_STEP[x.dtype] * size
    assert bool((err <= tol).all()), f"worst {((err - tol).max()).item():.3e} over the tolerance"


def heads(seed, B, T, H, D, dtype):
    """A projection output [B, T, H * D] seen as [B, H, T, D]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((B, T, H, D), generator=g, device="cuda").to(dtype).permute(0, 2, 1, 3)


def row(B, T, offset=0):
    return (torch.arange(T, device="cuda") + offset).expand(B, T)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H,Hk,D,rot", [
    (1, 1, 1, 1, 2, 2),          # the smallest call
    (16, 1, 32, 8, 128, 128),    # a decoded token per row
    (2, 33, 8, 2, 64, 64),
    (1, 257, 4, 4, 128, 64),     # half of the head
    (2, 5, 3, 1, 80, 24),        # 12 pairs: runs of 4
    (1, 19, 5, 5, 72, 20),       # 10 pairs: runs of 2
    (3, 7, 2, 1, 37, 6),         # an odd head size: single elements
    (1, 1030, 40, 1, 256, 250),
    (1, 300, 64, 64, 128, 128),
    (2, 20000, 2, 1, 64, 64),    # many tokens of few heads: a thread through all heads of a token
    (1, 30011, 3, 2, 40, 24),
    (3, 9001, 1, 1, 37, 6),
    (2, 41, 9, 2, 76, 24),       # what is copied is an odd number of runs
    (1, 12007, 6, 2, 76, 24),
])
def test_matches_the_rotation(layout, dtype, B, T, H, Hk, D, rot):
    q, k = heads(1, B, T, H, D, dtype), heads(2, B, T, Hk, D, dtype)
    freq, magnitude = rotary_frequencies(rot)
    assert magnitude == 1.0
    got_q, got_k = rotary_embed(q, freq, k=k, layout=layout)
    check(got_q, q, freq, row(B, T), layout)
    check(got_k, k, freq, row(B, T), layout)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_positions_of_every_row(dtype):
    B, T = 3, 50
    q, k = heads(3, B, T, 4, 64, torch.float32), heads(4, B, T, 2, 64, torch.float32)
    freq, _ = rotary_frequencies(64, theta=1e6)
    place = torch.tensor([[0], [1000000], [-77]], device="cuda") + torch.arange(T, device="cuda") * 3
    place[1, 7] = 2 ** 31 - 5
    got_q, got_k = rotary_embed(q, freq, k=k, positions=place.to(dtype), offset=4)
    check(got_q, q, freq, place + 4, "half")
    check(got_k, k, freq, place + 4, "half")
    # positions shared by the rows, as [tokens] and as [1, tokens], and with a stride
    for p in (place[0], place[:1], place[0].repeat_interleave(2)[::2]):
        check(rotary_embed(q, freq, positions=p.to(dtype)), q, freq, place[:1].expand(B, T), "half")


def test_far_positions_keep_their_angle():
    # past 32 bits: a float32 angle would have no digit of the turn left
    q = heads(5, 1, 3, 2, 64, torch.float32)
    freq, _ = rotary_frequencies(64)
    # the reference's own product rounds at 2^-53 of the angle: 2^33 radians leave 2^-20 of a radian
    place = torch.tensor([[2 ** 33 + 1, 2 ** 32 + 7, 12345678901]], device="cuda")
    got = rotary_embed(q, freq, positions=place)
    want, size = plain(q, freq, place, "half")
    assert bool(((got.double() - want).abs() <= (2.0 ** -21 + 2.0 ** -18) * size).all())
    assert torch.equal(rotary_embed(q, freq, positions=place - 2 ** 32, offset=2 ** 32), got)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_stretched_contexts(scaling, layout):
    q = heads(6, 2, 40, 4, 128, torch.bfloat16)
    freq, magnitude = rotary_frequencies(96, theta=5e5, scaling=scaling, factor=8.0, trained_length=8192.0)
    assert (magnitude > 1.2) == (scaling == "yarn")
    place = row(2, 40, 60000)
    got = rotary_embed(q, freq, positions=place, layout=layout, magnitude=magnitude)
    check(got, q, freq, place, layout, magnitude)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 40, 6])
def test_in_place_and_views(layout, rot):
    B, T, H, D = 2, 21, 4, 64
    g = torch.Generator(device="cuda").manual_seed(8)
    freq, _ = rotary_frequencies(rot)
    # q and k inside one projection output, turned where they lie; v and the padding stay
    qkv = torch.randn((B, T, 3 * H * D + 8), generator=g, device="cuda").bfloat16()
    before = qkv.clone()
    part = lambda t, i: t[:, :, i * H * D:(i + 1) * H * D].view(B, T, H, D).permute(0, 2, 1, 3)
    q, k = part(qkv, 0), part(qkv, 1)
    out = rotary_embed(q, freq, k=k, layout=layout, out_q=q, out_k=k)
    assert out[0] is q and out[1] is k
    check(q, part(before, 0), freq, row(B, T), layout)
    check(k, part(before, 1), freq, row(B, T), layout)
    assert torch.equal(qkv[:, :, 2 * H * D:], before[:, :, 2 * H * D:])
    # into the slots of a cache, whose other slots stay
    cache = torch.full((B, H, 64, D), 7.0, device="cuda").bfloat16()
    rotary_embed(part(before, 0), freq, layout=layout, offset=30, out_q=cache[:, :, 30:30 + T])
    check(cache[:, :, 30:30 + T], part(before, 0), freq, row(B, T, 30), layout)
    assert bool((cache[:, :, :30] == 7).all()) and bool((cache[:, :, 30 + T:] == 7).all())
    # rows that start on no 16-byte boundary, a contiguous [B, H, T, D], one head shared by all
    odd = torch.randn((B, T, H * D + 1), generator=g, device="cuda").bfloat16()[:, :, 1:].view(B, T, H, D)
    check(rotary_embed(odd.permute(0, 2, 1, 3), freq, layout=layout), odd.permute(0, 2, 1, 3), freq, row(B, T), layout)
    flat = odd.permute(0, 2, 1, 3).contiguous()
    check(rotary_embed(flat, freq, layout=layout), flat, freq, row(B, T), layout)
    shared = flat[:, :1].expand(B, H, T, D)
    check(rotary_embed(shared, freq, layout=layout), shared, freq, row(B, T), layout)


def test_cache_slots_past_32_bits():
    # two heads 2^31 elements apart: the offsets of the second need 64 bits
    slots, T, D = 2 ** 24 + 64, 40, 128
    cache = torch.empty((1, 2, slots, D), dtype=torch.bfloat16, device="cuda")
    cache[:, :, -T - 1] = 3.0
    q = heads(16, 1, T, 2, D, torch.bfloat16)
    freq, _ = rotary_frequencies(D)
    rotary_embed(q, freq, offset=slots - T, out_q=cache[:, :, -T:])
    check(cache[:, :, -T:], q, freq, row(1, T, slots - T), "half")
    assert bool((cache[:, :, -T - 1] == 3).all())
    # and read from there
    check(rotary_embed(cache[:, :, -T:], freq), cache[:, :, -T:], freq, row(1, T), "half")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward_is_the_transpose(layout, dtype):
    B, T, H, Hk, D, rot = 2, 45, 6, 2, 64, 48
    dq, dk = heads(9, B, T, H, D, dtype), heads(10, B, T, Hk, D, dtype)
    freq, magnitude = rotary_frequencies(rot, scaling="yarn", factor=4.0, trained_length=4096.0)
    place = row(B, T, 5000)
    got_q, got_k = rotary_embed_backward(dq, freq, k=dk, positions=place, layout=layout, magnitude=magnitude)
    check(got_q, dq, freq, place, layout, magnitude, inverse=True)
    check(got_k, dk, freq, place, layout, magnitude, inverse=True)
    # against differences: the call is linear, so (f(x + v) - f(x - v)) / 2 = f(v) and <dout, f(v)> = <dx, v>
    v, q = heads(11, B, T, H, D, dtype), heads(12, B, T, H, D, dtype).double()
    f = lambda x: plain(x, freq, place, layout, magnitude)[0]
    diff = (f(q + v.double()) - f(q - v.double())) / 2
    lhs, rhs = (dq.double() * diff).sum(), (got_q.double() * v.double()).sum()
    want, size = plain(dq, freq, place, layout, magnitude, True)
    tol = ((2.0 ** -21 * size + HALF_STEP[dtype] * want.abs()) * 1.001 * v.double().abs()).sum()
    assert abs(lhs - rhs) <= tol


def test_calls_without_work():
    freq, _ = rotary_frequencies(64)
    for B, H, T in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        x = torch.empty((B, H, T, 64), device="cuda", dtype=torch.bfloat16)
        assert rotary_embed(x, freq).shape == x.shape
    # no query heads, but keys
    q = torch.empty((2, 0, 5, 64), device="cuda")
    k = heads(13, 2, 5, 3, 64, torch.float32)
    check(rotary_embed(q, freq, k=k)[1], k, freq, row(2, 5), "half")


def test_streams_and_captured_replays():
    q, k = heads(14, 1, 64, 4, 64, torch.bfloat16), heads(15, 1, 64, 2, 64, torch.bfloat16)
    freq, _ = rotary_frequencies(64)
    place = torch.arange(64, device="cuda")
    want = rotary_embed(q, freq, k=k, positions=place)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rotary_embed(q, freq, k=k, positions=place, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_embed(q, freq, k=k, positions=place)
    for shift in (0, 17):  # the positions are read at each replay
        place.copy_(torch.arange(64, device="cuda") + shift)
        graph.replay()
        check(out[0], q, freq, row(1, 64, shift), "half")
        check(out[1], k, freq, row(1, 64, shift), "half")


def test_feeds_the_grouped_causal_attention():
    # rotation, then ltxattn_fwd with grouped KV heads, as a text encoder's layer calls them: moving
    # every position by the same amount changes no score, so the output stays up to rounding of q and k
    B, T, H, Hk, D = 1, 200, 8, 2, 64
    q, k, v = (heads(20 + i, B, T, n, D, torch.float32) for i, n in enumerate((H, Hk, Hk)))
    freq, _ = rotary_frequencies(D, theta=1e6, scaling="linear", factor=8.0)
    outs = []
    for offset in (0, 100000):
        rq, rk = rotary_embed(q, freq, k=k, offset=offset)
        outs.append(AttentionBackend.attention(rq, rk, v, causal=True)[0])
    # a score is off by at most 2 * 2^-20 |q||k| / sqrt(D) < 2^-19 * 17 * 17 / 8 < 7e-5 (rows of 64 normals stay
    # under 17 in norm), a weight relatively by twice that, an output by 1.4e-4 times the largest |v| < 6
    assert (outs[0] - outs[1]).abs().max().item() <= 1e-3
