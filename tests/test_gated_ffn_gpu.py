"""ltxattn_gated_ffn and ltxattn_gated_ffn_bwd on a B200 against the block in 64 bits.

Tolerances are bounds, element by element, carried through the formulas from
 - u = 2^-8, the most one rounding to bf16 is off, relative to the value;
 - 2^-22 per term of a sum relative to the sum of the terms' sizes: fp32
   accumulation on the tensor cores, which may cut where fp32 rounds;
 - 2^-18 for an activation and its slope (exp, division and erfc in fp32, a few
   units of 2^-24 each, over arguments of a few tens), relative to their size.
A tensor's bound is returned beside it by `forward` and `backward` below.
"""
import ctypes
import math

import pytest
import torch

from ltxattn import (AttentionBackend, _lib, device_status, gated_ffn, gated_ffn_backward, linear, rotary_embed,
                     rotary_embed_backward, rotary_frequencies)

pytestmark = pytest.mark.gpu

U, TERM, FUN = 2.0 ** -8, 2.0 ** -22, 2.0 ** -18
ACTS = ("silu", "gelu_tanh", "gelu")


@pytest.fixture(autouse=True)
def no_kernel_timeouts():
    yield
    assert device_status(clear=True) == 0, "a kernel wait timed out"


def act64(g, kind):
    """The activation and its slope."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    p = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def forward(x, wg, wu, wd, kind):
    """((y, bound), (gate, bound), (up, bound)); no activation is steeper than 1.2."""
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    gate, up = x @ wg.t(), x @ wu.t()
    eg, eu = (x.shape[1] * TERM * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a, _ = act64(gate, kind)
    h = a * up
    eh = (1.2 * eg + FUN * gate.abs()) * (up.abs() + eu) + a.abs() * eu
    eh = eh + U * (h.abs() + eh)
    y = h @ wd.t()
    ey = eh @ wd.abs().t() + wd.shape[1] * TERM * ((h.abs() + eh) @ wd.abs().t())
    return (y, ey + U * (y.abs() + ey)), (gate, eg + U * (gate.abs() + eg)), (up, eu + U * (up.abs() + eu))


def backward(x, wg, wu, wd, gate, up, dout, kind):
    """(dx, dwg, dwu, dwd), each with its bound, from gate and up as they are."""
    x, wg, wu, wd, gate, up, dout = (t.double() for t in (x, wg, wu, wd, gate, up, dout))
    a, slope = act64(gate, kind)
    dh = dout @ wd
    edh = dout.shape[1] * TERM * (dout.abs() @ wd.abs())
    fun = FUN * (1 + gate.abs())

    def rounded(v, e):
        return v, e + U * (v.abs() + e)

    dg, edg = rounded(dh * up * slope, edh * (up * slope).abs() + (dh.abs() + edh) * up.abs() * fun)
    du, edu = rounded(dh * a, edh * a.abs() + (dh.abs() + edh) * fun)
    h, eh = rounded(a * up, up.abs() * fun)
    n = x.shape[0]

    def product(l, el, r, er=0.0):
        v = l @ r
        e = el @ (r.abs() + er) + (l.abs() @ er if torch.is_tensor(er) else 0.0)
        return v, e + l.shape[1] * TERM * ((l.abs() + el) @ (r.abs() + er))

    zero = torch.zeros_like(dout)
    v1, e1 = product(dg, edg, wg)
    v2, e2 = product(du, edu, wu)
    return (rounded(v1 + v2, e1 + e2 + 2 * wg.shape[0] * TERM * (v1.abs() + v2.abs())),
            rounded(*product(dg.t(), edg.t(), x)), rounded(*product(du.t(), edu.t(), x)),
            rounded(*product(dout.t(), zero.t(), h, eh)))


def check(name, got, want):
    v, tol = want
    assert got.shape == v.shape and got.dtype == torch.bfloat16, name
    err = (got.double() - v).abs()
    assert bool((err <= tol).all()), f"{name}: {(err - tol).max().item():.3e} over the tolerance"


def make(seed, m, hidden, inner, out, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, k=1.0: (torch.randn(s, generator=g, device="cuda") * k).bfloat16()
    return (n(m, hidden, k=scale), n(inner, hidden, k=hidden ** -0.5), n(inner, hidden, k=hidden ** -0.5),
            n(out, inner, k=inner ** -0.5), n(m, out))


SIZES = [
    (1, 64, 128, 64),        # one token
    (1, 512, 1000, 520),
    (2, 8, 8, 8),            # the smallest widths
    (7, 72, 136, 200),       # no width fills a tile
    (16, 256, 640, 256),
    (33, 1032, 264, 136),
    (64, 128, 4096, 64),
    (101, 256, 688, 256),
    (110, 192, 264, 136),    # the first product exchanges its sums in two pieces
    (126, 64, 392, 72),
    (128, 256, 512, 256),    # one full row tile
    (129, 320, 384, 264),    # one row past it
    (300, 512, 1368, 512),
    (1000, 136, 328, 1048),
]


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,hidden,inner,out", SIZES)
def test_forward(kind, m, hidden, inner, out):
    x, wg, wu, wd, _ = make(m + inner, m, hidden, inner, out)
    want, want_gate, want_up = forward(x, wg, wu, wd, kind)
    check("y", gated_ffn(x, wg, wu, wd, kind), want)
    y, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    check("y with its gate kept", y, want)
    check("gate", gate, want_gate)
    check("up", up, want_up)


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,hidden,inner,out", SIZES)
def test_backward(kind, m, hidden, inner, out):
    x, wg, wu, wd, dout = make(m + inner + 1, m, hidden, inner, out)
    _, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    want = backward(x, wg, wu, wd, gate, up, dout, kind)
    got = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind)
    for name, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want):
        check(name, g, w)
    # parts of it are the same numbers
    only = gated_ffn_backward(None, wg, wu, wd, gate, up, dout, kind, need_dw=False)
    assert torch.equal(only[0], got[0]) and only[1:] == (None, None, None)
    only = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind, need_dx=False)
    assert only[0] is None and all(torch.equal(a, b) for a, b in zip(only[1:], got[1:]))


@pytest.mark.parametrize("kind", ACTS)
def test_gradient_against_differences(kind):
    # <d, v> for a direction v in each input, against central differences of the block in 64 bits: with a step
    # of 2^-12 the third-order term stays under 2^-24 of the direction's size, far under the bf16 bound
    m, hidden, inner, out = 40, 64, 96, 72
    x, wg, wu, wd, dout = make(5, m, hidden, inner, out)
    _, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    got = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind)
    bounds = backward(x, wg, wu, wd, gate, up, dout, kind)
    # the kept gate and up are rounded once more than the formula's: their own bound, through second slopes under 2
    exact = backward(x, wg, wu, wd, x.double() @ wg.double().t(), x.double() @ wu.double().t(), dout, kind)
    g = torch.Generator(device="cuda").manual_seed(6)
    args = [t.double() for t in (x, wg, wu, wd)]
    for i in range(4):
        v = torch.randn(args[i].shape, generator=g, device="cuda", dtype=torch.float64)
        step = 2.0 ** -12
        ends = []
        for s in (step, -step):
            moved = list(args)
            moved[i] = moved[i] + s * v
            ends.append((forward(*moved, kind)[0][0] * dout.double()).sum())
        diff = (ends[0] - ends[1]) / (2 * step)
        assert abs(diff - (exact[i][0] * v).sum()) <= 1e-4 * (exact[i][0].abs() * v.abs()).sum()
        tol = ((bounds[i][1] + (exact[i][0] - bounds[i][0]).abs()) * v.abs()).sum() + 1e-4 * (exact[i][0].abs() * v.abs()).sum()
        assert abs(diff - (got[i].double() * v).sum()) <= tol


def test_views_and_batches():
    B, T, hidden, inner, out = 3, 50, 128, 264, 136
    x, wg, wu, wd, dout = make(7, B * T, hidden, inner, out)
    want = gated_ffn(x, wg, wu, wd)
    # rows with padding between them, for every matrix; an output inside a wider buffer, whose rest stays
    wide = lambda t, pad: torch.nn.functional.pad(t, (8, pad))[:, 8:8 + t.shape[1]]
    buf = torch.full((B * T + 5, out + 24), 3.0, device="cuda").bfloat16()
    y = gated_ffn(wide(x, 16), wide(wg, 8), wide(wu, 40), wide(wd, 8), out=buf[:B * T, 8:8 + out])
    assert torch.equal(y, want)
    assert bool((buf[B * T:] == 3).all()) and bool((buf[:, :8] == 3).all()) and bool((buf[:, 8 + out:] == 3).all())
    # gate and up weights stacked in one matrix, batched tokens
    both = torch.cat((wg, wu))
    y3, gate, up = gated_ffn(x.view(B, T, hidden), both[:inner], both[inner:], wd, save=True)
    assert y3.shape == (B, T, out) and gate.shape == (B, T, inner) and torch.equal(y3.view(-1, out), want)
    got = gated_ffn_backward(x.view(B, T, hidden), wg, wu, wd, gate, up, dout.view(B, T, out))
    flat = gated_ffn_backward(wide(x, 8), wide(wg, 8), wide(wu, 8), wide(wd, 8), wide(gate.view(-1, inner), 8),
                              wide(up.view(-1, inner), 16), wide(dout, 8))
    assert got[0].shape == (B, T, hidden) and torch.equal(got[0].view(-1, hidden), flat[0])
    assert all(torch.equal(a, b) for a, b in zip(got[1:], flat[1:]))
    stacked = torch.full((2 * inner + 1, hidden), 5.0, device="cuda").bfloat16()
    gated_ffn_backward(x, wg, wu, wd, gate.view(-1, inner), up.view(-1, inner), dout, dw_gate=stacked[:inner],
                       dw_up=stacked[inner:2 * inner])
    assert torch.equal(stacked[:inner], got[1]) and torch.equal(stacked[inner:-1], got[2])
    assert bool((stacked[-1] == 5).all())


@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("which", ["dx", "dw_gate", "dw_up", "dw_down"])
def test_single_gradients_through_the_c_entry(m, which):
    # each output alone, with the inputs that only the others read left out
    hidden, inner, out = 64, 200, 72
    x, wg, wu, wd, dout = make(13, m, hidden, inner, out)
    _, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    want = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), gated_ffn_backward(x, wg, wu, wd, gate, up, dout)))[which]
    a = _lib.GatedFfnBwdArgs(_lib.BF16, 0, m, hidden, inner, out)
    got = torch.full_like(want, 7.0)
    given = dict(gate=gate, up=up, dout=dout, w_down=wd)
    given |= {"dx": dict(w_gate=wg, w_up=wu), "dw_down": {}}.get(which, dict(x=x))
    for name, t in {**given, which: got}.items():
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride", t.stride(0))
    L = _lib.load()
    ws = torch.empty(L.ltxattn_gated_ffn_bwd_workspace(ctypes.byref(a)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert L.ltxattn_gated_ffn_bwd(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.OK, _lib.last_error()
    assert torch.equal(got, want)


def test_rows_past_32_bits():
    # 140 thousand tokens of 16384: the planes between the kernels have 2.3e9 elements
    m, hidden, inner, out = 140001, 64, 16384, 72
    x, wg, wu, wd, dout = make(14, m, hidden, inner, out)
    tail = slice(m - 300, m)
    want, want_gate, want_up = forward(x[tail], wg, wu, wd, "silu")
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    check("y", y[tail], want)
    check("gate", gate[tail], want_gate)
    check("up", up[tail], want_up)
    dx, *_ = gated_ffn_backward(None, wg, wu, wd, gate, up, dout, need_dw=False)
    check("dx", dx[tail], backward(x[tail], wg, wu, wd, gate[tail], up[tail], dout[tail], "silu")[0])


def test_no_tokens():
    x, wg, wu, wd, dout = make(8, 0, 64, 128, 72)
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    assert y.shape == (0, 72) and gate.shape == up.shape == (0, 128)
    dirty = [torch.full(t.shape, 9.0, device="cuda").bfloat16() for t in (wg, wu, wd)]
    dx, *dw = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, dw_gate=dirty[0], dw_up=dirty[1], dw_down=dirty[2])
    assert dx.shape == (0, 64) and all(bool((t == 0).all()) for t in dw)


@pytest.mark.parametrize("m", [96, 6000])
@pytest.mark.parametrize("kind", ACTS)
def test_activations_far_out(m, kind):
    # gate = the value, up = 1 and y = h, so y is the activation, rounded once (U, relative).  Far out on the left it is
    # small and its exponent's error counts: arguments up to 88, three times rounded, and exp by under 2^-16 there:
    # 2^-14 of the result together.  Below 1e-35 the exponential's own range ends.
    gate = torch.cat((torch.linspace(-84, 84, m // 2), torch.linspace(-6, 6, m - m // 2))).cuda().bfloat16()
    x = torch.zeros(m, 8, device="cuda", dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = gate, 1.0
    w_gate, w_up = torch.zeros(2, 8, 8, device="cuda", dtype=torch.bfloat16)
    w_gate[:, 0], w_up[:, 1] = 1.0, 1.0
    w_down = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    got, kept, _ = gated_ffn(x, w_gate, w_up, w_down, kind, save=True)
    assert torch.equal(kept, gate[:, None].expand(m, 8))
    g = gate.double()[:, None]
    # (1 + tanh z) / 2 as sigmoid(2 z): near -1 a float64 tanh leaves 1 + tanh an error of 2^-54, more than what is left
    want = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) if kind == "gelu_tanh" else act64(g, kind)[0]
    assert bool(((got.double() - want).abs() <= (U + 2.0 ** -14) * want.abs() + 1e-35).all())


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("kind", ACTS)
def test_large_values_and_nan(m, kind):
    # gates far out on both sides: the activation is 0 or the gate itself; a NaN token spoils its own row alone
    x, wg, wu, wd, dout = make(9, m, 128, 256, 64, scale=200.0)
    want, *_ = forward(x, wg, wu, wd, kind)
    y, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    check("y", y, want)
    for name, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind),
                          backward(x, wg, wu, wd, gate, up, dout, kind)):
        check(name, g, w)
    spoiled = x.clone()
    spoiled[1, 5] = float("nan")
    z = gated_ffn(spoiled, wg, wu, wd, kind)
    keep = torch.arange(m, device="cuda") != 1
    assert bool(z[1].isnan().all()) and torch.equal(z[keep], y[keep])


@pytest.mark.parametrize("m", [1, 20, 300])
def test_repeated_calls_streams_and_graphs(m):
    x, wg, wu, wd, dout = make(10, m, 256, 520, 264)
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    grads = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    for _ in range(3):  # the same numbers every time
        assert torch.equal(gated_ffn(x, wg, wu, wd), y)
        assert all(torch.equal(a, b) for a, b in zip(gated_ffn_backward(x, wg, wu, wd, gate, up, dout), grads))
    # two streams at once
    sides = [torch.cuda.Stream() for _ in range(2)]
    other = make(11, m, 256, 520, 264)
    torch.cuda.synchronize()
    outs = [[gated_ffn(*t, stream=s) for _ in range(4)] for s, t in zip(sides, ((x, wg, wu, wd), other[:4]))]
    torch.cuda.synchronize()
    want_other = gated_ffn(*other[:4])
    assert all(torch.equal(o, y) for o in outs[0]) and all(torch.equal(o, want_other) for o in outs[1])
    # two graphs, replayed in turn with other inputs in their buffers
    bx, bd = x.clone(), dout.clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        cy, cg, cu = gated_ffn(bx, wg, wu, wd, save=True)
    with torch.cuda.graph(g2):
        cgrads = gated_ffn_backward(bx, wg, wu, wd, cg, cu, bd)
    for tx, td in ((x, dout), (other[0], other[4]), (x, dout)):
        bx.copy_(tx)
        bd.copy_(td)
        g1.replay()
        g2.replay()
        wy, wgate, wup = gated_ffn(tx, wg, wu, wd, save=True)
        assert torch.equal(cy, wy)
        assert all(torch.equal(a, b) for a, b in zip(cgrads, gated_ffn_backward(tx, wg, wu, wd, wgate, wup, td)))


def test_block_forward_and_backward():
    # a transformer block as it is called: projections, rotation, attention, projection, feed-forward -- and back.
    # Against the same chain in 64 bits with the library's own roundings left out: every stage rounds its output to
    # bf16 (2^-8) and there are 7 in a row forward and 14 with the way back; each is an independent error of under
    # 2^-9 in norm (a rounding's mean square is a third of its largest), and no stage more than doubles what it gets.
    B, T, H, D, inner = 1, 150, 4, 64, 512
    hidden = H * D
    g = torch.Generator(device="cuda").manual_seed(12)
    n = lambda *s, k=1.0: (torch.randn(s, generator=g, device="cuda") * k).bfloat16()
    x, dout = n(B, T, hidden), n(B, T, hidden)
    wq, wk, wv, wo = (n(hidden, hidden, k=hidden ** -0.5) for _ in range(4))
    wg, wu, wd = n(inner, hidden, k=hidden ** -0.5), n(inner, hidden, k=hidden ** -0.5), n(hidden, inner, k=inner ** -0.5)
    freq, magnitude = rotary_frequencies(D, scaling="yarn", factor=4.0, trained_length=64.0)
    split = lambda t: t.view(B, T, H, D).permute(0, 2, 1, 3)
    merge = lambda t: t.permute(0, 2, 1, 3).reshape(B, T, hidden)

    q, k = rotary_embed(split(linear(x, wq)), freq, k=split(linear(x, wk)), magnitude=magnitude)
    v = split(linear(x, wv))
    o, lse = AttentionBackend.attention(q, k, v, save_lse=True)
    a = linear(merge(o), wo)
    y, gate, up = gated_ffn(a, wg, wu, wd, "gelu_tanh", save=True)
    da, dwg, dwu, dwd = gated_ffn_backward(a, wg, wu, wd, gate, up, dout, "gelu_tanh")
    do = split(linear(da, wo.t().contiguous()))
    dq, dk, dv = AttentionBackend.attention_backward(q, k, v, o, do, lse)
    dq, dk = rotary_embed_backward(dq, freq, k=dk, magnitude=magnitude)
    dx = sum(linear(merge(d), w.t().contiguous()).double() for d, w in ((dq, wq), (dk, wk), (dv, wv)))

    leaf = [t.double().requires_grad_() for t in (x, wg, wu, wd)]
    X, WG, WU, WD = leaf
    place = torch.arange(T, device="cuda").double()[:, None] * freq
    cos, sin = place.cos() * magnitude, place.sin() * magnitude

    def turn(t):
        a_, b_ = t[..., :D // 2], t[..., D // 2:]
        return torch.cat((a_ * cos - b_ * sin, b_ * cos + a_ * sin), -1)

    Q, K, V = (split(X @ w.double().t()) for w in (wq, wk, wv))
    P = torch.softmax(turn(Q) @ turn(K).transpose(-1, -2) / math.sqrt(D), -1)
    A = merge(P @ V) @ wo.double().t()
    Y = (act64(A @ WG.t(), "gelu_tanh")[0] * (A @ WU.t())) @ WD.t()
    (Y * dout.double()).sum().backward()
    rel = lambda got, want: ((got.double() - want).norm() / want.norm()).item()
    assert rel(y, Y.detach()) <= 7 * 2.0 ** -9 * 2
    for got, want in ((dwg, WG.grad), (dwu, WU.grad), (dwd, WD.grad), (dx, X.grad)):
        assert rel(got, want) <= 14 * 2.0 ** -9 * 2
