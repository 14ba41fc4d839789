"""The rotary and gated feed-forward operators at the sizes they are measured at.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes what a program has in hand before
the call, ``run()`` is one pass through an operator -- in elementary torch operations, or, where
``own`` is true, through the library's entry points -- and ``exact()`` is the operator's definition
in 64 bits.

Two operators, each with its gradient:

* rotary positions: ``out = magnitude * R(position * frequency) x`` on the leading ``rotary`` elements of
  every head, in the half layout (element j turns with j + rotary/2) or the interleaved one
  (2j with 2j + 1); elements behind ``rotary`` pass through.  The gradient turns the other way.
* the gated feed-forward block: ``y = (act(x Wg^T) * (x Wu^T)) Wd^T``, and from the saved
  ``gate = x Wg^T`` and ``up = x Wu^T`` the gradients of x and of the three weights.
"""
import math
import os
import sys

import torch

own = False

_lib = None


def _ltxattn():
    """The framework's package, which lives in a folder that is no package name."""
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "ltx-2.5-swift_b200"))
        import ltxattn
        _lib = ltxattn
    return _lib


def listed():
    return [
        # one decoded token in each of 16 conversations, every row at a position of its own, grouped KV heads
        dict(name="rotary_step", op="rotary", batch=16, tokens=1, heads=32, kv_heads=8, head_dim=128, rotary=128,
             layout="half", dtype="bf16", scaling="linear", factor=8.0, theta=1e6, positions="rows", far=131072,
             backward=False),
        # a prompt of 1024 text tokens with left padding (the first positions repeat), grouped KV heads
        dict(name="rotary_text", op="rotary", batch=1, tokens=1024, heads=32, kv_heads=8, head_dim=128, rotary=128,
             layout="half", dtype="bf16", scaling="bands", factor=8.0, theta=5e5, positions="row", far=0,
             backward=False),
        # the queries and keys of the 29760-token video, interleaved pairs, positions counted from 0
        dict(name="rotary_video", op="rotary", batch=1, tokens=29760, heads=32, kv_heads=32, head_dim=128, rotary=128,
             layout="interleaved", dtype="bf16", scaling="none", factor=1.0, theta=1e4, positions="count", far=0,
             backward=False),
        # fp32, a part of the head (24 of 64), an odd token count, far positions in a stretched context
        dict(name="rotary_part_fp32", op="rotary", batch=2, tokens=3121, heads=32, kv_heads=4, head_dim=64, rotary=24,
             layout="half", dtype="fp32", scaling="yarn", factor=16.0, theta=1e4, positions="rows", far=1000000,
             backward=False),
        # the gradients of the 3120-token video's queries and keys
        dict(name="rotary_backward", op="rotary", batch=1, tokens=3120, heads=32, kv_heads=32, head_dim=128,
             rotary=128, layout="half", dtype="bf16", scaling="ntk", factor=4.0, theta=1e4, positions="row", far=0,
             backward=True),
        # one token: every weight is read once and used once
        dict(name="ffn_step", op="ffn", tokens=1, hidden=4096, inner=16384, act="silu", mode="forward"),
        # a few decoded tokens at the audio width
        dict(name="ffn_few", op="ffn", tokens=19, hidden=2048, inner=8192, act="gelu_tanh", mode="forward"),
        # the 101 audio tokens, with an inner width that fills no tile
        dict(name="ffn_audio", op="ffn", tokens=101, hidden=2048, inner=5464, act="gelu", mode="forward"),
        # a prompt of 1024 text tokens, with what the gradient needs kept
        dict(name="ffn_text_save", op="ffn", tokens=1024, hidden=4096, inner=16384, act="gelu_tanh", mode="save"),
        # the 3120-token video at the video width
        dict(name="ffn_video", op="ffn", tokens=3120, hidden=4096, inner=16384, act="silu", mode="forward"),
        # adapters trained below frozen weights: the gradient of x alone, 126 audio tokens
        dict(name="ffn_backward_input", op="ffn", tokens=126, hidden=2048, inner=8192, act="silu", mode="backward_x"),
        # training at the video width: the gradients of x and of the three weights
        dict(name="ffn_backward", op="ffn", tokens=3120, hidden=4096, inner=16384, act="gelu_tanh", mode="backward"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.45:
        head_dim = rng.choice((64, 128, 128, 8 * rng.randint(2, 32)))
        kv = rng.choice((1, 2, 4, 8, rng.randint(1, 16)))
        heads = kv * rng.choice((1, 2, 4, rng.randint(1, 8)))
        batch = rng.randint(1, 16)
        most = 29760 * 64 * 128 // (batch * (heads + kv) * head_dim * 2)
        positions = rng.choice(("count", "row", "rows"))
        return dict(op="rotary", batch=batch, tokens=_log_int(rng, 1, min(29760, max(1, most))), heads=heads,
                    kv_heads=kv, head_dim=head_dim,
                    rotary=rng.choice((head_dim, head_dim // 2 // 2 * 2, 2 * rng.randint(1, head_dim // 2))),
                    layout=rng.choice(("half", "interleaved")), dtype=rng.choice(("bf16", "bf16", "fp32")),
                    scaling=rng.choice(("none", "linear", "ntk", "yarn", "bands")),
                    factor=float(rng.choice((2, 4, 8, 32))), theta=float(rng.choice((1e4, 5e5, 1e6))),
                    positions=positions, far=_log_int(rng, 1, 1000000), backward=rng.random() < 0.4)
    hidden = 8 * _log_int(rng, 32, 512)
    inner = 8 * _log_int(rng, 64, 2048)
    return dict(op="ffn", tokens=_log_int(rng, 1, 3120), hidden=hidden, inner=inner,
                act=rng.choice(("silu", "gelu_tanh", "gelu")),
                mode=rng.choice(("forward", "forward", "save", "backward", "backward_x")))


# ---------------------------------------------------------------------------
# inputs


def _frequencies(case):
    """The angle that each pair turns by for a step of one position, in 64 bits, and the factor on what turns."""
    d, theta, s = case["rotary"], case["theta"], case["factor"]
    j = torch.arange(d // 2, dtype=torch.float64)
    if case["scaling"] == "ntk" and d > 2:  # the base grows, so that the slowest pair is stretched by the factor
        theta = theta * s ** (d / (d - 2))
    f = theta ** (-2.0 * j / d)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":  # fast pairs as they are, slow ones stretched, a ramp between 32 and 1 turns in 4096
        at = lambda turns: d * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        ramp = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1.0
    if case["scaling"] == "bands":  # the same, with the ramp over wavelengths of 1/4 to 1 times 8192
        turns = 8192 * f / (2 * math.pi)
        part = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f / s * (1 - part) + f * part, 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, scale=1.0: torch.randn(shape, generator=g, device="cuda") * scale
    if case["op"] == "rotary":
        B, T, D = case["batch"], case["tokens"], case["head_dim"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # projection outputs [B, T, heads * D], seen as heads
        q = normal(B, T, case["heads"], D).to(dtype).permute(0, 2, 1, 3)
        k = normal(B, T, case["kv_heads"], D).to(dtype).permute(0, 2, 1, 3)
        freq, magnitude = _frequencies(case)
        positions = None
        if case["positions"] == "row":  # one row for all: the first tokens are padding and stand at 0
            positions = (torch.arange(T, device="cuda") - T // 16).clamp(min=0)
        elif case["positions"] == "rows":  # every row starts at a place of its own
            start = torch.randint(0, case["far"] + 1, (B, 1), generator=g, device="cuda")
            positions = start + torch.arange(T, device="cuda")
        return dict(op="rotary", q=q, k=k, freq=freq.cuda(), magnitude=magnitude, positions=positions,
                    layout=case["layout"], backward=case["backward"])
    m, k, f = case["tokens"], case["hidden"], case["inner"]
    bf = torch.bfloat16
    s = dict(op="ffn", mode=case["mode"], act=case["act"], x=normal(m, k).to(bf),
             w_gate=normal(f, k, scale=k ** -0.5).to(bf), w_up=normal(f, k, scale=k ** -0.5).to(bf),
             w_down=normal(k, f, scale=f ** -0.5).to(bf))
    if case["mode"].startswith("backward"):  # what the forward pass kept, and the gradient that comes in
        s["gate"] = (s["x"] @ s["w_gate"].t()).to(bf)
        s["up"] = (s["x"] @ s["w_up"].t()).to(bf)
        s["dout"] = normal(m, k).to(bf)
    return s


# ---------------------------------------------------------------------------
# one pass


def _turn(x, cos, sin, layout):
    """x [B, H, T, D] with its leading pairs turned; cos and sin [1 or B, 1, T, pairs] in 32 bits."""
    n = cos.shape[-1]
    y = x.float()
    if layout == "half":
        a, b = y[..., :n], y[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, y[..., 2 * n:]), -1).to(x.dtype)


def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def run(state):
    s = state
    if s["op"] == "rotary":
        if own:
            call = _ltxattn().rotary_embed_backward if s["backward"] else _ltxattn().rotary_embed
            return call(s["q"], s["freq"], k=s["k"], positions=s["positions"], layout=s["layout"],
                        magnitude=s["magnitude"])
        positions = s["positions"]
        if positions is None:
            positions = torch.arange(s["q"].shape[2], device="cuda")
        angle = positions.reshape(-1, 1, positions.shape[-1], 1).double() * s["freq"]
        cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
        if s["backward"]:
            sin = -sin
        return _turn(s["q"], cos, sin, s["layout"]), _turn(s["k"], cos, sin, s["layout"])
    if own:
        L = _ltxattn()
        if s["mode"].startswith("backward"):
            dx, dg, du, dd = L.gated_ffn_backward(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["gate"], s["up"],
                                                  s["dout"], activation=s["act"], need_dw=s["mode"] == "backward")
            return (dx, dg, du, dd) if s["mode"] == "backward" else dx
        return L.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=s["act"],
                           save=s["mode"] == "save")
    x, wd = s["x"].float(), s["w_down"].float()
    wg, wu = s["w_gate"].float(), s["w_up"].float()
    bf = torch.bfloat16
    if s["mode"] in ("forward", "save"):
        gate, up = x @ wg.t(), x @ wu.t()
        y = ((_act(gate, s["act"])[0] * up) @ wd.t()).to(bf)
        return y if s["mode"] == "forward" else (y, gate.to(bf), up.to(bf))
    gate, up, dout = s["gate"].float(), s["up"].float(), s["dout"].float()
    a, slope = _act(gate, s["act"])
    dh = dout @ wd
    dgate, dup = dh * up * slope, dh * a
    dx = (dgate @ wg + dup @ wu).to(bf)
    if s["mode"] == "backward_x":
        return dx
    return dx, (dgate.t() @ x).to(bf), (dup.t() @ x).to(bf), (dout.t() @ (a * up)).to(bf)


def work(case):
    if case["op"] == "rotary":
        B, T, D = case["batch"], case["tokens"], case["head_dim"]
        size = 2 if case["dtype"] == "bf16" else 4
        n = B * T * (case["heads"] + case["kv_heads"])
        rows = {"count": 0, "row": T, "rows": B * T}[case["positions"]]
        return {"bytes": 2 * n * D * size + 8 * rows + 4 * case["rotary"], "flops": 3 * n * case["rotary"]}
    m, k, f = case["tokens"], case["hidden"], case["inner"]
    weights, rows, wide = 3 * k * f, m * k, m * f
    mode = case["mode"]
    if mode == "forward":
        return {"bytes": 2 * (weights + 2 * rows), "flops": 6 * m * k * f}
    if mode == "save":
        return {"bytes": 2 * (weights + 2 * rows + 2 * wide), "flops": 6 * m * k * f}
    if mode == "backward_x":  # the weights, dout, gate and up, and dx
        return {"bytes": 2 * (weights + 2 * rows + 2 * wide), "flops": 6 * m * k * f}
    return {"bytes": 2 * (2 * weights + 3 * rows + 2 * wide), "flops": 12 * m * k * f}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_rotary(case, s):
    B, T, D, d = case["batch"], case["tokens"], case["head_dim"], case["rotary"]
    place = torch.arange(T, device="cuda").expand(B, T) if s["positions"] is None else s["positions"].expand(B, T)
    angle = place.to(torch.float64)[:, :, None] * s["freq"][None, None, :]
    if case["backward"]:
        angle = -angle
    spin = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]  # complex numbers, [B, 1, T, d/2]

    def one(x):
        out = x.to(torch.float64, copy=True, memory_format=torch.contiguous_format)
        if case["layout"] == "half":
            z = torch.complex(out[..., :d // 2], out[..., d // 2:d]) * spin
            out[..., :d // 2], out[..., d // 2:d] = z.real, z.imag
        else:
            z = torch.view_as_complex(out[..., :d].reshape(*out.shape[:-1], d // 2, 2)) * spin
            out[..., :d] = torch.view_as_real(z).flatten(-2)
        return out

    return one(s["q"]), one(s["k"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    D = {n: t.double() for n, t in s.items() if torch.is_tensor(t)}
    gate = D.get("gate", None)
    if gate is None:
        gate = torch.einsum("mk,fk->mf", D["x"], D["w_gate"])
    up = D["up"] if "up" in D else torch.einsum("mk,fk->mf", D["x"], D["w_up"])
    # the activation is gate * share: the share's slope comes from the share itself
    if case["act"] == "silu":
        share = torch.sigmoid(gate)
        slope = torch.sigmoid(gate) * torch.sigmoid(-gate)
    elif case["act"] == "gelu_tanh":  # (1 + tanh z) / 2 is the sigmoid of 2 z
        z = 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        share = torch.sigmoid(z)
        slope = share * torch.sigmoid(-z) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * gate ** 2)
    else:
        share = 0.5 * torch.erfc(-gate / math.sqrt(2))
        slope = torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
    h = gate * share * up
    if case["mode"] in ("forward", "save"):
        y = torch.einsum("mf,nf->mn", h, D["w_down"])
        return y if case["mode"] == "forward" else (y, gate, up)
    dh = torch.einsum("mn,nf->mf", D["dout"], D["w_down"])
    dgate = dh * up * (share + gate * slope)
    dup = dh * gate * share
    dx = torch.einsum("mf,fk->mk", dgate, D["w_gate"]) + torch.einsum("mf,fk->mk", dup, D["w_up"])
    if case["mode"] == "backward_x":
        return dx
    return (dx, torch.einsum("mf,mk->fk", dgate, D["x"]), torch.einsum("mf,mk->fk", dup, D["x"]),
            torch.einsum("mn,mf->nf", D["dout"], h))
