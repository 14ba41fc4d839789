"""The gated feed-forward block on a B200, path by path: the kernel for many tokens in every product and with more than
a tile to a pair of CTAs, the exchange of sums in two pieces, and what stands before a call in its stream.

`forward` and `backward` of test_gated_ffn_gpu give the block in 64 bits and each tensor's bound.  Their 2^-18 for an
activation and its slope, relative to 1 + |gate|, holds for what the kernels compute: the exponential is off by
2 + 1.2 |x| units of 2^-24 at argument x and is multiplied by a share of at most e^x, so by under 3 units of the share's
size 1; the fast division adds 2, the fitted polynomial of the erf form 7, the products and sums around them 4; and a
slope is at most 1 + |gate| times as steep in the share: under 16 units, 2^-20.
"""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

from ltxattn import device_status, gated_ffn, gated_ffn_backward
from test_gated_ffn_gpu import ACTS, backward, check, forward, make

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(autouse=True)
def no_kernel_timeouts():
    yield
    assert device_status(clear=True) == 0, "a kernel wait timed out"


# tokens, hidden, inner, out: test_gated_ffn_plan.py holds what they are chosen for
WIDE = [
    (3001, 1544, 2056, 1800),
    (2817, 1800, 2312, 1544),  # one row past a tile, a few columns past a piece
    (5000, 2056, 2312, 2072),  # three tiles to some pairs
]
# and the tokens of a tile, and the CTAs that share one
EXCHANGE = [
    (105, 1024, 28672, 64, 112, 1),
    (112, 3328, 11776, 64, 112, 2),
    (105, 1792, 9728, 64, 112, 3),
    (112, 3840, 4608, 64, 112, 6),
    (128, 1536, 28672, 72, 128, 1),
    (126, 4096, 11776, 64, 128, 2),
    (128, 2048, 9728, 64, 128, 3),
    (113, 4096, 4608, 136, 128, 6),
    (300, 3328, 5120, 64, 112, 2),  # the last tile's tokens fit in one piece
]


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,hidden,inner,out", WIDE)
def test_many_tokens(kind, m, hidden, inner, out):
    x, wg, wu, wd, dout = make(m + inner, m, hidden, inner, out)
    want, want_gate, want_up = forward(x, wg, wu, wd, kind)
    check("y", gated_ffn(x, wg, wu, wd, kind), want)
    y, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    check("y with its gate kept", y, want)
    check("gate", gate, want_gate)
    check("up", up, want_up)
    got = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind)
    for name, g, w in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, backward(x, wg, wu, wd, gate, up, dout, kind)):
        check(name, g, w)
    only = gated_ffn_backward(None, wg, wu, wd, gate, up, dout, kind, need_dw=False)
    assert torch.equal(only[0], got[0])
    only = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind, need_dx=False)
    assert all(torch.equal(a, b) for a, b in zip(only[1:], got[1:]))


@pytest.mark.parametrize("m,hidden,inner,out,columns,cluster", EXCHANGE)
def test_sums_exchanged_in_two_pieces(m, hidden, inner, out, columns, cluster):
    x, wg, wu, wd, _ = make(m + inner, m, hidden, inner, out)
    want, want_gate, want_up = forward(x, wg, wu, wd, "silu")
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    check("y", y, want)
    check("gate", gate, want_gate)
    check("up", up, want_up)
    assert torch.equal(gated_ffn(x, wg, wu, wd), y)


@pytest.fixture(scope="module")
def stays_on(tmp_path_factory):
    lib = tmp_path_factory.mktemp("stays_on") / "stays_on.so"
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-shared", "-Xcompiler", "-fPIC",
                    os.path.join(HERE, "c", "stays_on.cu"), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib)).launch_stays_on


@pytest.mark.parametrize("m", [1, 60])
def test_a_call_behind_a_long_kernel(stays_on, m):
    # The kernel before lets the call's first kernel start at once and stays for 2.4 s, longer than a wait in a kernel
    # may take (2 s): those waits are for the kernel's own loads and products, and start when it may run.
    x, wg, wu, wd, dout = make(31, m, 256, 520, 264)
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    grads = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert stays_on(ctypes.c_uint32(2400), stream) == 0
    again = gated_ffn(x, wg, wu, wd, save=True)
    assert stays_on(ctypes.c_uint32(2400), stream) == 0
    grads_again = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    torch.cuda.synchronize()
    assert device_status(clear=True) == 0
    assert all(torch.equal(a, b) for a, b in zip(again, (y, gate, up)))
    assert all(torch.equal(a, b) for a, b in zip(grads_again, grads))


FAR = {"silu": (-91.5, -80.0), "gelu_tanh": (-10.0625, -9.0), "gelu": (-13.0, -11.0)}


def far64(g, kind):
    """The activation and its slope, without a sum of 1 and what it cancels."""
    if kind == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    z, dz = (g, 1.0) if kind == "silu" else (c * (g + 0.044715 * g ** 3), c * (1 + 0.134145 * g * g))
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * dz


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,hidden,inner,out", [(96, 64, 128, 72), WIDE[0]])
def test_activations_down_to_the_smallest_numbers(kind, m, hidden, inner, out):
    # Results from 1e-33 down to 1.6e-38, bf16's (and fp32's) smallest with all their digits being 1.2e-38.  With up = 1
    # and w_down the identity, y = act(gate), one rounding: 2^-8.  The exponential of arguments to 92 is off by under
    # 112 units of 2^-24, twice that with what its argument is off in the tanh form, shares down to 1e-40 have 2^-17
    # in fp32, and the sums and products around them a few 2^-24: under 2^-14 together.
    gate = torch.linspace(*FAR[kind], m).cuda().bfloat16()
    x = torch.zeros(m, hidden, device="cuda", dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = gate, 1.0
    w_gate, w_up = torch.zeros(2, inner, hidden, device="cuda", dtype=torch.bfloat16)
    w_gate[:, 0], w_up[:, 1] = 1.0, 1.0
    w_down = torch.eye(out, inner, device="cuda", dtype=torch.bfloat16)
    a, slope = far64(gate.double(), kind)
    near = lambda got, want: bool(((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -14) * want.abs()).all())
    y, kept, up = gated_ffn(x, w_gate, w_up, w_down, kind, save=True)
    assert torch.equal(kept, gate[:, None].expand(m, inner))
    assert near(y, a[:, None].expand(m, out))
    # with dout = 1 for the first output alone, dx has the slope beside the gate's input and the activation beside up's
    dout = torch.zeros(m, out, device="cuda", dtype=torch.bfloat16)
    dout[:, 0] = 1.0
    dx = gated_ffn_backward(x, w_gate, w_up, w_down, kept, up, dout, kind, need_dw=False)[0]
    assert near(dx[:, 0], slope) and near(dx[:, 1], a)


def test_outputs_given_by_the_caller_count_as_written():
    x, wg, wu, wd, dout = make(32, 5, 64, 128, 72)
    _, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    out, dx, dwg, dwu, dwd = (torch.empty_like(t) for t in (dout, x, wg, wu, wd))
    inputs = (x, wg, wu, wd, gate, up, dout)
    before = [t._version for t in inputs]
    gated_ffn(x, wg, wu, wd, out=out)
    gated_ffn_backward(x, wg, wu, wd, gate, up, dout, dx=dx, dw_gate=dwg, dw_up=dwu, dw_down=dwd)
    assert all(t._version > 0 for t in (out, dx, dwg, dwu, dwd))
    assert [t._version for t in inputs] == before


@pytest.mark.parametrize("m", [3, 100])
def test_weights_that_the_call_before_wrote(m):
    # The second product of a call loads its weights before the first is complete; what wrote them may be the call
    # before.  Outputs of one call are the next one's weights, each in turn, with nothing between the calls.
    hidden, inner, out = 256, 1024, 512
    x, wg, wu, wd, dout = make(33, m, hidden, inner, out)
    makers = {"w_gate": make(34, inner, 2048, 4096, hidden)[:4], "w_up": make(35, inner, 2048, 4096, hidden)[:4],
              "w_down": make(36, out, 2048, 4096, inner)[:4]}
    base = {"w_gate": wg, "w_up": wu, "w_down": wd}
    _, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    for name, maker in makers.items():
        new = gated_ffn(*maker)
        torch.cuda.synchronize()
        weights = {**base, name: new}
        want = gated_ffn(x, **weights)
        want_dx = gated_ffn_backward(None, **weights, gate=gate, up=up, dout=dout, need_dw=False)[0]
        for _ in range(3):
            buf = torch.full_like(new, float("nan"))
            torch.cuda.synchronize()
            gated_ffn(*maker, out=buf)
            assert torch.equal(gated_ffn(x, **{**base, name: buf}), want), name
            buf.fill_(float("nan"))
            torch.cuda.synchronize()
            gated_ffn(*maker, out=buf)
            dx = gated_ffn_backward(None, **{**base, name: buf}, gate=gate, up=up, dout=dout, need_dw=False)[0]
            assert torch.equal(dx, want_dx), name


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,hidden,inner,out", [(20, 64, 136, 72), WIDE[0]])
def test_infinite_tokens(kind, m, hidden, inner, out):
    # positive weights: an infinite input makes gate and up infinite, the activation of the one keeps its sign, and the
    # output is infinite with it; other tokens do not see it
    x, wg, wu, wd, dout = make(37, m, hidden, inner, out)
    wg, wu, wd = wg.abs() + 2.0 ** -9, wu.abs() + 2.0 ** -9, wd.abs() + 2.0 ** -9
    y, gate, up = gated_ffn(x, wg, wu, wd, kind, save=True)
    spoiled = x.clone()
    spoiled[1, 5] = float("inf")
    z, zgate, zup = gated_ffn(spoiled, wg, wu, wd, kind, save=True)
    rest = torch.arange(m, device="cuda") != 1
    assert bool((zgate[1] == float("inf")).all()) and bool((zup[1] == float("inf")).all())
    assert bool((z[1] == float("inf")).all()) and torch.equal(z[rest], y[rest])
    # an infinite gradient spoils its own token's dx, and the weights' gradients as sums over tokens
    dx = gated_ffn_backward(None, wg, wu, wd, gate, up, dout, kind, need_dw=False)[0]
    dout[2, 3] = float("inf")
    got = gated_ffn_backward(x, wg, wu, wd, gate, up, dout, kind)
    keep = torch.arange(m, device="cuda") != 2
    assert torch.equal(got[0][keep], dx[keep]) and not bool(got[0][2].isfinite().any())
    others = torch.arange(out, device="cuda") != 3
    assert bool(got[3][others].isfinite().all()) and not bool(got[3][3].isfinite().any())


def test_tokens_of_any_rank():
    x, wg, wu, wd, dout = make(38, 12, 64, 128, 72)
    y, gate, up = gated_ffn(x, wg, wu, wd, save=True)
    grads = gated_ffn_backward(x, wg, wu, wd, gate, up, dout)
    # one token without a leading dim
    one, g1, u1 = gated_ffn(x[4], wg, wu, wd, save=True)
    want1 = gated_ffn(x[4:5], wg, wu, wd, save=True)
    assert all(a.dim() == 1 and torch.equal(a, b[0]) for a, b in zip((one, g1, u1), want1))
    got1 = gated_ffn_backward(x[4], wg, wu, wd, g1, u1, dout[4])
    want1 = gated_ffn_backward(x[4:5], wg, wu, wd, want1[1], want1[2], dout[4:5])
    assert got1[0].shape == (64,) and torch.equal(got1[0], want1[0][0])
    assert all(torch.equal(a, b) for a, b in zip(got1[1:], want1[1:]))
    # leading dims that do not collapse into rows are copied, on the call's own stream
    t4 = lambda t: t.view(2, 3, 2, -1).transpose(1, 2).contiguous().transpose(1, 2)
    side = torch.cuda.Stream()
    x4, gate4, up4, dout4 = t4(x), t4(gate), t4(up), t4(dout)
    torch.cuda.synchronize()
    y4 = gated_ffn(x4, wg, wu, wd, stream=side)
    got4 = gated_ffn_backward(x4, wg, wu, wd, gate4, up4, dout4, stream=side)
    torch.cuda.synchronize()
    assert y4.shape == (2, 3, 2, 72) and torch.equal(y4.reshape(12, 72), y)
    assert got4[0].shape == (2, 3, 2, 64) and torch.equal(got4[0].reshape(12, 64), grads[0])
    assert all(torch.equal(a, b) for a, b in zip(got4[1:], grads[1:]))
