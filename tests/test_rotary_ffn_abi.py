"""The rotary and feed-forward entry points without a GPU: struct layouts, the frequency tables and
the refusals, all of which come before any device work."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from ltxattn import Failure, _lib, gated_ffn, gated_ffn_backward, rotary_embed, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"ltxattn_rotary_frequency_args": _lib.RotaryFrequencyArgs, "ltxattn_rotary_embed_args": _lib.RotaryEmbedArgs,
           "ltxattn_gated_ffn_args": _lib.GatedFfnArgs, "ltxattn_gated_ffn_bwd_args": _lib.GatedFfnBwdArgs}


def test_ctypes_layout_matches_the_header(tmp_path):
    lines = []
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ltxattn.h"\nint main(void) {\n' +
                   "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want


@pytest.mark.parametrize("packer,py", [(_lib.ROTARY_EMBED_ARGS, _lib.RotaryEmbedArgs),
                                       (_lib.GATED_FFN_ARGS, _lib.GatedFfnArgs),
                                       (_lib.GATED_FFN_BWD_ARGS, _lib.GatedFfnBwdArgs)])
def test_packed_arguments_are_the_struct(packer, py):
    def flat(c):  # every scalar field, in order
        return [x for n, t in c._fields_ for x in (flat(getattr(c, n)) if isinstance(getattr(c, n), ctypes.Structure)
                                                   else [getattr(c, n)])]

    assert packer.size == ctypes.sizeof(py)
    values = list(range(1, len(flat(py())) + 1))
    assert flat(py.from_buffer_copy(packer.pack(*values))) == values


# ---- frequencies ----

def table(*args, **kw):
    f, magnitude = rotary_frequencies(*args, device="cpu", **kw)
    assert f.dtype == torch.float64
    return f.tolist(), magnitude


def near(got, want):
    # pow and a few operations in double
    return all(abs(a - b) <= 1e-14 * abs(b) for a, b in zip(got, want)) and len(got) == len(want)


def test_plain_and_linear_frequencies():
    want = [10000.0 ** (-j / 32) for j in range(32)]
    assert near(table(64)[0], want)
    got, magnitude = table(64, scaling="linear", factor=8.0)
    assert near(got, [w / 8 for w in want]) and magnitude == 1.0
    assert table(2, theta=0.5) == ([1.0], 1.0)  # one pair turns by a radian per step whatever the base


def test_ntk_stretches_the_slowest_pair_by_the_factor():
    got, _ = table(64, scaling="ntk", factor=8.0)
    assert got[0] == 1.0 and near(got[-1:], [10000.0 ** (-31 / 32) / 8])
    assert table(2, scaling="ntk", factor=8.0)[0] == [1.0]


def test_yarn_bands():
    n, L, s = 64, 4096.0, 16.0
    plain_, _ = table(2 * n)
    got, magnitude = table(2 * n, scaling="yarn", factor=s, trained_length=L)
    assert magnitude == pytest.approx(0.1 * math.log(s) + 1, rel=2 ** -23)
    pair = lambda r: n * math.log(L / (2 * math.pi * r)) / math.log(1e4)
    low, high = math.floor(pair(32)), math.ceil(pair(1))
    for j in range(n):
        part = min(max((j - low) / (high - low), 0), 1)
        assert near([got[j]], [plain_[j] / s * part + plain_[j] * (1 - part)])
    assert got[:low + 1] == plain_[:low + 1]  # fast pairs are left alone
    assert table(2 * n, scaling="yarn", factor=1.0, trained_length=L) == (pytest.approx(plain_), 1.0)
    # a context so short that no pair turns `slow` times: every pair is stretched, none is NaN
    short, _ = table(8, scaling="yarn", factor=2.0, trained_length=1.0)
    assert all(math.isfinite(f) and f > 0 for f in short)


def test_bands_ramp_over_turns():
    L, s = 8192.0, 8.0
    plain_, _ = table(128, theta=5e5)
    got, magnitude = table(128, theta=5e5, scaling="bands", factor=s, trained_length=L, fast=4.0, slow=1.0)
    assert magnitude == 1.0
    for f, g in zip(plain_, got):
        turns = L * f / (2 * math.pi)
        want = f if turns > 4 else f / s if turns < 1 else f / s * (4 - turns) / 3 + f * (turns - 1) / 3
        assert abs(g - want) <= 1e-13 * want


@pytest.mark.parametrize("kw,kind", [
    (dict(rotary_dim=0), "shape"),
    (dict(rotary_dim=7), "shape"),
    (dict(rotary_dim=-2), "shape"),
    (dict(theta=0.0), "arg"),
    (dict(theta=float("nan")), "arg"),
    (dict(theta=float("inf")), "arg"),
    (dict(scaling="cubic"), "arg"),
    (dict(scaling="linear", factor=0.0), "arg"),
    (dict(scaling="linear", factor=float("nan")), "arg"),
    (dict(scaling="yarn", factor=2.0), "arg"),                                    # no trained length
    (dict(scaling="yarn", factor=2.0, trained_length=64.0, theta=1.0), "arg"),    # all pairs alike: no ramp
    (dict(scaling="bands", factor=2.0, trained_length=64.0, fast=1.0, slow=1.0), "arg"),
    (dict(scaling="bands", factor=2.0, trained_length=64.0, fast=1.0, slow=0.0), "arg"),
])
def test_frequency_refusals(kw, kind):
    with pytest.raises(Failure) as e:
        rotary_frequencies(**{"rotary_dim": 64, "device": "cpu", **kw})
    assert e.value.kind == kind


# ---- refusals of the C entries ----

def rotary_args(**kw):
    a = _lib.RotaryEmbedArgs(dtype=_lib.BF16, batch=2, tokens=4, heads=2, kv_heads=1, head_dim=64, rotary_dim=64,
                             magnitude=1.0, frequencies=1 << 20, position_bits=64)
    for i, n in enumerate(("q", "q_out", "k", "k_out")):
        setattr(a, n, _lib.Tensor(4096 * (i + 1), 512, 64, 128))
    for name, value in kw.items():
        if "." in name:
            setattr(getattr(a, name.split(".")[0]), name.split(".")[1], value)
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), _lib.ERR_DTYPE),
    (dict(batch=-1), _lib.ERR_SHAPE),
    (dict(tokens=-1), _lib.ERR_SHAPE),
    (dict(heads=-1), _lib.ERR_SHAPE),
    (dict(head_dim=0), _lib.ERR_SHAPE),
    (dict(rotary_dim=66), _lib.ERR_SHAPE),     # more than the head
    (dict(rotary_dim=63), _lib.ERR_SHAPE),
    (dict(rotary_dim=0), _lib.ERR_SHAPE),
    (dict(layout=2), _lib.ERR_ARG),
    (dict(frequencies=None), _lib.ERR_ARG),
    (dict(frequencies=(1 << 20) + 4), _lib.ERR_ALIGN),
    (dict(positions=4096, position_bits=16), _lib.ERR_DTYPE),
    (dict(positions=4100), _lib.ERR_ALIGN),
    (dict(positions=4096, position_stride_t=-1), _lib.ERR_SHAPE),
    (dict(head_dim=16384, rotary_dim=16384), _lib.ERR_UNSUPPORTED),
    (dict(tokens=2 ** 30), _lib.ERR_UNSUPPORTED),
    (dict(heads=2 ** 24 + 1), _lib.ERR_UNSUPPORTED),  # steps through the heads are counted in 32 bits
    (dict(kv_heads=2 ** 24 + 1), _lib.ERR_UNSUPPORTED),
    ({"q.data": None}, _lib.ERR_ARG),
    ({"k_out.data": None}, _lib.ERR_ARG),
    ({"q.data": 4097}, _lib.ERR_ALIGN),
    ({"q.stride_t": -64}, _lib.ERR_SHAPE),
    ({"q_out.stride_t": 0}, _lib.ERR_SHAPE),   # an output that repeats rows
    ({"q_out.stride_h": 0}, _lib.ERR_SHAPE),
    ({"q_out.data": 4096, "q_out.stride_t": 64}, _lib.ERR_ARG),  # in place with other strides
    ({"q_out.data": 4096 * 4}, _lib.ERR_ARG),  # both outputs in one place
    ({"k_out.data": 4096}, _lib.ERR_ARG),      # keys over the queries
])
def test_rotary_refusals(kw, status):
    L = _lib.load()
    rc = L.ltxattn_rotary_embed(ctypes.byref(rotary_args(**kw)), None)
    assert rc == status, (rc, _lib.last_error())
    assert "ltxattn_rotary_embed" in _lib.last_error()


def test_calls_without_work_return_before_the_device():
    L = _lib.load()
    for kw in (dict(batch=0), dict(tokens=0), dict(heads=0, kv_heads=0)):
        assert L.ltxattn_rotary_embed(ctypes.byref(rotary_args(frequencies=None, **kw)), None) == _lib.OK
    assert L.ltxattn_rotary_embed(None, None) == _lib.ERR_ARG
    assert L.ltxattn_gated_ffn(ctypes.byref(ffn_args(m=0, x=None)), None) == _lib.OK
    assert L.ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(m=0, dw_gate=None, dw_up=None, dw_down=None)), None) == _lib.OK
    # nothing wanted
    none = dict(dx=None, dw_gate=None, dw_up=None, dw_down=None)
    assert L.ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(**none)), None) == _lib.OK


def _fill(a, names, kw):
    widths = {"x": 64, "w_gate": 64, "w_up": 64, "w_down": 128, "out": 72, "gate": 128, "up": 128, "dout": 72, "dx": 64,
              "dw_gate": 64, "dw_up": 64, "dw_down": 128}
    for i, n in enumerate(names):
        setattr(a, n, 4096 * (i + 1))
        setattr(a, n + "_stride", widths[n])
    a.dtype, a.m, a.hidden, a.inner, a.out_dim = _lib.BF16, 5, 64, 128, 72
    a.workspace, a.workspace_bytes = 1 << 20, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def ffn_args(**kw):
    return _fill(_lib.GatedFfnArgs(), ("x", "w_gate", "w_up", "w_down", "out"), kw)


def bwd_args(**kw):
    return _fill(_lib.GatedFfnBwdArgs(), ("x", "w_gate", "w_up", "w_down", "gate", "up", "dout", "dx", "dw_gate",
                                          "dw_up", "dw_down"), kw)


BOTH = [
    (dict(dtype=_lib.F32), _lib.ERR_DTYPE),
    (dict(activation=3), _lib.ERR_ARG),
    (dict(activation=-1), _lib.ERR_ARG),
    (dict(m=-1), _lib.ERR_SHAPE),
    (dict(inner=0), _lib.ERR_SHAPE),
    (dict(hidden=60), _lib.ERR_UNSUPPORTED),
    (dict(inner=100), _lib.ERR_UNSUPPORTED),
    (dict(out_dim=71), _lib.ERR_UNSUPPORTED),
    (dict(x=None), _lib.ERR_ARG),
    (dict(w_up=None), _lib.ERR_ARG),
    (dict(w_down=None), _lib.ERR_ARG),
    (dict(x=4098), _lib.ERR_ALIGN),
    (dict(w_gate_stride=68), _lib.ERR_ALIGN),
    (dict(w_down_stride=120), _lib.ERR_SHAPE),
    (dict(workspace=None), _lib.ERR_WORKSPACE),
    (dict(workspace_bytes=1000), _lib.ERR_WORKSPACE),
    (dict(workspace=(1 << 20) + 16), _lib.ERR_ALIGN),
]


@pytest.mark.parametrize("kw,status", BOTH + [
    (dict(out=None), _lib.ERR_ARG),
    (dict(gate=1 << 16, gate_stride=128), _lib.ERR_ARG),                             # gate without up
    (dict(gate=1 << 16, gate_stride=64, up=1 << 17, up_stride=128), _lib.ERR_SHAPE),
    (dict(gate=1 << 16, gate_stride=128, up=1 << 16, up_stride=128), _lib.ERR_ARG),  # gate and up in one place
    (dict(out=4096, out_stride=72), _lib.ERR_ARG),                                   # y over x
])
def test_ffn_refusals(kw, status):
    rc = _lib.load().ltxattn_gated_ffn(ctypes.byref(ffn_args(**kw)), None)
    assert rc == status, (rc, _lib.last_error())


@pytest.mark.parametrize("kw,status", BOTH + [
    (dict(gate=None), _lib.ERR_ARG),
    (dict(up_stride=64), _lib.ERR_SHAPE),
    (dict(dout=4104), _lib.ERR_ALIGN),
    (dict(dx_stride=8), _lib.ERR_SHAPE),
    (dict(dw_down=4097), _lib.ERR_ALIGN),
    (dict(dx=4096), _lib.ERR_ARG),              # dx over x
    (dict(dw_up=4096 * 9), _lib.ERR_ARG),       # over dw_gate
])
def test_ffn_backward_refusals(kw, status):
    rc = _lib.load().ltxattn_gated_ffn_bwd(ctypes.byref(bwd_args(**kw)), None)
    assert rc == status, (rc, _lib.last_error())


def test_workspaces_grow_with_the_tokens():
    L = _lib.load()
    for args, query, planes in ((ffn_args, L.ltxattn_gated_ffn_workspace, 1), (bwd_args, L.ltxattn_gated_ffn_bwd_workspace, 3)):
        assert query(None) == 0 and query(ctypes.byref(args(m=0))) == 0
        for m in (1, 5, 129, 100000):
            need = query(ctypes.byref(args(m=m)))
            assert need == planes * ((m * 128 * 2 + 255) // 256 * 256)


# ---- refusals of the Python calls ----

def test_host_tensors_are_refused():
    f, _ = rotary_frequencies(64, device="cpu")
    with pytest.raises(Failure) as e:
        rotary_embed(torch.zeros(1, 2, 3, 64), f)
    assert e.value.kind == "arg"
    w = torch.zeros(64, 64, dtype=torch.bfloat16)
    for call in (lambda: gated_ffn(w, w, w, w), lambda: gated_ffn_backward(w, w, w, w, w, w, w),
                 lambda: gated_ffn(w, w, w, w, activation="relu")):
        with pytest.raises(Failure) as e:
            call()
        assert e.value.kind == "arg"
