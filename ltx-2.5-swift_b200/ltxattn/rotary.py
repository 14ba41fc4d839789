"""Rotary positions from token indices (``ltxattn_rotary_embed``).

* ``rotary_frequencies(rotary_dim, ...)`` gives the angle of every pair per
  position, stretched for long contexts if asked, and the factor on what is
  turned; both are made once and kept.
* ``rotary_embed(q, frequencies, k=k, ...)`` turns queries and (grouped) keys in
  one launch, as an attention with grouped KV heads needs before it
  (GemmaTextEncoder.swift:173,193).
* ``rotary_embed_backward(dq, frequencies, k=dk, ...)`` takes their gradients back.

The DiT's own split RoPE, which reads per-head tables and rounds every product
to bf16, is ``apply_split_rope``.
"""
from __future__ import annotations

import ctypes
import operator
from typing import Optional, Tuple

import torch

from . import _lib
from .backend import Failure, _check_cuda, _dtype_code, _on, _written

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       trained_length: float = 0.0, fast: float = 32.0, slow: float = 1.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """Angles per position of ``rotary_dim / 2`` pairs (float64, on ``device``) and the magnitude.

    ``scaling`` stretches them for contexts ``factor`` times the trained one:
    "linear" all alike; "ntk" through the base, so that the fastest pair stays;
    "yarn" and "bands" leave pairs of more than ``fast`` turns in
    ``trained_length`` alone, stretch those of fewer than ``slow`` and ramp
    between (over the pair index, or over the number of turns; "yarn" also
    scales what is turned by 0.1 ln(factor) + 1).
    """
    if scaling not in SCALINGS:
        raise Failure("arg", f"scaling {scaling!r} is none of {', '.join(SCALINGS)}", _lib.ERR_ARG)
    rotary_dim = operator.index(rotary_dim)
    if not 0 <= rotary_dim < 2 ** 31:  # the C call's field would wrap
        raise Failure("shape", f"rotary_dim ({rotary_dim}) must be even and >= 2, in 32 bits", _lib.ERR_SHAPE)
    a = _lib.RotaryFrequencyArgs(rotary_dim, SCALINGS[scaling], float(theta), float(factor),
                                 float(trained_length), float(fast), float(slow))
    out = (ctypes.c_double * max(1, rotary_dim // 2))()
    magnitude = ctypes.c_float(1.0)
    rc = _lib.load().ltxattn_rotary_frequencies(ctypes.byref(a), out, ctypes.byref(magnitude))
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    return torch.tensor(list(out), dtype=torch.float64).to(device), magnitude.value


def _refuse(name: str, t, shape, dtype, device: int):
    """The failure that describes why t is not a [B, heads, tokens, D] view of that kind."""
    _check_cuda(name, t)
    if t.get_device() != device:
        raise Failure("arg", f"{name} is on {t.device}, q on cuda:{device}", _lib.ERR_ARG)
    if t.shape != shape:
        raise Failure.shape(name, t.shape, str(list(shape)))
    if t.dtype != dtype:
        raise Failure("dtype", f"{name} is {t.dtype}, expected {dtype}", _lib.ERR_DTYPE)
    raise Failure("align", f"{name} must have a unit stride in its last dim", _lib.ERR_ALIGN)


def _view(name: str, t: torch.Tensor, shape, dtype, device: int):
    """(address, stride_b, stride_h, stride_t) of a [B, heads, tokens, D] tensor."""
    if not isinstance(t, torch.Tensor) or t.get_device() != device or t.shape != shape or t.dtype != dtype:
        _refuse(name, t, shape, dtype, device)
    sb, sh, st, sd = t.stride()
    if sd != 1:
        _refuse(name, t, shape, dtype, device)
    return t.data_ptr(), sb, sh, st


def _new_like(t: torch.Tensor):
    """An output in the layout of its input, and its view."""
    out = torch.empty_like(t)
    sb, sh, st, sd = out.stride()
    if sd != 1:
        out = t.new_empty(t.shape)
        sb, sh, st, sd = out.stride()
    return out, (out.data_ptr(), sb, sh, st)


_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_NOTHING = (0, 0, 0, 0)


# A small call is bound by what happens here, so each property is read once and the arguments are packed straight
# into the C struct's bytes: 10 us a call, of which 4 are the launch and 3 the outputs, against 15 with one ctypes
# object per view.
def _embed(q, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, inverse):
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        _check_cuda("q", q)
    shape, dtype, device = q.shape, q.dtype, q.get_device()
    if len(shape) != 4:
        raise Failure.shape("q", shape, "[B, heads, tokens, headDim]")
    B, H, T, D = shape
    code, order = _DTYPES.get(dtype), LAYOUTS.get(layout)
    if code is None:
        _dtype_code(q)
    if order is None:
        raise Failure("arg", f"layout {layout!r} is neither 'half' nor 'interleaved'", _lib.ERR_ARG)
    if not isinstance(frequencies, torch.Tensor) or frequencies.get_device() != device:
        _refuse("frequencies", frequencies, None, torch.float64, device)
    pairs = frequencies.shape
    if frequencies.dtype != torch.float64 or len(pairs) != 1 or not frequencies.is_contiguous():
        raise Failure.shape("frequencies", pairs, "[rotaryDim / 2] float64, contiguous")
    q_sb, q_sh, q_st, unit = q.stride()
    if unit != 1:
        _refuse("q", q, shape, dtype, device)
    kv_heads, vk, v_out_k = 0, _NOTHING, _NOTHING
    if k is not None:
        k_shape = k.shape if isinstance(k, torch.Tensor) else ()
        kv_heads = k_shape[1] if len(k_shape) == 4 else 0
        k_shape = (B, kv_heads, T, D)
        vk = _view("k", k, k_shape, dtype, device)
    elif out_k is not None:
        raise Failure("arg", "out_k without k", _lib.ERR_ARG)
    at, bits, at_sb, at_st = 0, 0, 0, 0
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.get_device() != device:
            _refuse("positions", positions, None, None, device)
        kind, at_shape, strides = positions.dtype, positions.shape, positions.stride()
        bits = 64 if kind == torch.int64 else 32
        if bits == 32 and kind != torch.int32:
            raise Failure("dtype", f"positions are {kind}, expected int64 or int32", _lib.ERR_DTYPE)
        if at_shape != (B, T) and at_shape != (T,) and at_shape != (1, T):
            raise Failure.shape("positions", at_shape, f"[{T}] or [1|{B}, {T}]")
        at, at_st = positions.data_ptr(), strides[-1]
        if len(at_shape) == 2 and at_shape[0] > 1:
            at_sb = strides[0]
    given = [t for t in (out_q, out_k) if t is not None]
    with _on(device, stream) as st:
        if out_q is None:
            out_q, v_out_q = _new_like(q)
        else:
            v_out_q = _view("out_q", out_q, shape, dtype, device)
        if k is not None:
            if out_k is None:
                out_k, v_out_k = _new_like(k)
            else:
                v_out_k = _view("out_k", out_k, k_shape, dtype, device)
        try:
            args = _lib.ROTARY_EMBED_ARGS.pack(code, B, T, H, kv_heads, D, 2 * pairs[0], order, inverse, magnitude,
                                               q.data_ptr(), q_sb, q_sh, q_st, *v_out_q, *vk, *v_out_k,
                                               frequencies.data_ptr(), at, bits, at_sb, at_st, offset)
        except _lib.PACK_ERRORS as e:
            raise Failure("arg", f"a size, offset or magnitude that the call cannot take: {e}", _lib.ERR_ARG) from None
        rc = _lib.load().ltxattn_rotary_embed(args, st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    if given:
        _written(given)
    return out_q if k is None else (out_q, out_k)


def rotary_embed(q: torch.Tensor, frequencies: torch.Tensor, k: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, offset: int = 0, layout: str = "half",
                 magnitude: float = 1.0, out_q: Optional[torch.Tensor] = None,
                 out_k: Optional[torch.Tensor] = None, stream=None):
    """q [B, heads, tokens, D] (and k [B, kvHeads, tokens, D]) with their leading
    ``2 * len(frequencies)`` elements per head turned by ``position * frequency``.

    ``positions`` is int64 or int32, [tokens] or [1|B, tokens]; without it token t
    stands at t.  ``offset`` is added to every position (a decoded token's place in
    its cache).  ``layout`` "half" turns element j with j + rotaryDim / 2,
    "interleaved" 2j with 2j + 1.  Angles are formed in fp64, each element is
    rounded once.  Outputs may be the inputs themselves, or a cache's slots.
    Results carry no graph: gradients are ``rotary_embed_backward``'s.
    Returns the turned q, or (q, k).
    """
    return _embed(q, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, 0)


def rotary_embed_backward(dq: torch.Tensor, frequencies: torch.Tensor, k: Optional[torch.Tensor] = None,
                          positions: Optional[torch.Tensor] = None, offset: int = 0, layout: str = "half",
                          magnitude: float = 1.0, out_q: Optional[torch.Tensor] = None,
                          out_k: Optional[torch.Tensor] = None, stream=None):
    """The gradients with respect to ``rotary_embed``'s inputs, from those of its
    outputs ``dq`` (and ``k``, the gradient of the turned keys): the same turn the
    other way, with the same magnitude."""
    return _embed(dq, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, 1)
