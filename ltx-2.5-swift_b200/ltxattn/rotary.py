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
from typing import Optional, Tuple

import torch

from . import _lib
from .backend import Failure, _check_cuda, _dtype_code, _view, _on

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
    a = _lib.RotaryFrequencyArgs(int(rotary_dim), SCALINGS[scaling], float(theta), float(factor),
                                 float(trained_length), float(fast), float(slow))
    out = (ctypes.c_double * max(1, int(rotary_dim) // 2))()
    magnitude = ctypes.c_float(1.0)
    rc = _lib.load().ltxattn_rotary_frequencies(ctypes.byref(a), out, ctypes.byref(magnitude))
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    return torch.tensor(list(out), dtype=torch.float64).to(device), magnitude.value


def _embed(q, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, inverse):
    _check_cuda("q", q)
    if q.dim() != 4:
        raise Failure.shape("q", q.shape, "[B, heads, tokens, headDim]")
    B, H, T, D = q.shape
    device = q.device
    if layout not in LAYOUTS:
        raise Failure("arg", f"layout {layout!r} is neither 'half' nor 'interleaved'", _lib.ERR_ARG)
    _check_cuda("frequencies", frequencies)
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise Failure.shape("frequencies", frequencies.shape, "[rotaryDim / 2] float64, contiguous")
    Hk = 0
    tensors = [frequencies]
    if k is not None:
        _check_cuda("k", k)
        if k.dim() != 4 or k.shape[0] != B or k.shape[2] != T or k.shape[3] != D:
            raise Failure.shape("k", k.shape, f"[{B}, kvHeads, {T}, {D}]")
        if k.dtype != q.dtype:
            raise Failure("dtype", "q and k must share one dtype", _lib.ERR_DTYPE)
        Hk = k.shape[1]
        tensors.append(k)
    pos_ptr, pos_bits, pos_sb, pos_st = None, 0, 0, 0
    if positions is not None:
        _check_cuda("positions", positions)
        if positions.dtype not in (torch.int64, torch.int32):
            raise Failure("dtype", f"positions are {positions.dtype}, expected int64 or int32", _lib.ERR_DTYPE)
        shape = tuple(positions.shape)
        if shape not in ((T,), (1, T), (B, T)):
            raise Failure.shape("positions", shape, f"[{T}] or [1|{B}, {T}]")
        pos_ptr, pos_bits, pos_st = positions.data_ptr(), 8 * positions.element_size(), positions.stride(-1)
        pos_sb = positions.stride(0) if len(shape) == 2 and shape[0] > 1 else 0
        tensors.append(positions)
    for name, o, x in (("out_q", out_q, q), ("out_k", out_k, k)):
        if o is not None:
            if x is None:
                raise Failure("arg", f"{name} without its input", _lib.ERR_ARG)
            _check_cuda(name, o)
            if o.dtype != x.dtype:
                raise Failure("dtype", f"{name} must have the dtype of its input", _lib.ERR_DTYPE)
            tensors.append(o)
    for t in tensors:
        if t.device != device:
            raise Failure("arg", f"q is on {device}, another tensor on {t.device}", _lib.ERR_ARG)
    with _on(device, stream) as st:
        out_q = torch.empty_like(q) if out_q is None else out_q
        none = _lib.Tensor()
        if k is not None:
            out_k = torch.empty_like(k) if out_k is None else out_k
            vk, vok = _view("k", k, (B, Hk, T, D)), _view("out_k", out_k, (B, Hk, T, D))
        else:
            vk = vok = none
        a = _lib.RotaryEmbedArgs(_dtype_code(q), B, T, H, Hk, D, 2 * frequencies.shape[0], LAYOUTS[layout],
                                 1 if inverse else 0, magnitude, _view("q", q, (B, H, T, D)),
                                 _view("out_q", out_q, (B, H, T, D)), vk, vok, frequencies.data_ptr(), pos_ptr,
                                 pos_bits, pos_sb, pos_st, offset)
        rc = _lib.load().ltxattn_rotary_embed(ctypes.byref(a), st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
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
    Returns the turned q, or (q, k).
    """
    return _embed(q, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, False)


def rotary_embed_backward(dq: torch.Tensor, frequencies: torch.Tensor, k: Optional[torch.Tensor] = None,
                          positions: Optional[torch.Tensor] = None, offset: int = 0, layout: str = "half",
                          magnitude: float = 1.0, out_q: Optional[torch.Tensor] = None,
                          out_k: Optional[torch.Tensor] = None, stream=None):
    """The gradients with respect to ``rotary_embed``'s inputs, from those of its
    outputs ``dq`` (and ``k``, the gradient of the turned keys): the same turn the
    other way, with the same magnitude."""
    return _embed(dq, frequencies, k, positions, offset, layout, magnitude, out_q, out_k, stream, True)
