"""The gated feed-forward block (``ltxattn_gated_ffn``) and its gradient.

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

bf16, fp32 accumulation; the product between the projections is rounded once.
``linear`` is the plain projection beside it.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .backend import Failure, _check_cuda, _on

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "gelu": 2}


def _matrix(name: str, t: torch.Tensor, rows: int, cols: int, device: int) -> tuple:
    """(address, row stride) of a bf16 [rows, cols] matrix on that device."""
    _check_cuda(name, t)
    if t.dtype != torch.bfloat16:
        raise Failure("dtype", f"{name} must be bfloat16", _lib.ERR_DTYPE)
    if t.shape != (rows, cols):
        raise Failure.shape(name, t.shape, f"[{rows}, {cols}]")
    if t.get_device() != device:
        raise Failure("arg", f"{name} is on {t.device}, the tokens on cuda:{device}", _lib.ERR_ARG)
    stride, unit = t.stride()
    if unit != 1 and cols > 1:
        raise Failure("align", f"{name} must have a unit stride along its last dim", _lib.ERR_ALIGN)
    return t.data_ptr(), stride if rows > 1 else cols


def _rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """[..., cols] as rows: a view when the leading dims collapse into one row stride, else a copy."""
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise Failure("arg", f"activation {name!r} is none of {', '.join(ACTIVATIONS)}", _lib.ERR_ARG)
    return ACTIVATIONS[name]


def _output(name: str, t: Optional[torch.Tensor], shape, like: torch.Tensor):
    """An output of that shape: the caller's, or a new one on the device of ``like``."""
    if t is None:
        return like.new_empty(shape, dtype=torch.bfloat16)
    if t.shape != tuple(shape):
        raise Failure.shape(name, t.shape, str(list(shape)))
    return t


def _workspace(need: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return like.new_empty((need,), dtype=torch.uint8) if need else None


def _out_rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """The same for an output, of which a copy is no use."""
    rows = _rows(name, t)
    if rows.numel() and rows.data_ptr() != t.data_ptr():
        raise Failure("align", f"{name}'s leading dims must collapse into rows of one stride", _lib.ERR_ALIGN)
    return rows


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu", save: bool = False, out: Optional[torch.Tensor] = None, stream=None):
    """x [..., hidden] -> [..., out]; w_gate and w_up [inner, hidden], w_down [out, inner] (the
    checkpoint's [out, in] layout).

    ``activation`` is "silu", "gelu_tanh" or "gelu" (erf).  With ``save`` the result
    is ``(y, gate, up)``, the last two being what ``gated_ffn_backward`` needs:
    ``x w_gate^T`` and ``x w_up^T``, [..., inner].  hidden, inner and out are
    multiples of 8 and rows 16-byte aligned.
    """
    act = _activation(activation)
    _check_cuda("x", x)
    if x.dim() < 1:
        raise Failure.shape("x", x.shape, "[..., hidden]")
    device = x.get_device()
    for name, w in (("w_gate", w_gate), ("w_down", w_down)):
        if not isinstance(w, torch.Tensor) or w.dim() != 2:
            raise Failure.shape(name, getattr(w, "shape", ()), "a matrix")
    inner, out_dim = w_gate.shape[0], w_down.shape[0]
    lead = x.shape[:-1]
    with _on(device, stream) as st:
        x2 = _rows("x", x)
        m, hidden = x2.shape
        y = _output("out", out, lead + (out_dim,), x)
        a = _lib.GatedFfnArgs(_lib.BF16, act, m, hidden, inner, out_dim, *_matrix("x", x2, m, hidden, device),
                              *_matrix("w_gate", w_gate, inner, hidden, device),
                              *_matrix("w_up", w_up, inner, hidden, device),
                              *_matrix("w_down", w_down, out_dim, inner, device),
                              *_matrix("out", _out_rows("out", y), m, out_dim, device))
        gate = up = None
        if save:
            gate = x.new_empty(lead + (inner,))
            up = torch.empty_like(gate)
            a.gate, a.gate_stride, a.up, a.up_stride = gate.data_ptr(), inner, up.data_ptr(), inner
        L = _lib.load()
        need = L.ltxattn_gated_ffn_workspace(ctypes.byref(a))
        ws = _workspace(need, x)
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        rc = L.ltxattn_gated_ffn(ctypes.byref(a), st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    return (y, gate, up) if save else y


def gated_ffn_backward(x: Optional[torch.Tensor], w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       gate: torch.Tensor, up: torch.Tensor, dout: torch.Tensor, activation: str = "silu",
                       need_dx: bool = True, need_dw: bool = True, dx: Optional[torch.Tensor] = None,
                       dw_gate: Optional[torch.Tensor] = None, dw_up: Optional[torch.Tensor] = None,
                       dw_down: Optional[torch.Tensor] = None, stream=None):
    """``(dx, dw_gate, dw_up, dw_down)`` of sum(dout * y), from the ``gate`` and ``up`` that
    ``gated_ffn(..., save=True)`` kept.

    What is not needed is not computed and is None in the result: ``need_dw=False``
    for frozen weights (x may then be None), ``need_dx=False`` for a first layer.
    The ``d...`` arguments give outputs to be written (overwritten, not added to).
    """
    act = _activation(activation)
    _check_cuda("dout", dout)
    if dout.dim() < 1:
        raise Failure.shape("dout", dout.shape, "[..., out]")
    device = dout.get_device()
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2:
        raise Failure.shape("w_gate", getattr(w_gate, "shape", ()), "a matrix")
    inner, hidden = w_gate.shape
    if x is None and need_dw:
        raise Failure("missing", "x is needed for the gradients of w_gate and w_up")
    lead = dout.shape[:-1]
    for name, t, cols in (("x", x, hidden), ("gate", gate, inner), ("up", up, inner)):
        if t is None and name == "x":
            continue
        _check_cuda(name, t)
        if tuple(t.shape) != tuple(lead) + (cols,):
            raise Failure.shape(name, t.shape, str(list(lead) + [cols]))
    with _on(device, stream) as st:
        d2 = _rows("dout", dout)
        m, out_dim = d2.shape
        a = _lib.GatedFfnBwdArgs(_lib.BF16, act, m, hidden, inner, out_dim)

        def put(name, t, rows, cols):
            ptr, stride = _matrix(name, t, rows, cols, device)
            setattr(a, name, ptr)
            setattr(a, name + "_stride", stride)

        if x is not None:
            put("x", _rows("x", x), m, hidden)
        put("w_gate", w_gate, inner, hidden)
        put("w_up", w_up, inner, hidden)
        put("w_down", w_down, out_dim, inner)
        put("gate", _rows("gate", gate), m, inner)
        put("up", _rows("up", up), m, inner)
        put("dout", d2, m, out_dim)
        if need_dx:
            dx = _output("dx", dx, tuple(lead) + (hidden,), dout)
            put("dx", _out_rows("dx", dx), m, hidden)
        else:
            dx = None
        if need_dw:
            dw_gate = _output("dw_gate", dw_gate, (inner, hidden), dout)
            dw_up = _output("dw_up", dw_up, (inner, hidden), dout)
            dw_down = _output("dw_down", dw_down, (out_dim, inner), dout)
            put("dw_gate", dw_gate, inner, hidden)
            put("dw_up", dw_up, inner, hidden)
            put("dw_down", dw_down, out_dim, inner)
        else:
            dw_gate = dw_up = dw_down = None
        L = _lib.load()
        need = L.ltxattn_gated_ffn_bwd_workspace(ctypes.byref(a))
        ws = _workspace(need, dout)
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        rc = L.ltxattn_gated_ffn_bwd(ctypes.byref(a), st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    return dx, dw_gate, dw_up, dw_down
