"""The gated feed-forward block (``ltxattn_gated_ffn``) and its gradient.

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

bf16, fp32 accumulation; the product between the projections is rounded once.
``linear`` is the plain projection beside it.
"""
from __future__ import annotations

import math
import operator
from typing import Optional

import torch

from . import _lib
from .backend import Failure, _check_cuda, _on, _written

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "gelu": 2}


def _matrix(name: str, t: torch.Tensor, rows: int, cols: int, device: int) -> tuple:
    """(address, row stride) of a bf16 [rows, cols] matrix on that device."""
    if isinstance(t, torch.Tensor) and t.shape == (rows, cols) and t.dtype == torch.bfloat16 and t.get_device() == device:
        stride, unit = t.stride()
        if unit == 1 or cols <= 1:
            return t.data_ptr(), stride if rows > 1 else cols
    _check_cuda(name, t)
    if t.dtype != torch.bfloat16:
        raise Failure("dtype", f"{name} must be bfloat16", _lib.ERR_DTYPE)
    if t.shape != (rows, cols):
        raise Failure.shape(name, t.shape, f"[{rows}, {cols}]")
    if t.get_device() != device:
        raise Failure("arg", f"{name} is on {t.device}, the tokens on cuda:{device}", _lib.ERR_ARG)
    raise Failure("align", f"{name} must have a unit stride along its last dim", _lib.ERR_ALIGN)


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
        return like.new_empty(shape) if like.dtype == torch.bfloat16 else like.new_empty(shape, dtype=torch.bfloat16)
    _check_cuda(name, t)
    if t.shape != tuple(shape):
        raise Failure.shape(name, t.shape, str(list(shape)))
    return t


def _pack(packer, *args) -> bytes:
    try:
        return packer.pack(*args)
    except _lib.PACK_ERRORS as e:
        raise Failure("arg", f"a size that the call cannot take: {e}", _lib.ERR_ARG) from None


def _planes(n: int, m: int, inner: int, like: torch.Tensor) -> torch.Tensor:
    """A workspace of n bf16 [m, inner] planes, each rounded up to 256 bytes, as ltxattn_gated_ffn_workspace counts
    them (asking it would take another packing of the arguments).  ``like`` is bf16."""
    return like.new_empty(n * ((2 * m * inner + 255) // 256 * 128))


def _out_rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """The same for an output, of which a copy is no use."""
    rows = _rows(name, t)
    if rows.numel() and rows.data_ptr() != t.data_ptr():
        raise Failure("align", f"{name}'s leading dims must collapse into rows of one stride", _lib.ERR_ALIGN)
    return rows


def _gradient(name: str, t: Optional[torch.Tensor], of: Optional[torch.Tensor], like: torch.Tensor, shape, rows: int,
              cols: int, device: int):
    """The caller's output, or a new one, and its (address, row stride)."""
    if t is None:
        if of is not None and of.shape == shape and of.is_contiguous() and of.dtype == torch.bfloat16 and \
                of.get_device() == device:
            t = torch.empty_like(of)
        else:
            t = _output(name, None, shape, like)
        return t, (t.data_ptr(), cols)
    return t, _matrix(name, _out_rows(name, _output(name, t, shape, like)), rows, cols, device)


def _first_dim(name: str, w: torch.Tensor) -> int:
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise Failure.shape(name, getattr(w, "shape", ()), "a matrix")
    return w.shape[0]


def gated_ffn_plan(m: int, hidden: int, inner: int, out: int) -> dict:
    """How the block's products are made at these sizes: for "inner", "out", "dinner" and "dx" a
    ``(kernel, columns, cluster)`` (``ltxattn_gated_ffn_plan``; kernel 1 is the one for many tokens)."""
    for n in (m, hidden, inner, out):
        if not -2 ** 31 <= operator.index(n) < 2 ** 31:  # the C call's arguments would wrap
            raise Failure("shape", f"{n} is no 32-bit size", _lib.ERR_SHAPE)
    info = _lib.GatedFfnPlanInfo()
    rc = _lib.load().ltxattn_gated_ffn_plan(m, hidden, inner, out, info)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    return {n: (p.kernel, p.columns, p.cluster) for n, p in ((n, getattr(info, n)) for n, _ in info._fields_)}


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu", save: bool = False, out: Optional[torch.Tensor] = None, stream=None):
    """x [..., hidden] -> [..., out]; w_gate and w_up [inner, hidden], w_down [out, inner] (the
    checkpoint's [out, in] layout).

    ``activation`` is "silu", "gelu_tanh" or "gelu" (erf).  With ``save`` the result
    is ``(y, gate, up)``, the last two being what ``gated_ffn_backward`` needs:
    ``x w_gate^T`` and ``x w_up^T``, [..., inner].  hidden, inner and out are
    multiples of 8 and rows 16-byte aligned.  Results carry no graph.
    """
    act = _activation(activation)
    _check_cuda("x", x)
    if x.dim() < 1:
        raise Failure.shape("x", x.shape, "[..., hidden]")
    device = x.get_device()
    inner, out_dim = _first_dim("w_gate", w_gate), _first_dim("w_down", w_down)
    lead = x.shape[:-1]
    with _on(device, stream) as st:
        x2 = _rows("x", x)
        m, hidden = x2.shape
        y = torch.empty_like(x) if out is None and out_dim == hidden and x.is_contiguous() else \
            _output("out", out, lead + (out_dim,), x)
        gate = up = None
        kept = (0, 0, 0, 0)
        if save:
            gate = _output("gate", None, lead + (inner,), x)
            up = torch.empty_like(gate)
            kept = (gate.data_ptr(), inner, up.data_ptr(), inner)
        args = (_lib.BF16, act, m, hidden, inner, out_dim, *_matrix("x", x2, m, hidden, device),
                *_matrix("w_gate", w_gate, inner, hidden, device), *_matrix("w_up", w_up, inner, hidden, device),
                *_matrix("w_down", w_down, out_dim, inner, device),
                *((y.data_ptr(), out_dim) if out is None else _matrix("out", _out_rows("out", y), m, out_dim, device)),
                *kept)
        ws = _planes(1, m, inner, x)
        rc = _lib.load().ltxattn_gated_ffn(_pack(_lib.GATED_FFN_ARGS, *args, ws.data_ptr(), 2 * ws.numel()), st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    if out is not None:
        _written([out])
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
    The ``d...`` arguments give outputs to be written (overwritten, not added to); one
    of a gradient that is not needed is refused.
    """
    act = _activation(activation)
    for name, t, needed in (("dx", dx, need_dx), ("dw_gate", dw_gate, need_dw), ("dw_up", dw_up, need_dw),
                            ("dw_down", dw_down, need_dw)):
        if t is not None and not needed:
            raise Failure("arg", f"{name} is given, but not needed", _lib.ERR_ARG)
    if x is None and need_dw:
        raise Failure("missing", "x is needed for the gradients of w_gate and w_up")
    _check_cuda("dout", dout)
    if dout.dim() < 1:
        raise Failure.shape("dout", dout.shape, "[..., out]")
    device = dout.get_device()
    inner = _first_dim("w_gate", w_gate)
    hidden = w_gate.shape[1]
    lead = dout.shape[:-1]
    if len(lead) != 1:  # a matrix is checked as such below
        for name, t, cols in (("x", x, hidden), ("gate", gate, inner), ("up", up, inner)):
            if t is not None or name != "x":
                _check_cuda(name, t)
                if t.shape != lead + (cols,):
                    raise Failure.shape(name, t.shape, str(list(lead) + [cols]))
    given = [t for t in (dx, dw_gate, dw_up, dw_down) if t is not None]
    with _on(device, stream) as st:
        if len(lead) == 1:
            d2, x2, gate2, up2 = dout, x, gate, up
        else:
            d2, gate2, up2 = _rows("dout", dout), _rows("gate", gate), _rows("up", up)
            x2 = None if x is None else _rows("x", x)
        m, out_dim = d2.shape
        nothing = (0, 0)
        to = [nothing] * 4
        if need_dx:
            dx, to[0] = _gradient("dx", dx, x, dout, lead + (hidden,), m, hidden, device)
        if need_dw:
            dw_gate, to[1] = _gradient("dw_gate", dw_gate, w_gate, dout, (inner, hidden), inner, hidden, device)
            dw_up, to[2] = _gradient("dw_up", dw_up, w_up, dout, (inner, hidden), inner, hidden, device)
            dw_down, to[3] = _gradient("dw_down", dw_down, w_down, dout, (out_dim, inner), out_dim, inner, device)
        ws = _planes(3, m, inner, dout)
        rc = _lib.load().ltxattn_gated_ffn_bwd(
            _pack(
                _lib.GATED_FFN_BWD_ARGS, _lib.BF16, act, m, hidden, inner, out_dim,
                *(nothing if x is None else _matrix("x", x2, m, hidden, device)),
                *_matrix("w_gate", w_gate, inner, hidden, device), *_matrix("w_up", w_up, inner, hidden, device),
                *_matrix("w_down", w_down, out_dim, inner, device), *_matrix("gate", gate2, m, inner, device),
                *_matrix("up", up2, m, inner, device), *_matrix("dout", d2, m, out_dim, device), *to[0], *to[1],
                *to[2], *to[3], ws.data_ptr(), 2 * ws.numel()), st)
    if rc != _lib.OK:
        raise Failure.from_status(rc)
    if given:
        _written(given)
    return (dx if need_dx else None,) + ((dw_gate, dw_up, dw_down) if need_dw else (None, None, None))
