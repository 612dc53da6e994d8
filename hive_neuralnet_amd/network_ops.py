"""The entry points of a wider network's operators, bound onto HiveGpuExtension:

    ext.gated_linear                               act(x Wg^T + bg) * (x Wu^T + bu), for inference
    ext.gated_linear_forward / _backward           the same for training, and its gradients

They take float32, float16 or bfloat16 tensors, sum in float32, run on
torch.cuda.current_stream() without synchronising it, and raise ValueError for
what they do not serve before anything is launched.  training.py builds
autograd functions and an optimizer on them.
"""
from __future__ import annotations

import ctypes

import torch

from .training_ops import TYPES, _check, _float_tensor, _place, _raw_stream, _rows, _vector

_c_void_p = ctypes.c_void_p
_c_i64 = ctypes.c_int64
_c_int = ctypes.c_int

ACTIVATIONS = {"sigmoid": 0, "silu": 1, "gelu": 2}  # HG_SIGMOID, HG_SILU, HG_GELU
MAX_ROWS, MAX_COLS = 1 << 20, 1 << 19

SIGS = {
    "hg_gated_forward": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64, _c_void_p, _c_void_p,
                         _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p],
    "hg_gated_backward": [_c_void_p, _c_i64, _c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64,
                          _c_void_p, _c_void_p, _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                          _c_void_p, _c_void_p],
}
SIGS_I64 = {
    "hg_gated_forward_workspace": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64],
    "hg_gated_backward_workspace": [_c_int, _c_i64, _c_i64, _c_i64],
}


def _activation(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _matrix(t, name: str, shape, like: torch.Tensor) -> int:
    """The address of a contiguous tensor of like's type and device."""
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise ValueError(f"{name} must be a tensor on {like.device}")
    if t.dtype != like.dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)} {like.dtype}, got {tuple(t.shape)} {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _gated_sizes(x, w_gate, w_up):
    """(device, rows, cols, row stride, hidden) of x and the two weights."""
    dev = _float_tensor(x, "x")
    rows, cols, stride = _rows(x, "x")
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2 or w_gate.shape[0] == 0:
        raise ValueError("w_gate must be [hidden, cols]")
    hidden = w_gate.shape[0]
    for w, name in ((w_gate, "w_gate"), (w_up, "w_up")):
        _matrix(w, name, (hidden, cols), x)
    if rows > MAX_ROWS or cols > MAX_COLS or hidden > MAX_COLS:
        raise ValueError(f"at most {MAX_ROWS} rows, {MAX_COLS} columns and hidden units, got {rows}, {cols}, {hidden}")
    if stride < 0:
        raise ValueError("x's rows must be in order")
    return dev, rows, cols, stride, hidden


def _gated_forward(self, x, w_gate, w_up, b_gate, b_up, activation, keep: bool):
    act = _activation(activation)
    dev, rows, cols, stride, hidden = _gated_sizes(x, w_gate, w_up)
    bg = None if b_gate is None else _vector(b_gate, "b_gate", hidden, x.dtype, dev)
    bu = None if b_up is None else _vector(b_up, "b_up", hidden, x.dtype, dev)
    shape, kind = (*x.shape[:-1], hidden), TYPES[x.dtype]
    h = x.new_empty(shape)
    gate, up = (x.new_empty(shape), x.new_empty(shape)) if keep else (None, None)
    need = self._lib.hg_gated_forward_workspace(x.data_ptr(), kind, rows, cols, stride, w_gate.data_ptr(),
                                                w_up.data_ptr(), hidden)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    _check(self._lib.hg_gated_forward(
        x.data_ptr(), kind, rows, cols, stride, w_gate.data_ptr(), w_up.data_ptr(), hidden, bg, bu, act, h.data_ptr(),
        gate.data_ptr() if keep else None, up.data_ptr() if keep else None, None if ws is None else ws.data_ptr(),
        _raw_stream(dev)), "gated_linear_forward")
    return h, gate, up


def gated_linear(self, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate=None, b_up=None,
                 activation="silu") -> torch.Tensor:
    """h [..., hidden] = act(x w_gate^T + b_gate) * (x w_up^T + b_up), both
    products, the activation and the product of the two in one kernel.

    x [..., cols] float32 / float16 / bfloat16, its rows contiguous and evenly
    spaced; w_gate, w_up [hidden, cols] contiguous, b_gate, b_up [hidden] or
    None, all of x's type.  activation: "sigmoid", "silu" (g sigmoid(g)) or
    "gelu" (of the error function).  float32 values are multiplied in 24 bits.
    x, weights or rows that 16-byte loads cannot take (odd widths, strides or
    addresses) and float32 are laid out in a workspace first."""
    return _gated_forward(self, x, w_gate, w_up, b_gate, b_up, activation, False)[0]


def gated_linear_forward(self, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate=None, b_up=None,
                         activation="silu"):
    """(h, gate, up): gated_linear and the two products, rounded to x's type,
    which gated_linear_backward takes."""
    return _gated_forward(self, x, w_gate, w_up, b_gate, b_up, activation, True)


def gated_linear_backward(self, dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                          gate: torch.Tensor, up: torch.Tensor, activation="silu", need_dx: bool = True,
                          need_weights: bool = True, need_bias: bool = True):
    """(dx, dw_gate, dw_up, db_gate, db_up): the gradients of gated_linear from
    dh, the gradient of h, with the forward pass's x, weights, gate, up and
    activation; None for what is not needed.  They have x's type and are
    contiguous; sums over rows are the same bits on every call.  The gradients of
    gate and up are rounded to x's type before they are multiplied, as gate
    and up were."""
    act = _activation(activation)
    dev, rows, cols, stride, hidden = _gated_sizes(x, w_gate, w_up)
    shape = (*x.shape[:-1], hidden)
    _place(dh, "dh")
    if tuple(dh.shape) != shape or dh.dtype != x.dtype:
        raise ValueError(f"dh must be {shape} {x.dtype}, got {tuple(dh.shape)} {dh.dtype}")
    dh_stride = _rows(dh, "dh")[2]
    g, u = _matrix(gate, "gate", shape, x), _matrix(up, "up", shape, x)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_dx else None
    dw = (torch.empty_like(w_gate), torch.empty_like(w_up)) if need_weights else (None, None)
    db = (x.new_empty((hidden,)), x.new_empty((hidden,))) if need_bias else (None, None)
    kind = TYPES[x.dtype]
    ws = x.new_empty((self._lib.hg_gated_backward_workspace(kind, rows, cols, hidden),), dtype=torch.uint8)
    _check(self._lib.hg_gated_backward(
        dh.data_ptr(), dh_stride, x.data_ptr(), kind, rows, cols, stride, w_gate.data_ptr(), w_up.data_ptr(), hidden, g,
        u, act, *[None if t is None else t.data_ptr() for t in (dx, *dw, *db)], ws.data_ptr(), _raw_stream(dev)),
        "gated_linear_backward")
    return dx, *dw, *db


METHODS = (gated_linear, gated_linear_forward, gated_linear_backward)
