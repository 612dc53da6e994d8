"""The entry points of a wider network's operators, bound onto HiveGpuExtension:

    ext.gated_linear                               act(x Wg^T + bg) * (x Wu^T + bu), for inference
    ext.gated_linear_forward / _backward           the same for training, and its gradients
    ext.orthogonalize                              the Newton-Schulz iteration of a matrix or a batch of them
    ext.prepare_muon(params).step(grads, ...)      one step of many matrices by their orthogonalised momentum
    ext.sample_actions                             a slot of each row of logits: temperature, top-k, top-p, min-p

They take float32, float16 or bfloat16 tensors, sum in float32, run on
torch.cuda.current_stream() without synchronising it, and raise ValueError for
what they do not serve before anything is launched.  training.py builds
autograd functions and an optimizer on them.
"""
from __future__ import annotations

import bisect
import ctypes
import numbers

import torch

from .training_ops import (TYPES, _bytes, _calls, _check, _current_device, _float_tensor, _place, _raw_stream, _rows,
                           _vector)

_c_void_p = ctypes.c_void_p
_c_i64 = ctypes.c_int64
_c_int = ctypes.c_int
_c_float = ctypes.c_float
_c_double = ctypes.c_double

ACTIVATIONS = {"sigmoid": 0, "silu": 1, "gelu": 2}  # HG_SIGMOID, HG_SILU, HG_GELU
MAX_ROWS, MAX_COLS = 1 << 20, 1 << 19
MAX_AREA = 1 << 35  # of each two of a gated block's rows, columns and hidden units
MAX_WIDTH = 1 << 20  # slots of a row that a slot is drawn from
MAX_DRAWS, HELD, MAX_LONG_DRAWS = 1 << 25, 1024, 1 << 21  # rows, and rows of more slots than a wave holds
MAX_SIDE = 1 << 17  # of a matrix that is orthogonalised
MAX_MATRICES, MAX_PIECES = 1 << 16, 2049 ** 2  # of a batch: matrices, pieces of 64 x 64 of them
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # five steps: singular values from 0.0015 up end in 0.67 .. 1.21

SIGS = {
    "hg_gated_forward": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64, _c_void_p, _c_void_p,
                         _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p],
    "hg_gated_backward": [_c_void_p, _c_i64, _c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64,
                          _c_void_p, _c_void_p, _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                          _c_void_p, _c_void_p],
    "hg_gated_tiles": [_c_int, _c_i64, _c_i64, _c_i64, _c_void_p],
    "hg_orthogonalize": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_i64, _c_i64, _c_int, _c_void_p, _c_int, _c_float,
                         _c_void_p, _c_void_p, _c_void_p],
    "hg_orthogonalize_tiles": [_c_i64, _c_i64, _c_i64, _c_void_p],
    "hg_muon_step": [_c_void_p, _c_i64, _c_int, _c_int, _c_double, _c_double, _c_int, _c_double, _c_int, _c_void_p,
                     _c_int, _c_float, _c_void_p, _c_void_p],
    "hg_sample_actions": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_void_p, _c_double,
                          _c_void_p, _c_i64, _c_void_p, _c_double, _c_void_p, _c_double, _c_void_p, _c_void_p,
                          _c_void_p],
}
SIGS_I64 = {
    "hg_orthogonalize_workspace": [_c_i64, _c_i64, _c_i64],
    "hg_muon_step_workspace": [_c_void_p, _c_i64],
    "hg_gated_forward_workspace": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_i64],
    "hg_gated_backward_workspace": [_c_int, _c_i64, _c_i64, _c_i64],
}


def bind(lib) -> None:
    """Gives train_calls.cpp the library's function (training_ops.bind comes first)."""
    if _calls is not None:
        _calls.bind_network(ctypes.cast(lib.hg_sample_actions, _c_void_p).value)


def _number(value, name: str, whole: bool = False):
    """A float, or an int where it has to be whole; any kind of real number is taken (numpy's, too)."""
    if not isinstance(value, numbers.Integral if whole else numbers.Real):
        raise ValueError(f"{name} must be a {'whole ' if whole else ''}number, got {value!r}")
    try:
        return int(value) if whole else float(value)
    except OverflowError:
        raise ValueError(f"{name} is past a float's range") from None


def _activation(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _matrix(t, name: str, shape, like: torch.Tensor, dtype=None) -> int:
    """The address of a contiguous tensor on like's device, of its type or `dtype`."""
    dtype = dtype or like.dtype
    if not isinstance(t, torch.Tensor) or t.device != like.device:
        raise ValueError(f"{name} must be a tensor on {like.device}")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
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
    if max(rows * cols, rows * hidden, hidden * cols) > MAX_AREA:
        raise ValueError(f"rows, columns and hidden units at most {MAX_AREA} each two of them, got {rows}, {cols}, {hidden}")
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
    gate, up = (x.new_empty(shape, dtype=torch.float32) for _ in range(2)) if keep else (None, None)
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
    """(h, gate, up): gated_linear and the two products in float32 (to round
    them to 16 bits would be a third of the gradients' error), which
    gated_linear_backward takes."""
    return _gated_forward(self, x, w_gate, w_up, b_gate, b_up, activation, True)


def gated_linear_backward(self, dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                          gate: torch.Tensor, up: torch.Tensor, activation="silu", need_dx: bool = True,
                          need_weights: bool = True, need_bias: bool = True):
    """(dx, dw_gate, dw_up, db_gate, db_up): the gradients of gated_linear from
    dh, the gradient of h, with the forward pass's x, weights, gate, up and
    activation; None for what is not needed.  They have x's type and are
    contiguous; sums over rows are the same bits on every call.  The gradients of
    gate and up are rounded to x's type before they are multiplied, which makes
    those of 16-bit x and weights 1.35 to 1.4 times as far off as their own
    rounding does (float16's are scaled to its range for that)."""
    act = _activation(activation)
    dev, rows, cols, stride, hidden = _gated_sizes(x, w_gate, w_up)
    shape = (*x.shape[:-1], hidden)
    _place(dh, "dh")
    if tuple(dh.shape) != shape or dh.dtype != x.dtype:
        raise ValueError(f"dh must be {shape} {x.dtype}, got {tuple(dh.shape)} {dh.dtype}")
    dh_stride = _rows(dh, "dh")[2]
    g, u = _matrix(gate, "gate", shape, x, torch.float32), _matrix(up, "up", shape, x, torch.float32)
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


def _iteration(steps, coefficients, eps):
    """(steps, eps, coefficients as an array of float triples, how many): one triple for all steps, or one each."""
    steps, eps = _number(steps, "steps", whole=True), _number(eps, "eps")
    if not 1 <= steps <= 100:
        raise ValueError(f"steps must be 1 to 100, got {steps}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    try:
        triples = list(coefficients)
        if triples and isinstance(triples[0], numbers.Real):
            triples = [triples]
        triples = [[_number(v, "a coefficient") for v in t] for t in triples]
    except TypeError:
        triples = []
    if not triples or any(len(t) != 3 for t in triples):
        raise ValueError(f"coefficients must be (a, b, c) or a list of such, got {coefficients}")
    return steps, eps, (ctypes.c_float * (3 * len(triples)))(*[v for t in triples for v in t]), len(triples)


def orthogonalize(self, u: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """The Newton-Schulz iteration of each matrix of u [..., rows, cols]:
    from X = U / (|U| + eps), |U| the root of its sum of squares, `steps` times
    X <- a X + (b A + c A A) X with A = X X^T (X turned where U is taller than
    wide), which takes each singular value s to a s + b s^3 + c s^5; with the
    default coefficients all but the smallest end near 1.  coefficients:
    (a, b, c), or a list of them, one a step (the last serves those past it).

    u float32 / float16 / bfloat16, its rows contiguous, rows and matrices
    evenly spaced; the result has its shape and type and is contiguous.  Matrices
    are held in 22 bits a value between the products (or to within 2^-36 of their
    norm, where that is more), which are summed in float32; a, b and c may be such that X's entries stay below 7.9 in size and
    those of a I + b A + c A A below 63."""
    dev = _float_tensor(u, "u")
    if u.dim() < 2 or u.shape[-1] == 0 or u.shape[-2] == 0:
        raise ValueError(f"u must be [..., rows, cols], got {tuple(u.shape)}")
    rows, cols = u.shape[-2:]
    if rows > MAX_SIDE or cols > MAX_SIDE:
        raise ValueError(f"at most {MAX_SIDE} rows and columns, got {rows} and {cols}")
    count = u.numel() // (rows * cols)
    if count > MAX_MATRICES or count * (rows // 64 + 1) * (cols // 64 + 1) > MAX_PIECES:
        raise ValueError(f"at most {MAX_MATRICES} matrices and {MAX_PIECES} pieces of 64 x 64 of them a call, got {count} "
                         f"of {rows} x {cols}")
    steps, eps, c, triples = _iteration(steps, coefficients, eps)
    out = torch.empty_like(u, memory_format=torch.contiguous_format)
    if u.numel() == 0:
        return out
    if cols > 1 and u.stride(-1) != 1:
        raise ValueError("u's last dimension must be contiguous")
    try:
        batch = u.view(-1, rows, cols) if u.dim() != 3 else u
    except RuntimeError:
        raise ValueError("u's matrices must be evenly spaced") from None
    ws = u.new_empty((self._lib.hg_orthogonalize_workspace(count, rows, cols),), dtype=torch.uint8)
    _check(self._lib.hg_orthogonalize(u.data_ptr(), TYPES[u.dtype], count, rows, cols, batch.stride(1), batch.stride(0),
                                      steps, c, triples, eps, out.data_ptr(), ws.data_ptr(), _raw_stream(dev)),
           "orthogonalize")
    return out


class HgMuonMatrix(ctypes.Structure):
    """C layout of `hg_muon_matrix` (include/hive_gpu.h)."""

    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("momentum", ctypes.c_void_p),
                ("rows", ctypes.c_int64), ("cols", ctypes.c_int64), ("scale", ctypes.c_double)]


class MuonPlan:
    """hg_muon_step over a fixed list of matrices, checked and laid out once.

    `momentum` holds a float32 tensor of each matrix's shape.  The plan enters
    the parameters by address: updates in place are seen, a parameter whose
    memory is replaced needs a new plan.  Parameters and momenta that share
    memory are refused, and gradients that lie in them."""

    def __init__(self, lib, params, scale: str = "spectral", momentum=None):
        params = list(params)
        if not params:
            raise ValueError("prepare_muon needs at least one matrix")
        if scale not in ("spectral", "rms"):
            raise ValueError(f"scale must be 'spectral' or 'rms', got {scale!r}")
        for i, p in enumerate(params):
            _float_tensor(p, f"params[{i}]")
            if p.dtype != params[0].dtype:
                raise ValueError(f"params[{i}] is {p.dtype}, params[0] {params[0].dtype}: one plan serves one type")
            if p.dim() != 2 or p.numel() == 0 or max(p.shape) > MAX_SIDE:
                raise ValueError(f"params[{i}] must be a matrix of 1 to {MAX_SIDE} rows and columns, got {tuple(p.shape)}")
            if not p.is_contiguous():
                raise ValueError(f"params[{i}] must be contiguous")
        if momentum is None:
            momentum = [torch.zeros_like(p, dtype=torch.float32) for p in params]
        momentum = list(momentum)
        if len(momentum) != len(params):
            raise ValueError(f"{len(momentum)} momenta for {len(params)} matrices")
        for i, (m, p) in enumerate(zip(momentum, params)):
            if not isinstance(m, torch.Tensor) or m.device != p.device or m.dtype != torch.float32 or \
                    m.shape != p.shape or not m.is_contiguous():
                raise ValueError(f"momentum[{i}] must be a contiguous float32 tensor {tuple(p.shape)} on {p.device}")
        self._lib, self.params, self.momentum = lib, params, momentum
        held = sorted((*_bytes(t), f"{name}[{i}]") for name, ts in (("params", params), ("momentum", momentum))
                      for i, t in enumerate(ts))
        for (_, end, a), (begin, _, b) in zip(held, held[1:]):
            if begin < end:
                raise ValueError(f"{a} and {b} share memory: a step writes both")
        self._written = [x for begin, end, _ in held for x in (begin, end)]
        self._ptrs = [p.data_ptr() for p in params]
        self._table = (HgMuonMatrix * len(params))()
        for t, p, m in zip(self._table, params, momentum):
            rows, cols = p.shape
            t.param, t.momentum, t.rows, t.cols = p.data_ptr(), m.data_ptr(), rows, cols
            t.scale = max(1.0, rows / cols) ** 0.5 if scale == "spectral" else 0.2 * max(rows, cols) ** 0.5
        self._need = lib.hg_muon_step_workspace(self._table, len(params))
        self._type = TYPES[params[0].dtype]
        self._device = params[0].get_device()

    def _apart(self, t: torch.Tensor) -> bool:
        """Whether a step writes nothing of t."""
        begin, end = _bytes(t)
        i = bisect.bisect_right(self._written, begin)
        return i % 2 == 0 and (i == len(self._written) or self._written[i] >= end)

    def step(self, grads, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
             steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> None:
        """m = momentum m + g; u = g + momentum m (nesterov) or m; p = p (1 - lr
        weight_decay) - lr scale orthogonalize(u), of every matrix, in place.
        scale: sqrt(max(1, rows / cols)) of a "spectral" plan, 0.2 sqrt(max(rows,
        cols)) of an "rms" one.  grads: one type, contiguous, the parameters'
        shapes; None leaves its matrix and momentum as they are.  The stepped
        parameters' versions rise."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        for i, g in enumerate(grads):
            if g is not None and (not isinstance(g, torch.Tensor) or g.layout is not torch.strided):
                raise ValueError(f"the gradient of params[{i}] must be a dense tensor or None, got {type(g).__name__}")
        steps, eps, c, triples = _iteration(steps, coefficients, eps)
        lr, momentum, weight_decay = (_number(v, name) for v, name in (
            (lr, "lr"), (momentum, "momentum"), (weight_decay, "weight_decay")))
        kind = next((g.dtype for g in grads if g is not None), torch.float32)
        if kind not in TYPES:
            raise ValueError(f"gradients must be float32, float16 or bfloat16, got {kind}")
        if self._device != _current_device():
            raise ValueError(f"the parameters are on device {self._device}, the current one is {_current_device()}")
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if p.data_ptr() != self._ptrs[i]:
                raise ValueError("a parameter's memory was replaced: make a new plan")
            if g is None:
                continue
            if g.dtype is not kind or g.shape != p.shape or g.device != p.device or not g.is_contiguous():
                raise ValueError(f"a gradient must be a contiguous {kind} tensor {tuple(p.shape)} on {p.device}, got "
                                 f"{g.dtype} {tuple(g.shape)} on {g.device}")
            if not self._apart(g):
                raise ValueError(f"the gradient of params[{i}] shares memory with a parameter or momentum")
        for t, g in zip(self._table, grads):
            t.grad = None if g is None else g.data_ptr()
        ws = torch.empty((self._need,), dtype=torch.uint8, device=self.params[0].device)
        _check(self._lib.hg_muon_step(self._table, len(grads), self._type, TYPES[kind], lr, momentum, int(nesterov),
                                      weight_decay, steps, c, triples, eps, ws.data_ptr(), _raw_stream(self._device)),
               "muon_step")
        for p, m, g in zip(self.params, self.momentum, grads):
            if g is not None:
                for t in (p, m):
                    if not t.is_inference():
                        torch.autograd.graph.increment_version(t)


def prepare_muon(self, params, scale: str = "spectral", momentum=None) -> MuonPlan:
    """A MuonPlan of contiguous matrices of one type.  `momentum`: those of an
    earlier plan over matrices of the same shapes (a checkpoint), taken as they
    are, not copied; None: zeros."""
    return MuonPlan(self._lib, params, scale, momentum)


def _setting(value, name: str, B: int, dtype: torch.dtype, dev: int):
    """(address or None, number) of a setting: a tensor of one value a row, or a number for all."""
    if isinstance(value, torch.Tensor):
        return _vector(value, name, B, dtype, dev), 0
    return None, _number(value, f"{name}, where it is no tensor of one a row,", whole=dtype is torch.int64)


def sample_actions(self, logits: torch.Tensor, uniforms: torch.Tensor, num_actions=None, temperature=1.0, top_k=0,
                   top_p=1.0, min_p=0.0):
    """(actions int64 [B], log_probs float32 [B]): a slot of each row of logits
    [B, width], drawn from uniforms [B] (float32 in [0, 1)), and the logarithm of
    its probability among the slots kept.

    logits: float32 / float16 / bfloat16, rows contiguous and evenly spaced.
    num_actions [B] int64: a row's slots are its first ones, as the legal lists'
    (clamped to [0, width]; None: all); slots of -inf or NaN are left out.  No
    slot left: -1, and a log probability of 0.  Kept, in order of falling logits
    (ties by rising slots): the first top_k (0: all); of these the fewest first
    ones that hold top_p of their mass; of these the ones at least min_p as
    likely as the first.  The slot drawn is the first, in order of the slots, at
    which the running sum of exp((x - max) / temperature) passes u times the
    whole; a temperature of 0 takes the largest logit's first slot.  Each
    setting is a number, or a tensor of a value a row (float32; top_k int64; what
    lies past its range counts as its end; NaN as a temperature of 0, a top_p of 1,
    a min_p or uniform number of 0)."""
    if _calls is not None:
        done = _calls.sample_actions(logits, uniforms, num_actions, temperature, top_k, top_p, min_p)
        if done is not None:
            return done
    dev = _float_tensor(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [B, width], got {tuple(logits.shape)}")
    B, width, stride = _rows(logits, "logits")
    if width > MAX_WIDTH:
        raise ValueError(f"rows of at most {MAX_WIDTH} slots, got {width}")
    if B > (MAX_DRAWS if width <= HELD else MAX_LONG_DRAWS):
        raise ValueError(f"at most {MAX_DRAWS} rows, {MAX_LONG_DRAWS} of more than {HELD} slots, got {B} of {width}")
    u = _vector(uniforms, "uniforms", B, torch.float32, dev)
    n = None if num_actions is None else _vector(num_actions, "num_actions", B, torch.int64, dev)
    t, t_all = _setting(temperature, "temperature", B, torch.float32, dev)
    k, k_all = _setting(top_k, "top_k", B, torch.int64, dev)
    p, p_all = _setting(top_p, "top_p", B, torch.float32, dev)
    m, m_all = _setting(min_p, "min_p", B, torch.float32, dev)
    if not t_all >= 0.0 or k_all < 0 or not 0.0 <= p_all or not 0.0 <= m_all <= 1.0:
        raise ValueError(f"temperature, top_k and top_p must not be negative and min_p be in [0, 1], got {t_all}, {k_all}, "
                         f"{p_all} and {m_all}")
    actions = logits.new_empty((B,), dtype=torch.int64)
    log_probs = logits.new_empty((B,), dtype=torch.float32)
    _check(self._lib.hg_sample_actions(logits.data_ptr(), TYPES[logits.dtype], B, width, stride, n, u, t, t_all, k,
                                       min(k_all, width), p, p_all, m, m_all, actions.data_ptr(), log_probs.data_ptr(),
                                       _raw_stream(dev)),
           "sample_actions")
    return actions, log_probs


METHODS = (gated_linear, gated_linear_forward, gated_linear_backward, orthogonalize, prepare_muon, sample_actions)
