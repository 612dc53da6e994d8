"""The training operators' entry points, bound onto HiveGpuExtension:

    ext.layer_norm_forward / layer_norm_backward   layer norm (of x or sigmoid(x)) and its gradients
    ext.policy_value_loss                          the loss of a batch of positions and its gradient
    ext.prepare_adamw(params).step(grads, ...)     one AdamW step of many tensors, moments in 32 or 8 bits

They work in float32 inside, on float32, float16 or bfloat16 tensors, on
torch.cuda.current_stream() without synchronising it, and raise ValueError
for what they do not serve before anything is launched (RuntimeError for sizes
past a launch's bounds, which include/hive_gpu.h names).  training.py builds
autograd functions, an optimizer and a training step of HiveFNN on them.
"""
from __future__ import annotations

import bisect
import ctypes

import numpy as np
import torch

try:  # train_calls.cpp: these entry points without Python's share of a call
    from . import _train_calls as _calls
except ImportError:  # the library built by itself: all of a call from here, twice the time of a small one
    _calls = None

_c_void_p = ctypes.c_void_p
_c_i64 = ctypes.c_int64
_c_int = ctypes.c_int
_c_float = ctypes.c_float
_c_double = ctypes.c_double

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # HG_F32, HG_F16, HG_BF16
ADAMW_BLOCK = 256  # HG_ADAMW_BLOCK: elements under one scale of 8-bit moments

SIGS = {
    "hg_layer_norm_forward": [_c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p, _c_int, _c_float,
                              _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p],
    "hg_layer_norm_backward": [_c_void_p, _c_i64, _c_void_p, _c_int, _c_i64, _c_i64, _c_i64, _c_void_p, _c_void_p,
                               _c_void_p, _c_int, _c_int, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p],
    "hg_policy_value_loss": [_c_void_p, _c_int, _c_i64, _c_void_p, _c_void_p, _c_void_p, _c_int, _c_i64, _c_void_p,
                             _c_void_p, _c_void_p, _c_i64, _c_float, _c_float, _c_void_p, _c_void_p, _c_void_p,
                             _c_void_p, _c_void_p],
    "hg_adamw_step": [_c_void_p, _c_i64, _c_int, _c_int, _c_int, _c_i64, _c_double, _c_double, _c_double, _c_double,
                      _c_double, _c_void_p, ctypes.c_uint32, _c_void_p],
}
SIGS_I64 = {
    "hg_layer_norm_backward_workspace": [_c_i64, _c_i64],
    "hg_policy_value_loss_workspace": [_c_i64, _c_i64],
}


def bind(lib) -> None:
    """Gives train_calls.cpp the library's functions."""
    if _calls is not None:
        _calls.bind(*[ctypes.cast(getattr(lib, name), _c_void_p).value for name in (
            "hg_layer_norm_forward", "hg_layer_norm_backward", "hg_layer_norm_backward_workspace",
            "hg_policy_value_loss", "hg_policy_value_loss_workspace", "hg_adamw_step")], _current_device, _raw_stream)


class HgAdamwTensor(ctypes.Structure):
    """C layout of `hg_adamw_tensor` (include/hive_gpu.h)."""

    _fields_ = [(name, ctypes.c_void_p) for name in (
        "param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")] + [
        ("count", ctypes.c_int64), ("place", ctypes.c_int64)]


# the current stream's handle without a Stream object around it (2.8 us of a call's 10)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _check(err: int, what: str) -> None:
    if err != 0:
        raise RuntimeError(f"{what}: HIP error {err}")


_current_device = torch._C._cuda_getDevice


def _place(t, name: str) -> int:
    """The device of a GPU tensor on the current device."""
    if isinstance(t, torch.Tensor) and t.is_cuda:
        dev = t.get_device()
        if dev == _current_device():
            return dev
        raise ValueError(f"{name} is on {t.device}, the current device is {_current_device()}")
    raise ValueError(f"{name} must be a GPU tensor")


def _float_tensor(t, name: str) -> int:
    dev = _place(t, name)
    if t.dtype not in TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return dev


def _vector(t, name: str, n: int, dtype: torch.dtype, dev: int) -> int:
    """The address of a contiguous tensor of n elements, [n] or [n, 1], on `dev`."""
    if not isinstance(t, torch.Tensor) or t.get_device() != dev:
        raise ValueError(f"{name} must be a GPU tensor on device {dev}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != (n,) and t.shape != (n, 1):
        raise ValueError(f"{name} must have shape ({n},) or ({n}, 1), got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str):
    """(rows, cols, row stride) of a tensor whose last dimension is contiguous
    and whose other dimensions are evenly spaced rows."""
    shape = t.shape
    if len(shape) == 0:
        raise ValueError(f"{name} must have at least one dimension")
    cols = shape[-1]
    if cols == 0:
        raise ValueError(f"{name} must have at least one column")
    if t.is_contiguous():
        return t.numel() // cols, cols, cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if len(shape) == 2:
        return shape[0], cols, t.stride(0)
    try:
        v = t.view(-1, cols)
    except RuntimeError:
        raise ValueError(f"{name}'s rows must be evenly spaced") from None
    return v.shape[0], cols, v.stride(0)


def _activation(activation) -> int:
    if activation is None:
        return 0
    if activation != "sigmoid":
        raise ValueError(f"activation must be None or 'sigmoid', got {activation!r}")
    return 1


def _norm_params(weight, bias, cols: int, dev: int):
    """(weight pointer, bias pointer, type): one type for both."""
    w = b = None
    kind = torch.float32
    if weight is not None:
        kind = weight.dtype
        w = _vector(weight, "weight", cols, kind, dev)
    if bias is not None:
        if weight is not None and bias.dtype != kind:
            raise ValueError(f"weight and bias must have one type, got {kind} and {bias.dtype}")
        kind = bias.dtype
        b = _vector(bias, "bias", cols, kind, dev)
    if kind not in TYPES:
        raise ValueError(f"weight and bias must be float32, float16 or bfloat16, got {kind}")
    return w, b, TYPES[kind]


def layer_norm_forward(self, x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, activation=None):
    """(y, mean, rstd): layer norm over the last dimension of x, or of
    sigmoid(x) with activation="sigmoid" (HiveFNN's encoder,
    fnn_network.py:175-187).  x [..., cols] float32 / float16 / bfloat16, its
    rows contiguous and evenly spaced (a slice of a wider tensor's columns
    is); weight, bias [cols] of one type, or None; y has x's shape and type
    and is contiguous, mean and rstd = 1 / sqrt(var + eps) are float32
    [...]."""
    if _calls is not None:
        done = _calls.layer_norm_forward(x, weight, bias, eps, activation)
        if done is not None:
            return done
    dev = _float_tensor(x, "x")
    rows, cols, stride = _rows(x, "x")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    sigmoid = _activation(activation)
    w, b, kind = _norm_params(weight, bias, cols, dev)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean, rstd = x.new_empty((2, *x.shape[:-1]), dtype=torch.float32).unbind(0)
    _check(self._lib.hg_layer_norm_forward(x.data_ptr(), TYPES[x.dtype], rows, cols, stride, w, b, kind, eps, sigmoid,
                                           y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _raw_stream(dev)),
           "layer_norm_forward")
    return y, mean, rstd


def layer_norm_backward(self, dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight=None,
                        bias=None, activation=None, need_dx: bool = True):
    """(dx, dweight, dbias): the gradients of layer_norm_forward from dy, the
    gradient of y, with the forward pass's x, mean, rstd, weight and
    activation.  dweight and dbias (of the parameters' type; None for a
    parameter that is None) are sums over all rows, the same bits on every
    call; dx (x's shape and type, contiguous; None with need_dx=False)."""
    if _calls is not None:
        done = _calls.layer_norm_backward(dy, x, mean, rstd, weight, bias, activation, need_dx)
        if done is not None:
            return done
    dev = _float_tensor(x, "x")
    _place(dy, "dy")
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {tuple(x.shape)} {x.dtype}, got {tuple(dy.shape)} {dy.dtype}")
    rows, cols, stride = _rows(x, "x")
    dy_stride = _rows(dy, "dy")[2]
    sigmoid = _activation(activation)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != dev or t.dtype != torch.float32 or \
                t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be the forward pass's: {rows} float32 values on {x.device}")
    w, b, kind = _norm_params(weight, bias, cols, dev)
    dx = dw = db = ws = None
    if need_dx:
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    if w is not None:
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
    if b is not None:
        db = torch.empty_like(bias, memory_format=torch.contiguous_format)
    if dw is not None or db is not None:
        ws = x.new_empty((self._lib.hg_layer_norm_backward_workspace(rows, cols),), dtype=torch.uint8)
    _check(self._lib.hg_layer_norm_backward(
        dy.data_ptr(), dy_stride, x.data_ptr(), TYPES[x.dtype], rows, cols, stride, mean.data_ptr(), rstd.data_ptr(), w,
        kind, sigmoid, None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
        None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(), _raw_stream(dev)),
        "layer_norm_backward")
    return dx, dw, db


def policy_value_loss(self, logits: torch.Tensor, values: torch.Tensor, num_actions: torch.Tensor,
                      policy_targets: torch.Tensor, policy_weights: torch.Tensor, value_targets: torch.Tensor,
                      value_weights: torch.Tensor, value_coef: float = 1.0, loss_scale: float = 1.0):
    """(losses, dlogits, dvalues): the training loss of B positions and its
    gradient in one call.

    logits [N]: each position's logits over its legal moves, the positions
    one after the other (build_forward_batch's rows); num_actions [B] int64
    (clamped to [0, width], as there); policy_targets [B, width] (the slots
    past num_actions are not used); policy_weights, value_targets,
    value_weights float32 [B] or [B, 1], the weights not negative; values
    [B] or [B, 1] of the logits' type.
    losses is float32 [total, policy, value], total = policy + value_coef
    value: the weighted means of the cross-entropy and of the squared error.
    dlogits and dvalues are loss_scale times the gradients of the total.
    Positions of weight 0, without moves, or with no logit above -inf add
    nothing and have gradients of zero."""
    if _calls is not None:
        done = _calls.policy_value_loss(logits, values, num_actions, policy_targets, policy_weights, value_targets,
                                        value_weights, value_coef, loss_scale)
        if done is not None:
            return done
    dev = _float_tensor(logits, "logits")
    if logits.dim() != 1 or not logits.is_contiguous():
        raise ValueError(f"logits must be one contiguous row, got {tuple(logits.shape)}")
    _float_tensor(policy_targets, "policy_targets")
    if policy_targets.dim() != 2 or not policy_targets.is_contiguous():
        raise ValueError("policy_targets must be contiguous [B, width]")
    B, width = policy_targets.shape
    N = logits.shape[0]
    if B == 0 and N > 0:
        raise ValueError(f"{N} logits of no position")
    v = _vector(values, "values", B, logits.dtype, dev)
    n = _vector(num_actions, "num_actions", B, torch.int64, dev)
    pw = _vector(policy_weights, "policy_weights", B, torch.float32, dev)
    vt = _vector(value_targets, "value_targets", B, torch.float32, dev)
    vw = _vector(value_weights, "value_weights", B, torch.float32, dev)
    losses = logits.new_empty((3,), dtype=torch.float32)
    dlogits = torch.empty_like(logits)
    dvalues = torch.empty_like(values)
    ws = logits.new_empty((self._lib.hg_policy_value_loss_workspace(B, width),), dtype=torch.uint8)
    _check(self._lib.hg_policy_value_loss(
        logits.data_ptr(), TYPES[logits.dtype], N, v, n, policy_targets.data_ptr(), TYPES[policy_targets.dtype], width,
        pw, vt, vw, B, value_coef, loss_scale, losses.data_ptr(), dlogits.data_ptr(), dvalues.data_ptr(),
        ws.data_ptr(), _raw_stream(dev)), "policy_value_loss")
    return losses, dlogits, dvalues


def _bytes(t: torch.Tensor):
    """(first byte, one past the last) of a contiguous tensor."""
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class AdamWPlan:
    """hg_adamw_step over a fixed list of tensors, checked and laid out once.

    The moments of all tensors are flat arrays, each tensor's at a multiple
    of 256 elements (`places`): exp_avg and exp_avg_sq in float32, or with
    state_bits=8 as float8_e4m3fn codes with exp_avg_scale and
    exp_avg_sq_scale, a float32 per 256 elements; a code stands for code *
    scale, in exp_avg_sq for the square root of the moment.  The plan enters
    the parameters by address: updates in place are seen, a parameter whose
    memory is replaced needs a new plan.

    A step's blocks run beside each other, so nothing that it writes may be
    written or read through another of its tensors: parameters and moments
    that share memory, and gradients that lie in them, are refused (but a
    gradient that is its own parameter's memory, element for element)."""

    def __init__(self, lib, params, state_bits: int = 32, state=None):
        params = list(params)
        if not params:
            raise ValueError("prepare_adamw needs at least one parameter")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        for i, p in enumerate(params):
            _float_tensor(p, f"params[{i}]")
            if p.dtype != params[0].dtype:
                raise ValueError(f"params[{i}] is {p.dtype}, params[0] {params[0].dtype}: one plan serves one type")
            if not p.is_contiguous():
                raise ValueError(f"params[{i}] must be contiguous")
        self._lib, self.params, self.state_bits = lib, params, state_bits
        self._ptrs = [p.data_ptr() for p in params]
        self.places, total = [], 0
        for p in params:
            self.places.append(total)
            total += -(-p.numel() // ADAMW_BLOCK) * ADAMW_BLOCK
        self.total = total
        dev = params[0].device
        kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        want = {"exp_avg": (total, kind), "exp_avg_sq": (total, kind)}
        if state_bits == 8:
            want["exp_avg_scale"] = want["exp_avg_sq_scale"] = (total // ADAMW_BLOCK, torch.float32)
        if state is None:
            state = {k: torch.zeros((n,), dtype=t, device=dev) for k, (n, t) in want.items()}
        if set(state) != set(want):
            raise ValueError(f"the state must hold {sorted(want)}, got {sorted(state)}")
        for k, (n, t) in want.items():
            v = state[k]
            if not isinstance(v, torch.Tensor) or v.device != dev or v.dtype != t or tuple(v.shape) != (n,) or \
                    not v.is_contiguous():
                raise ValueError(f"{k} must be a contiguous {t} tensor of {n} values on {dev}")
            if v.data_ptr() % 4:
                raise ValueError(f"{k} must be 4-byte aligned: codes are read four at a time")
        self.state = {k: state[k] for k in want}
        named = [(f"params[{i}]", p) for i, p in enumerate(params)] + list(self.state.items())
        held = sorted((*_bytes(t), name) for name, t in named if t.numel())
        for (_, end, a), (begin, _, b) in zip(held, held[1:]):
            if begin < end:
                raise ValueError(f"{a} and {b} share memory: a step writes both at once")
        self._written = [x for begin, end, _ in held for x in (begin, end)]  # in order: inside one past an odd number
        self._written_table = np.array(self._written, dtype=np.uint64)
        self._table = np.zeros((len(params),), dtype=np.dtype(HgAdamwTensor))
        at = np.array(self.places, dtype=np.uint64)
        size = np.uint64(4 if state_bits == 32 else 1)
        self._table["param"] = self._ptrs
        for k in ("exp_avg", "exp_avg_sq"):
            self._table[k] = np.uint64(self.state[k].data_ptr()) + size * at
            if state_bits == 8:
                self._table[k + "_scale"] = np.uint64(self.state[k + "_scale"].data_ptr()) + \
                    np.uint64(4) * (at // np.uint64(ADAMW_BLOCK))
        self._counts = [p.numel() for p in params]
        self._table["count"] = self._counts
        self._partial = False  # whether the last step left a parameter out
        self._table["place"] = self.places
        self._shapes = [p.shape for p in params]
        self._grad, self._count = self._table["grad"], self._table["count"]
        self._table_ptr = self._table.ctypes.data
        self._written_ptr = self._written_table.ctypes.data
        self._type = TYPES[params[0].dtype]
        self._device = params[0].get_device()

    def _apart(self, t: torch.Tensor) -> bool:
        """Whether a step writes nothing of t."""
        begin, end = _bytes(t)
        i = bisect.bisect_right(self._written, begin)
        return begin == end or i % 2 == 0 and (i == len(self._written) or self._written[i] >= end)

    def step(self, grads, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
             weight_decay: float = 0.01, grad_scale: torch.Tensor | None = None, seed: int = 0) -> None:
        """Step number `step` (the first is 1) of every parameter, in place, from
        the list `grads` (one type, contiguous, the parameters' shapes; None
        leaves its parameter and moments as they are).  grad_scale: a float32
        tensor of one value that multiplies the gradients (1 / the loss scale, a
        clipping factor).  seed: of the 8-bit moments' rounding; give each step
        another one.  The stepped parameters' versions rise: autograd finds that
        a weight it saved has changed."""
        if _calls is not None and not self._partial and _calls.adamw_step(
                self.params, grads, self._table_ptr, self._type, self.state_bits, step, lr, betas[0], betas[1], eps,
                weight_decay, grad_scale, seed & 0xFFFFFFFF, self._written_ptr, len(self._written)):
            return
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        dev = self._device
        kind = next((g.dtype for g in grads if g is not None), torch.float32)
        if kind not in TYPES:
            raise ValueError(f"gradients must be float32, float16 or bfloat16, got {kind}")
        if dev != _current_device():
            raise ValueError(f"the parameters are on device {dev}, the current one is {_current_device()}")
        ptrs = []
        for g, shape in zip(grads, self._shapes):
            if g is None:
                ptrs.append(0)
            elif g.dtype is kind and g.shape == shape and g.get_device() == dev and g.is_contiguous():
                ptrs.append(g.data_ptr())
            else:
                raise ValueError(f"a gradient must be a contiguous {kind} tensor {tuple(shape)} on device {dev}, got "
                                 f"{g.dtype} {tuple(g.shape)} on {g.device}")
        if step < 1:
            raise ValueError(f"steps count from 1, got {step}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
            raise ValueError(f"betas must be in [0, 1) and eps not negative, got {betas} and {eps}")
        if [p.data_ptr() for p in self.params] != self._ptrs:
            raise ValueError("a parameter's memory was replaced: make a new plan")
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is not None and not self._apart(g) and (g.data_ptr() != p.data_ptr() or g.dtype != p.dtype):
                raise ValueError(f"the gradient of params[{i}] shares memory with a parameter or moment")
        scale = None
        if grad_scale is not None:
            if grad_scale.numel() != 1 or grad_scale.dtype != torch.float32 or grad_scale.get_device() != dev:
                raise ValueError(f"grad_scale must be one float32 value on device {dev}")
            if not self._apart(grad_scale):
                raise ValueError("grad_scale lies in memory that the step writes")
            scale = grad_scale.data_ptr()
        self._grad[:] = ptrs
        missing = 0 in ptrs and any(g is None for g in grads)
        if missing or self._partial:
            self._count[:] = [0 if g is None else n for g, n in zip(grads, self._counts)]
            self._partial = missing
        _check(self._lib.hg_adamw_step(
            self._table_ptr, len(grads), self._type, TYPES[kind], self.state_bits, step, lr, betas[0], betas[1], eps,
            weight_decay, scale, seed & 0xFFFFFFFF, _raw_stream(dev)), "adamw_step")
        for p, g in zip(self.params, grads):
            if g is not None and not p.is_inference():
                torch.autograd.graph.increment_version(p)


def prepare_adamw(self, params, state_bits: int = 32, state=None) -> AdamWPlan:
    """An AdamWPlan of contiguous parameters of one type.  `state`: the
    `state` of an earlier plan over tensors of the same sizes (a checkpoint),
    taken as it is, not copied; None: moments of zero."""
    return AdamWPlan(self._lib, params, state_bits, state)


METHODS = (layer_norm_forward, layer_norm_backward, policy_value_loss, prepare_adamw)
