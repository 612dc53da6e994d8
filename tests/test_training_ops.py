"""The training operators' boundary without a GPU: the C structure's layout, and
calls that the library refuses on the host before any launch."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from hive_neuralnet_amd import hive_gpu, training_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1  # hipErrorInvalidValue

needs_library = pytest.mark.skipif(not os.path.exists(hive_gpu.LIB_PATH), reason="libhive_gpu.so not built")


def test_struct_layout_matches_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    fields = [f for f, _ in training_ops.HgAdamwTensor._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "hive_gpu.h"\nint main(void) {\n'
                   'printf("size %zu\\nblock %d\\ntypes %d%d%d\\n", sizeof(hg_adamw_tensor), HG_ADAMW_BLOCK, HG_F32, '
                   'HG_F16, HG_BF16);\n'
                   + "\n".join(f'printf("{f} %zu\\n", offsetof(hg_adamw_tensor, {f}));' for f in fields)
                   + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                         text=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(training_ops.HgAdamwTensor)
    for f in fields:
        assert int(got[f]) == getattr(training_ops.HgAdamwTensor, f).offset, f
    assert int(got["block"]) == training_ops.ADAMW_BLOCK
    assert got["types"] == "".join(str(v) for v in training_ops.TYPES.values())


@needs_library
def test_norm_refusals():
    lib = hive_gpu.load_library()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def forward(x=p, kind=0, rows=1, cols=4, w_kind=0, y=p, mean=p):
        return lib.hg_layer_norm_forward(x, kind, rows, cols, cols, p, p, w_kind, 1e-5, 0, y, mean, p, None)

    for bad in (dict(kind=3), dict(kind=-1), dict(w_kind=9), dict(rows=-1), dict(cols=-1), dict(x=None),
                dict(y=None), dict(mean=None), dict(rows=1 << 40)):
        assert forward(**bad) == INVALID, bad
    assert forward(rows=0) == 0 and forward(cols=0) == 0

    def backward(dy=p, kind=0, rows=1, cols=4, dw=p, ws=p):
        return lib.hg_layer_norm_backward(dy, cols, p, kind, rows, cols, cols, p, p, p, 0, 0, p, dw, None, ws, None)

    for bad in (dict(kind=7), dict(rows=-1), dict(dy=None), dict(ws=None), dict(ws=p + 4)):
        assert backward(**bad) == INVALID, bad
    assert backward(cols=0) == 0
    assert lib.hg_layer_norm_backward_workspace(0, 64) >= 0
    assert lib.hg_layer_norm_backward_workspace(1000, 64) >= 2 * 64 * 4


@needs_library
def test_loss_refusals():
    lib = hive_gpu.load_library()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def loss(logits=p, kind=0, N=4, values=p, target_kind=0, width=4, B=1, losses=p, dv=p, ws=p):
        return lib.hg_policy_value_loss(logits, kind, N, values, p, p, target_kind, width, p, p, p, B, 1.0, 1.0, losses,
                                        p, dv, ws, None)

    for bad in (dict(kind=3), dict(target_kind=-1), dict(N=-1), dict(B=-1), dict(width=-1), dict(logits=None),
                dict(values=None), dict(losses=None), dict(dv=None), dict(ws=None), dict(ws=p + 8), dict(B=0),
                dict(B=1 << 40)):
        assert loss(**bad) == INVALID, bad
    assert lib.hg_policy_value_loss_workspace(0, 256) > 0
    assert lib.hg_policy_value_loss_workspace(100, 256) >= 100 * 8


@needs_library
def test_adamw_refusals():
    lib = hive_gpu.load_library()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def step(count=1, kind=0, grad_kind=0, bits=8, number=1, beta1=0.9, beta2=0.999, eps=1e-8, null=False, **fields):
        t = training_ops.HgAdamwTensor(p, p, p, p, p, p, 4, 0)
        for k, v in fields.items():
            setattr(t, k, v)
        return lib.hg_adamw_step(None if null else ctypes.byref(t), count, kind, grad_kind, bits, number, 1e-3, beta1,
                                 beta2, eps, 0.0, None, 0, None)

    nan = float("nan")
    for bad in (dict(count=-1), dict(kind=3), dict(grad_kind=-1), dict(bits=16), dict(number=0), dict(beta1=1.0),
                dict(beta2=-0.1), dict(beta1=nan), dict(eps=-1.0), dict(eps=nan), dict(null=True), dict(param=None),
                dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(exp_avg_scale=None),
                dict(exp_avg_sq_scale=None), dict(place=100), dict(exp_avg=p + 1), dict(bits=32, param=None)):
        assert step(**bad) == INVALID, bad
    assert step(count=0) == 0


@needs_library
def test_sizes_past_a_launch_are_refused():
    """Before anything is launched: a grid of 2^32 threads, also where only a later launch or tensor has one."""
    lib = hive_gpu.load_library()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15
    for width in (4, 512, 5000):
        assert lib.hg_policy_value_loss(p, 0, 4, p, p, p, 0, width, p, p, p, (1 << 26) - 3, 1.0, 1.0, p, p, p, p,
                                        None) == INVALID, width
    cols = (1 << 25) + 1
    assert lib.hg_layer_norm_forward(p, 0, 1, cols, cols, p, p, 0, 1e-5, 0, p, p, p, None) == INVALID
    assert lib.hg_layer_norm_backward(p, cols, p, 0, 1, cols, cols, p, p, p, 0, 0, p, p, None, p, None) == INVALID
    assert lib.hg_layer_norm_forward(p, 0, (1 << 21) + 1, 20000, 20000, p, p, 0, 1e-5, 0, p, p, p, None) == INVALID
    two = (training_ops.HgAdamwTensor * 2)()
    two[0] = training_ops.HgAdamwTensor(p, p, p, p, p, p, 4, 0)
    two[1] = training_ops.HgAdamwTensor(p, p, p, p, p, p, (1 << 34) - 1023, 256)
    assert lib.hg_adamw_step(two, 2, 0, 0, 8, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0, None) == INVALID


@pytest.mark.skipif(training_ops._calls is None, reason="_train_calls.so not built")
def test_native_calls_leave_what_they_do_not_serve():
    """None, and no error, for arguments that are not plainly right: nothing here is on a GPU."""
    if os.path.exists(hive_gpu.LIB_PATH):
        hive_gpu.load_library()
    calls, x = training_ops._calls, torch.zeros((4, 8))
    for first in (x, None, "x", 3, [x]):
        assert calls.layer_norm_forward(first, None, None, 1e-5, None) is None
        assert calls.layer_norm_backward(first, first, x, x, None, None, "sigmoid", True) is None
        assert calls.policy_value_loss(first, x, x, x, x, x, x, 1.0, 1.0) is None
        assert calls.adamw_step([first], [x], 0, 0, 32, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0) is None
    assert calls.layer_norm_forward(x, None, None, "eps", None) is None
    assert calls.layer_norm_forward(x) is None
    assert calls.adamw_step([], [], 0, 0, 32, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0) is None
    assert calls.adamw_step(x, x, 0, 0, 32, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0) is None
    with pytest.raises(TypeError):
        calls.bind(1, 2)
