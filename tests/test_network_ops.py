"""The boundary of a wider network's operators without a GPU: the C structure's
layout, workspaces, and calls that the library refuses on the host before any
launch."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from hive_neuralnet_amd import hive_gpu, network_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1  # hipErrorInvalidValue

needs_library = pytest.mark.skipif(not os.path.exists(hive_gpu.LIB_PATH), reason="libhive_gpu.so not built")


def _memory():
    buf = (ctypes.c_float * 256)()
    return buf, (ctypes.addressof(buf) + 255) & ~255


def test_struct_layout_matches_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    fields = [f for f, _ in network_ops.HgMuonMatrix._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "hive_gpu.h"\nint main(void) {\n'
                   'printf("size %zu\\nacts %d%d%d\\n", sizeof(hg_muon_matrix), HG_SIGMOID, HG_SILU, HG_GELU);\n'
                   + "\n".join(f'printf("{f} %zu\\n", offsetof(hg_muon_matrix, {f}));' for f in fields)
                   + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True,
                                                         text=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(network_ops.HgMuonMatrix)
    for f in fields:
        assert int(got[f]) == getattr(network_ops.HgMuonMatrix, f).offset, f
    assert got["acts"] == "".join(str(network_ops.ACTIVATIONS[a]) for a in ("sigmoid", "silu", "gelu"))


@needs_library
def test_gated_refusals():
    lib = hive_gpu.load_library()
    _, p = _memory()

    def forward(x=p, kind=1, rows=1, cols=8, wg=p, wu=p, hidden=8, act=0, h=p, gate=None, up=None, ws=p):
        return lib.hg_gated_forward(x, kind, rows, cols, cols, wg, wu, hidden, None, None, act, h, gate, up, ws, None)

    for bad in (dict(kind=3), dict(kind=-1), dict(rows=-1), dict(cols=0), dict(hidden=0), dict(act=3), dict(act=-1),
                dict(x=None), dict(wg=None), dict(wu=None), dict(h=None), dict(gate=p), dict(up=p),
                dict(rows=(1 << 20) + 1), dict(cols=(1 << 19) + 1), dict(hidden=(1 << 19) + 1),
                dict(rows=1 << 20, cols=1 << 16), dict(cols=1 << 18, hidden=1 << 18), dict(kind=0, ws=None),
                dict(kind=0, ws=p + 16), dict(cols=9, ws=None), dict(x=p + 2, ws=None)):
        assert forward(**bad) == INVALID, bad
    assert forward(rows=0, x=None, h=None) == 0
    # tensors that are taken as they are need no workspace; float32, odd widths and odd addresses do
    need = lib.hg_gated_forward_workspace
    assert need(p, 1, 4, 64, 64, p, p, 32) == 0
    assert need(p, 0, 4, 64, 64, p, p, 32) >= (4 + 32 + 32) * 64 * 6
    assert need(p, 2, 4, 63, 63, p, p, 32) >= (4 + 32 + 32) * 64 * 2
    assert need(p + 2, 2, 4, 64, 64, p, p, 32) >= 4 * 64 * 2
    assert need(p, 2, 4, 64, 65, p, p, 32) >= 4 * 64 * 2

    def backward(dh=p, x=p, kind=1, rows=1, cols=8, wg=p, hidden=8, gate=p, up=p, act=0, dx=p, dwg=p, dwu=p, ws=p):
        return lib.hg_gated_backward(dh, hidden, x, kind, rows, cols, cols, wg, p, hidden, gate, up, act, dx, dwg, dwu,
                                     None, None, ws, None)

    for bad in (dict(kind=5), dict(rows=-1), dict(cols=0), dict(act=9), dict(dh=None), dict(x=None), dict(wg=None),
                dict(gate=None), dict(up=None), dict(dwg=None), dict(dwu=None), dict(ws=None), dict(ws=p + 4),
                dict(rows=(1 << 20) + 1)):
        assert backward(**bad) == INVALID, bad
    assert backward(dx=None, dwg=None, dwu=None, ws=None) == 0  # nothing is asked for
    assert lib.hg_gated_backward_workspace(1, 0, 8, 8) == 0


@needs_library
def test_orthogonalize_refusals():
    lib = hive_gpu.load_library()
    _, p = _memory()
    c = (ctypes.c_float * 3)(1.0, 0.0, 0.0)
    nan = float("nan")

    def call(u=p, kind=0, count=1, rows=4, cols=4, steps=5, coefficients=c, triples=1, eps=1e-7, out=p, ws=p):
        return lib.hg_orthogonalize(u, kind, count, rows, cols, cols, rows * cols, steps, coefficients, triples, eps, out,
                                    ws, None)

    for bad in (dict(kind=3), dict(count=-1), dict(rows=0), dict(cols=0), dict(rows=(1 << 17) + 1), dict(steps=0),
                dict(steps=101), dict(coefficients=None), dict(triples=0), dict(eps=-1.0), dict(eps=nan), dict(u=None),
                dict(out=None), dict(ws=None), dict(ws=p + 8), dict(count=(1 << 16) + 1),
                dict(count=2, rows=1 << 17, cols=1 << 17)):
        assert call(**bad) == INVALID, bad
    assert call(count=0, u=None, out=None, ws=None) == 0
    assert lib.hg_orthogonalize_workspace(3, 10, 40) >= 3 * (2 * 10 * 64 + 2 * 10 * 32) * 4
    assert lib.hg_orthogonalize_workspace(1, 0, 40) == 0


@needs_library
def test_muon_refusals():
    lib = hive_gpu.load_library()
    _, p = _memory()
    c = (ctypes.c_float * 3)(1.0, 0.0, 0.0)

    def call(count=1, kind=0, grad_kind=0, steps=5, coefficients=c, triples=1, eps=1e-7, ws=p, null=False, **fields):
        t = network_ops.HgMuonMatrix(p, p, p, 4, 4, 1.0)
        for k, v in fields.items():
            setattr(t, k, v)
        return lib.hg_muon_step(None if null else ctypes.byref(t), count, kind, grad_kind, 0.1, 0.9, 1, 0.0, steps,
                                coefficients, triples, eps, ws, None)

    for bad in (dict(count=-1), dict(kind=3), dict(grad_kind=-1), dict(steps=0), dict(coefficients=None),
                dict(triples=0), dict(eps=-1.0), dict(ws=None), dict(ws=p + 4), dict(null=True), dict(param=None),
                dict(momentum=None), dict(momentum=p + 2), dict(rows=0), dict(cols=(1 << 17) + 1)):
        assert call(**bad) == INVALID, bad
    assert call(count=0, ws=None) == 0
    assert call(grad=None) == 0  # nothing to step
    t = (network_ops.HgMuonMatrix * 2)(*[network_ops.HgMuonMatrix(p, p, p, 64, 64, 1.0)] * 2)
    assert lib.hg_muon_step_workspace(t, 2) == 2 * lib.hg_muon_step_workspace(t, 1) > 0


@needs_library
def test_sample_refusals():
    lib = hive_gpu.load_library()
    _, p = _memory()

    def call(logits=p, kind=0, rows=1, width=4, u=p, actions=p):
        return lib.hg_sample_actions(logits, kind, rows, width, width, None, u, None, 1.0, None, 0, None, 1.0, None, 0.0,
                                     actions, None, None)

    for bad in (dict(kind=3), dict(rows=-1), dict(width=0), dict(width=(1 << 20) + 1), dict(rows=(1 << 25) + 1),
                dict(rows=(1 << 21) + 1, width=1025), dict(logits=None), dict(u=None), dict(actions=None)):
        assert call(**bad) == INVALID, bad
    assert call(rows=0, logits=None, u=None, actions=None) == 0


def test_python_refuses_what_is_not_on_a_gpu():
    ext = hive_gpu.HiveGpuExtension.__new__(hive_gpu.HiveGpuExtension)  # no call below reaches the library
    ext._lib = None
    x, w = torch.zeros((2, 8)), torch.zeros((4, 8))
    for call in (lambda: ext.gated_linear(x, w, w), lambda: ext.orthogonalize(x), lambda: ext.prepare_muon([w]),
                 lambda: ext.prepare_muon([]), lambda: ext.sample_actions(x, torch.zeros(2)),
                 lambda: ext.gated_linear(x, w, w, activation="relu"), lambda: ext.prepare_muon([w], scale="none"),
                 lambda: ext.gated_linear_backward(x, x, w, w, x, x)):
        with pytest.raises(ValueError):
            call()


def test_every_kernel_source_is_built():
    """The library is linked from all of the package's sources: a missing one would leave entry points out."""
    import glob

    from hive_neuralnet_amd import build
    assert sorted(build.SOURCES) == sorted(glob.glob(os.path.join(build.PKG, "csrc", "*.hip")))
