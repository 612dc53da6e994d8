"""The gated block at the ends of its numbers: float16
gradients past its range.  References and tolerances:
test_gpu_network_ops.py."""
import pytest
import torch

from test_gpu_network_ops import F16, U, _act, _gated, ext  # noqa: F401

pytestmark = pytest.mark.gpu


def _float16_case(rows, scale_dh, scale_x, scale_w, gate_bias, up_bias, seed):
    x, wg, wu, _, _, dh = _gated(rows, 72, 56, F16, seed)
    bg, bu = torch.full((56,), gate_bias, device="cuda", dtype=F16), torch.full((56,), up_bias, device="cuda", dtype=F16)
    return ((scale_x * x.float()).half(), (scale_w * wg.float()).half(), (scale_w * wu.float()).half(), bg, bu,
            (scale_dh * dh.float()).clamp(-6e4, 6e4).half())


@pytest.mark.parametrize("rows", [33, 4100])
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("large", [True, False])
def test_float16_gradients_between_past_its_range(ext, rows, act, large):  # noqa: F811
    """The gradients of gate and up go past float16's 65,504 (dh of a scaled loss), or under its smallest 6e-8, where the
    gradients that come of them are well within it.  They are held in 11 bits at the size of the largest (half a unit off, or
    2^-40 of the largest)."""
    if large:
        x, wg, wu, bg, bu, dh = _float16_case(rows, 1.5e5, 2e-4, 0.02, 1.0, 40.0, 3)
    else:
        x, wg, wu, bg, bu, dh = _float16_case(rows, 1e-6, 300.0, 300.0, -6.0, 1e-3, 4)
        wg, x = wg * 0 + 1e-4, x.abs()
        bg = bg * 0 - 4.0
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu, act)
    dx, dwg, dwu, _, _ = ext.gated_linear_backward(dh, x, wg, wu, gate, up, act, need_bias=False)
    g, u, V, X = gate.double(), up.double(), dh.double(), x.double()
    a, slope, _ = _act(act, g)
    dgate, dup = V * u * slope, V * a
    most = float(torch.maximum(dgate.abs().max(), dup.abs().max()))
    assert most > 2e5 if large else float(dup.abs().max()) < 1e-5
    d_eval = (g.square() + g.abs() + 16) * U
    off_g = (2.0 ** -11 * 1.01 + 4 * U) * dgate.abs() + 2 * d_eval * V.abs() * u.abs() * (slope.abs() + a.abs()) + 2.0 ** -40 * most
    off_u = (2.0 ** -11 * 1.01 + 4 * U + d_eval) * dup.abs() + 2.0 ** -40 * most
    chain = (rows / 16 + 400) * U
    for got, want, off in (
            (dx, dgate @ wg.double() + dup @ wu.double(),
             (off_g + chain * dgate.abs()) @ wg.double().abs() + (off_u + chain * dup.abs()) @ wu.double().abs()),
            (dwg, dgate.t() @ X, (off_g + chain * dgate.abs()).t() @ X.abs()),
            (dwu, dup.t() @ X, (off_u + chain * dup.abs()).t() @ X.abs())):
        assert float(want.abs().max()) < 6e4 and float(want.abs().max()) > 1e-6, float(want.abs().max())
        over = (got.double() - want).abs() - off - 2.0 ** -11 * want.abs() * 1.01 - 2.0 ** -25
        assert got.isfinite().all() and float(over.max()) <= 0, float(over.max())
