"""The gated block at the ends of its numbers: infinities of float32 tensors,
float16 gradients past its range; under autocast.  References and tolerances:
test_gpu_network_ops.py."""
import math

import pytest
import torch

from test_gpu_network_ops import BF16, F16, F32, U, _act, _gated, ext  # noqa: F401

pytestmark = pytest.mark.gpu


def _same_kind(got, want, what):
    """inf, -inf and NaN where `want` has them, and nowhere else."""
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), (what, "nan")
    assert torch.equal(got.isposinf(), want.isposinf()), (what, "inf")
    assert torch.equal(got.isneginf(), want.isneginf()), (what, "-inf")
    some = want.isfinite()
    # 6 (K / 16) + 80 roundings of sums of under 512 terms that are a few times the result's size at most, here loosely
    assert not some.any() or float((got - want)[some].abs().max()) <= 2.0 ** -14 * max(1.0, float(want[some].abs().max())), what


@pytest.mark.parametrize("rows,cols,hidden", [(40, 122, 70), (3, 9, 5), (8192, 122, 64), (1, 300, 40)])
def test_infinities_of_float32(ext, rows, cols, hidden):  # noqa: F811
    """An infinity times a number is an infinity of its sign and times 0 NaN, as of 16-bit tensors: in x, in the weights, in
    both, in a sum with one of the other sign."""
    x, wg, wu, _, _, _ = _gated(rows, cols, hidden, F32, 5)
    x[rows // 2, cols - 1] = math.inf
    wg[:, cols - 1], wu[:, cols - 1] = 0.5, -0.5  # whose second and third parts are 0
    wu[hidden - 1, cols - 1] = 0.0
    wg[hidden // 2, cols - 1] = -0.75
    wu[0, 2], wg[1, 1] = -math.inf, math.inf
    x[0, 2] = math.inf
    if rows > 2:
        x[2, 2], x[1, 1] = 0.0, -2.0
    _, gate, up = ext.gated_linear_forward(x, wg, wu, activation="sigmoid")
    for got, w, what in ((gate, wg, "gate"), (up, wu, "up")):
        _same_kind(got, _products(x, w), what)
    h = ext.gated_linear(x, wg, wu, activation="sigmoid")
    _same_kind(h, torch.sigmoid(_products(x, wg)) * _products(x, wu), "h")


def _products(x, w):
    """x w^T in 64 bits, each product for itself, so that infinities meet nothing but their own factor."""
    return torch.stack([(x.double() * one).sum(1) for one in w.double()], 1)


@pytest.mark.parametrize("rows,cols,hidden", [(40, 122, 70), (8192, 122, 64)])
def test_infinities_of_float32_gradients(ext, rows, cols, hidden):  # noqa: F811
    """An infinite gradient of one unit of one row: the infinities of its row of dx, of its unit's weights, and no others."""
    x, wg, wu, bg, bu, dh = _gated(rows, cols, hidden, F32, 6)
    x[7] = x[7].bfloat16().float()  # one part each
    x[7, 5] = 0.0
    wg[9], wu[9] = wg[9].bfloat16().float(), wu[9].bfloat16().float()
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    dh[7, 9] = math.inf
    dx, dwg, dwu, dbg, dbu = ext.gated_linear_backward(dh, x, wg, wu, gate, up)
    a, slope, _ = _act("silu", gate.double())
    dgate, dup = dh.double() * up.double() * slope, dh.double() * a
    rest = torch.arange(rows, device="cuda") != 7
    assert dx[rest].isfinite().all()
    _same_kind(dx[7], (dgate[7].unsqueeze(1) * wg.double()).sum(0) + (dup[7].unsqueeze(1) * wu.double()).sum(0), "dx")
    for got, d, what in ((dwg, dgate, "dw_gate"), (dwu, dup, "dw_up")):
        one = torch.arange(hidden, device="cuda") == 9
        assert got[~one].isfinite().all(), what
        _same_kind(got[9], (d[:, 9:10] * x.double()).sum(0), what)
    assert dbg[9] == dgate[7, 9] and dbu[9] == dup[7, 9]


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


@pytest.mark.parametrize("to", [BF16, F16], ids=str)
def test_autocast(ext, to):  # noqa: F811
    """What a layer under autocast hands over: float32 weights beside a float32 or 16-bit x.  The result and the gradients are
    those of tensors cast by hand; the weights' come back in their own type."""
    from hive_neuralnet_amd.training import gated_linear
    x, wg, wu, bg, bu, dh = _gated(50, 40, 24, F32, 3)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    by_hand = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    with torch.autocast("cuda", dtype=to):
        h = gated_linear(*leaves)
        with torch.no_grad():
            assert torch.equal(gated_linear(x.to(to), *leaves[1:]), h)
        with pytest.raises(ValueError):
            gated_linear(leaves[0], *[t.double() for t in leaves[1:]])
    want = gated_linear(*[t.to(to) for t in by_hand])
    assert h.dtype == to and torch.equal(h, want)
    h.backward(dh.to(to))
    want.backward(dh.to(to))
    for a, b in zip(leaves, by_hand):
        assert a.grad.dtype == F32 and torch.equal(a.grad, b.grad) and bool(a.grad.any())
    with torch.autocast("cuda", dtype=to, enabled=False):
        assert gated_linear(*leaves).dtype == F32


def test_float16_gradients_in_graphs_and_streams(ext):  # noqa: F811
    """The pass that finds the largest: a call repeats its bits beside another whose values are of another size, and in a graph
    replayed on values of other sizes."""
    x, wg, wu, bg, bu, dh = _gated(700, 72, 56, F16, 3)
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    sizes = (1.0, 2.0 ** -12, 2.0 ** 15)

    def call(v):
        return ext.gated_linear_backward(v, x, wg, wu, gate, up, need_bias=False)[:3]

    grads = [(s * dh.float()).clamp(-6e4, 6e4).half() for s in sizes]
    want = [call(v) for v in grads]
    outs, streams = [], [torch.cuda.Stream() for _ in sizes]
    for s, v in zip(streams, grads):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call(v))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    held = grads[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(held)
    for i in (1, 2, 0, 2):
        held.copy_(grads[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
        call(grads[0])
    zero = call(dh * 0)
    assert not any(t.any() for t in zero)
    # a power of two more of dh is as much more of its gradients, but for what float16 rounds them to
    for a, b in zip(call((dh.float() * 4).half()), want[0]):
        big = b.abs() > 2.0 ** -12
        assert torch.equal(a[big].float(), 4 * b[big].float())


def test_float16_gradients_that_are_not_finite(ext):  # noqa: F811
    """An infinity or NaN in dh stays in its row of dx and its unit's weights, and does not scale the rest."""
    x, wg, wu, bg, bu, dh = _gated(90, 72, 56, F16, 3)
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    clean = ext.gated_linear_backward(dh, x, wg, wu, gate, up)
    bad = dh.clone()
    bad[7, 9], bad[30, 11] = math.inf, math.nan
    got = ext.gated_linear_backward(bad, x, wg, wu, gate, up)
    rows = torch.ones((90,), dtype=torch.bool, device="cuda")
    rows[[7, 30]] = False
    units = torch.ones((56,), dtype=torch.bool, device="cuda")
    units[[9, 11]] = False
    # the largest that scales them may have stood in the two rows: equal to half a unit of the last place
    for a, b, which in zip(got, clean, (rows, units, units, units, units)):
        off = (a[which].double() - b[which].double()).abs()
        assert float((off - 2.0 ** -10 * b[which].double().abs()).max()) <= 2.0 ** -10 * float(b.abs().max())
    assert not got[0][7].isfinite().all() and got[0][30].isnan().all()
    assert not any(t[9].isfinite().all() for t in got[1:]) and all(t[11].isnan().all() for t in got[1:])
