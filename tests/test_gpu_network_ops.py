"""A wider network's operators against plain implementations in 64 bits: the
gated block and its gradients, orthogonalised updates and the steps of matrices
with them, slots drawn from rows of logits, at the sizes, strides and masks
where they can go wrong, and what they refuse.

Tolerances are bounds on the rounding of float32 sums.  u = 2^-24 is half a unit
in the last place of 1.  A sum of K products on the matrix cores has a chain of
K / 32 instructions for each product of parts, and at most 32 additions within
one, each taken as off by a unit in the last place (they may cut instead of
rounding): (parts K / 16 + 80) u sum |terms|.  16-bit products are exact in 32
bits.  What is rounded to 16 bits between (the gradients of gate and up) is off by half
a unit of its type."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def ext():
    from hive_neuralnet_amd import hive_gpu
    return hive_gpu.load_extension()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, scale=1.0, dtype=F32):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dtype)


def _close(got, want, bound, what):
    """|got - want| <= bound + the rounding to got's type, element by element."""
    g, w = got.double(), want.double()
    assert g.shape == w.shape, what
    assert torch.isfinite(g).all(), what
    b = torch.as_tensor(bound, dtype=torch.float64, device=g.device).expand_as(w)
    over = (g - w).abs() - b - HALF_ULP[got.dtype] * w.abs() * (1 + HALF_ULP[got.dtype]) - TINY[got.dtype]
    assert over.numel() == 0 or float(over.max()) <= 0.0, (what, float(over.max()), float(b.max()))


def _chain(K, t):
    return ((6 if t == F32 else 1) * K / 16 + 80) * U


# ---- the gated block --------------------------------------------------------


def _act(name, g):
    """act, its slope, a bound on the slope's slope; 64 bits"""
    if name == "gelu":
        share = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        bell = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * share, share + g * bell, 0.8
    share = torch.sigmoid(g)
    if name == "sigmoid":
        return share, share * (1 - share), 0.1
    return g * share, share * (1 + g * (1 - share)), 0.5


def _check_gated(ext, x, wg, wu, bg, bu, dh, act):
    t = x.dtype
    h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu, act)
    assert torch.equal(h, ext.gated_linear(x, wg, wu, bg, bu, act))
    assert h.shape == (*x.shape[:-1], wg.shape[0]) and h.dtype == t and h.is_contiguous()
    D, H = wg.shape[1], wg.shape[0]
    X, G, W = x.double().reshape(-1, D), wg.double(), wu.double()
    B, C = (0.0 if b is None else b.double() for b in (bg, bu))
    g, u = X @ G.t() + B, X @ W.t() + C
    a, slope, bend = _act(act, g)
    d_g = _chain(D, t) * (X.abs() @ G.abs().t()) + 2 * U * g.abs()
    d_u = _chain(D, t) * (X.abs() @ W.abs().t()) + 2 * U * u.abs()
    d_eval = (g.square() + g.abs() + 16) * U  # of sigmoid and erfc, relative
    d_a = 1.13 * d_g + d_eval * a.abs()
    flat = lambda v: v.reshape(-1, H)
    _close(flat(gate), g, d_g, "gate")
    _close(flat(up), u, d_u, "up")
    _close(flat(h), a * u, u.abs() * d_a + a.abs() * d_u + d_a * d_u + 2 * U * (a * u).abs(), "h")

    grads = ext.gated_linear_backward(dh, x, wg, wu, gate, up, act)
    for got, like in zip(grads, (x, wg, wu, wg[:, 0], wg[:, 0])):
        assert got.shape == like.shape and got.dtype == t and got.is_contiguous()
    V = dh.double().reshape(-1, H)
    assert gate.dtype == up.dtype == F32
    e_g, e_u = d_g + U * g.abs(), d_u + U * u.abs()  # of what is kept
    dg, du = V * u * slope, V * a
    e_dg = V.abs() * ((u.abs() + e_u) * (bend * e_g + 2 * d_eval * (slope.abs() + a.abs())) + slope.abs() * e_u) + 4 * U * dg.abs()
    e_du = V.abs() * (1.13 * e_g + d_eval * a.abs()) + 2 * U * du.abs()
    rows = X.shape[0]
    for got, want, e in ((grads[3], dg, e_dg), (grads[4], du, e_du)):
        _close(got, want.sum(0), e.sum(0) + (rows / 64 + 80) * U * want.abs().sum(0), "db")
    e_dg = e_dg + HALF_ULP[t] * (dg.abs() + e_dg) + TINY[t]  # rounded for the products
    e_du = e_du + HALF_ULP[t] * (du.abs() + e_du) + TINY[t]
    c = _chain(2 * (H + 32), t)
    _close(grads[0].reshape(-1, D), dg @ G + du @ W,
           (e_dg + c * dg.abs()) @ G.abs() + (e_du + c * du.abs()) @ W.abs(), "dx")
    c = _chain(rows + 64, t) + 260 * U  # at most 256 parts of the sum joined
    for got, want, e in ((grads[1], dg, e_dg), (grads[2], du, e_du)):
        _close(got, want.t() @ X, (e + c * want.abs()).t() @ X.abs(), "dw")


def _gated(rows, cols, hidden, t, seed, bias=True):
    s = 1.0 / math.sqrt(cols)
    return (_randn((rows, cols), seed, 1.0, t), _randn((hidden, cols), seed + 1, s, t), _randn((hidden, cols), seed + 2, s, t),
            _randn((hidden,), seed + 3, 0.3, t) if bias else None, _randn((hidden,), seed + 4, 0.3, t) if bias else None,
            _randn((rows, hidden), seed + 5, 0.1, t))


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,hidden", [(1, 1, 1), (1, 8, 16), (2, 7, 5), (1, 64, 64), (3, 33, 129), (16, 72, 40),
                                              (17, 122, 64), (65, 65, 65), (64, 256, 128), (257, 8, 600), (130, 514, 33),
                                              (1000, 96, 257)])
def test_gated(ext, rows, cols, hidden, t, act):
    _check_gated(ext, *_gated(rows, cols, hidden, t, rows + cols), act)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,hidden", [(2100, 136, 1550), (3000, 64, 4100), (20000, 40, 72), (5, 4096, 3000),
                                              (1, 2048, 5000), (4100, 1030, 2052)])
def test_gated_large(ext, rows, cols, hidden, t):
    """Every size of tile, and sums cut into parts."""
    _check_gated(ext, *_gated(rows, cols, hidden, t, 5), "silu")


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("rows,cols,hidden", [(8192, 122, 64), (8191, 122, 64), (8193, 1, 1), (9001, 128, 64), (20011, 33, 17),
                                              (40000, 64, 8), (10000, 127, 33), (8200, 129, 64), (8200, 128, 65)])
def test_gated_many_rows_of_a_narrow_block(ext, rows, cols, hidden, act):
    """Up to 128 columns and 64 units, which float32 tensors of many rows have kernels of their own for, and one past them."""
    _check_gated(ext, *_gated(rows, cols, hidden, F32, cols, bias=hidden != 33), act)


def test_gated_many_rows_of_a_narrow_block_cut_from_wider_tensors(ext):
    x, wg, wu, bg, bu, dh = _gated(8500, 101, 50, F32, 9)
    wide, wide_dh = _randn((8500, 130), 20), _randn((8500, 57), 21, 0.1)
    _check_gated(ext, wide[:, 3:104], wg, wu, bg, None, wide_dh[:, 7:], "silu")
    _check_gated(ext, wide[:1, :101].expand(8500, 101), wg, wu, None, bu, dh, "sigmoid")
    _check_gated(ext, x.view(85, 100, 101), wg, wu, bg, bu, dh[:1].expand(8500, 50).view(85, 100, 50), "gelu")


def test_gated_many_rows_of_a_narrow_block_on_their_own(ext):
    """A row's NaN and inf stay in it, what is not needed is not given and changes nothing else, a call repeats its bits in a
    graph and beside another, a unit that is off stays off."""
    x, wg, wu, bg, bu, dh = _gated(9000, 122, 64, F32, 4)
    h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    assert torch.equal(h, ext.gated_linear(x, wg, wu, bg, bu))
    whole = ext.gated_linear_backward(dh, x, wg, wu, gate, up)
    for need in ((True, False, False), (False, True, False), (False, False, True), (True, True, False)):
        some = ext.gated_linear_backward(dh, x, wg, wu, gate, up, need_dx=need[0], need_weights=need[1], need_bias=need[2])
        for a, b, n in zip(some, whole, (need[0], need[1], need[1], need[2], need[2])):
            assert torch.equal(a, b) if n else a is None
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:  # two at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append((ext.gated_linear(x, wg, wu, bg, bu), *ext.gated_linear_backward(dh, x, wg, wu, gate, up)))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = (ext.gated_linear(x, wg, wu, bg, bu), *ext.gated_linear_backward(dh, x, wg, wu, gate, up))
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        outs.append([t.clone() for t in held])
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, (h, *whole)))
    bad = x.clone()
    bad[7, 3], bad[8999, 121] = float("nan"), float("inf")
    rest = torch.ones((9000,), dtype=torch.bool, device="cuda")
    rest[[7, 8999]] = False
    out = ext.gated_linear(bad, wg, wu, bg, bu)
    assert torch.equal(out[rest], h[rest]) and torch.isnan(out[7]).all() and not torch.isfinite(out[8999]).all()
    off = bg.clone()
    off[5] = float("-inf")
    h, gate, up = ext.gated_linear_forward(x, wg, wu, off, bu)
    dx, dwg, dwu, dbg, dbu = ext.gated_linear_backward(dh, x, wg, wu, gate, up)
    assert not h[:, 5].any() and torch.isfinite(dx).all()
    assert not any(t[5].any() for t in (dwg, dwu, dbg, dbu)) and torch.isfinite(dwg).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("first,pad", [(0, 8), (1, 7), (8, 0), (3, 61)])
def test_gated_rows_cut_from_a_wider_tensor(ext, t, first, pad):
    x, wg, wu, bg, bu, dh = _gated(70, 104, 48, t, 9)
    wide = _randn((70, first + 104 + pad), 20, 1.0, t)
    wide_dh = _randn((70, 48 + pad), 21, 0.1, t)
    _check_gated(ext, wide[:, first: first + 104], wg, wu, bg, None, wide_dh[:, :48], "silu")
    _check_gated(ext, wide[::2, first: first + 104], wg, wu, None, bu, wide_dh[::2, :48], "gelu")
    flat = _randn((48 * 104 + 3,), 22, 0.1, t)
    _check_gated(ext, x, flat[1: 1 + 48 * 104].view(48, 104), flat[3: 3 + 48 * 104].view(48, 104), bg, bu, dh, "sigmoid")


def test_gated_shapes(ext):
    """Leading dimensions, one row of them, a broadcast row, no rows, one weight for both."""
    _, wg, wu, bg, bu, _ = _gated(1, 64, 40, BF16, 1)
    _check_gated(ext, _randn((3, 4, 5, 64), 1, 1.0, BF16), wg, wu, bg, bu, _randn((3, 4, 5, 40), 2, 1.0, BF16), "silu")
    _check_gated(ext, _randn((64,), 1, 1.0, BF16), wg, wu, bg, bu, _randn((40,), 2, 1.0, BF16), "silu")
    _check_gated(ext, _randn((1, 64), 1, 1.0, BF16).expand(9, 64), wg, wg, bg, bg,
                 _randn((1, 40), 2, 1.0, BF16).expand(9, 40), "gelu")
    x = torch.empty((0, 64), dtype=BF16, device="cuda")
    h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    assert h.shape == gate.shape == (0, 40)
    dx, dwg, dwu, dbg, dbu = ext.gated_linear_backward(h, x, wg, wu, gate, up)
    assert dx.shape == (0, 64) and not any(t.any() for t in (dwg, dwu, dbg, dbu)) and dwg.shape == wg.shape


def test_gated_gradients_that_are_not_needed(ext):
    x, wg, wu, bg, bu, dh = _gated(90, 64, 40, F16, 3)
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    whole = ext.gated_linear_backward(dh, x, wg, wu, gate, up)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        some = ext.gated_linear_backward(dh, x, wg, wu, gate, up, need_dx=need[0], need_weights=need[1], need_bias=need[2])
        for a, b, n in zip(some, whole, (need[0], need[1], need[1], need[2], need[2])):
            assert torch.equal(a, b) if n else a is None


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gated_far_values(ext, t):
    """Gates far on either side, where sigmoid is 0 or 1 and exp overflows."""
    x = torch.ones((4, 8), device="cuda", dtype=t)
    wg = torch.tensor([-2000.0, -100.0, -30.0, -5.0, 0.0, 5.0, 30.0, 100.0, 2000.0], device="cuda").to(t)
    wg = torch.nn.functional.pad(wg.unsqueeze(1), (0, 7))
    wu = torch.ones((9, 8), device="cuda", dtype=t)
    for act in ("sigmoid", "silu", "gelu"):
        _check_gated(ext, x, wg, wu, None, None, torch.ones((4, 9), device="cuda", dtype=t), act)


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gated_units_that_a_bias_turns_off(ext, t, act):
    """A bias of -inf: the unit's output and all that comes back through it are 0."""
    x, wg, wu, bg, bu, dh = _gated(50, 40, 36, t, 13)
    bg[[3, 35]] = float("-inf")
    h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu, act)
    assert torch.isfinite(h).all() and not h[:, [3, 35]].any() and torch.isneginf(gate[:, [3, 35]]).all()
    got = ext.gated_linear_backward(dh, x, wg, wu, gate, up, act)
    for g in got[1:]:
        assert not g[[3, 35]].any()
    off = dh.clone()
    off[:, [3, 35]] = 0
    bg[[3, 35]] = 0
    _, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu, act)
    for a, b in zip(got, ext.gated_linear_backward(off, x, wg, wu, gate, up, act)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_sample_top_k_of_any_size(ext):
    x, u = _randn((4, 70), 3), torch.tensor([0.1, 0.4, 0.7, 0.999], device="cuda")
    for a, b in zip(ext.sample_actions(x, u, top_k=2 ** 64), ext.sample_actions(x, u)):
        assert torch.equal(a, b)


def test_rows_more_than_31_bits_apart(ext):
    """Offsets and strides of tensors of more than 2^31 values."""
    apart = 2 ** 31 + 24
    store = torch.zeros((2 * apart + 512,), dtype=F16, device="cuda")
    for cols in (48, 200):
        wide = store.as_strided((3, cols), (apart, 1), 0)
        wide.copy_(_randn((3, cols), cols, 1.0, F16))
        x = wide.contiguous()
        assert torch.equal(ext.orthogonalize(wide), ext.orthogonalize(x))
        assert torch.equal(ext.orthogonalize(store.as_strided((3, 2, cols // 2), (apart, cols // 2, 1))),
                           ext.orthogonalize(x.view(3, 2, cols // 2)))
        _, wg, wu, bg, bu, dh = _gated(3, cols, 40, F16, 7)
        h, gate, up = ext.gated_linear_forward(wide, wg, wu, bg, bu)
        again = ext.gated_linear_forward(x, wg, wu, bg, bu)
        assert all(torch.equal(a, b) for a, b in zip((h, gate, up), again))
        grads = [ext.gated_linear_backward(dh, v, wg, wu, gate, up) for v in (wide, x)]
        assert all(torch.equal(a, b) for a, b in zip(*grads))
        u = torch.tensor([0.1, 0.5, 0.9], device="cuda")
        for a, b in zip(ext.sample_actions(wide, u, top_k=9), ext.sample_actions(x, u, top_k=9)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gated_activations_over_their_range(ext, t, act):
    """Gates from -12 to 12, each to what the card's own functions, polynomials and rounding allow of itself, tails too.  The
    weights' gradients are left out: sums of x silu(x) come to 9,001 / 2 * 12^2 / 3 = 216,000, past float16's 65,504."""
    x = torch.linspace(-12.0, 12.0, 9001, device="cuda").to(t).unsqueeze(1)
    one = torch.ones((1, 1), device="cuda", dtype=t)
    h, gate, up = ext.gated_linear_forward(x, one, one * 0, None, one[0], act)
    assert torch.equal(gate, x.float()) and bool((up == 1).all())
    dx = ext.gated_linear_backward(torch.ones_like(x), x, one, one * 0, gate, up, act, need_weights=False)[0]
    g = x.double()
    a, slope, _ = _act(act, g)
    d_eval = (g.square() + g.abs() + 16) * U
    _close(h, a, (d_eval + 2 * U) * a.abs(), "h")
    _close(dx, slope, 2 * d_eval * (slope.abs() + a.abs()) + (HALF_ULP[t] + _chain(64, t)) * slope.abs() * 1.01 + TINY[t], "dx")


def test_gated_float32_keeps_its_range(ext):
    """Values near the largest and the smallest floats: parts neither overflow nor vanish.  bfloat16's smallest step is
    2^-133, so the parts of a value hold it to 2^-134 (1e-38 has 7 of its bits left), which meets the other factor:
    0.5 * 2^-134 * 3.4e38 here."""
    x = torch.tensor([[3.4e38, 0.0], [1e-30, 0.0], [0.0, 3.3e38]], device="cuda")
    wu = torch.tensor([[1.0, 0.0], [1e-8, 1e-38]], device="cuda")
    wg = torch.zeros((2, 2), device="cuda")
    h = ext.gated_linear(x, wg, wu, activation="sigmoid")
    want = 0.5 * (x.double() @ wu.double().t())
    held = 0.5 * 2.0 ** -134 * (x.double().abs().sum(1, keepdim=True) + wu.double().abs().sum(1))
    assert bool(((h.double() - want).abs() <= 2.0 ** -20 * want.abs() + held).all())


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gated_nan_and_inf_stay_in_their_row(ext, t):
    x, wg, wu, bg, bu, _ = _gated(40, 122, 70, t, 4)
    clean = ext.gated_linear(x, wg, wu, bg, bu)
    x[7, 3], x[20, 121] = float("nan"), float("inf")
    h = ext.gated_linear(x, wg, wu, bg, bu)
    rest = torch.ones((40,), dtype=torch.bool, device="cuda")
    rest[[7, 20]] = False
    assert torch.equal(h[rest], clean[rest]) and torch.isnan(h[7]).all() and not torch.isfinite(h[20]).all()


def test_gated_same_bits_on_every_call_and_stream(ext):
    x, wg, wu, bg, bu, dh = _gated(5000, 136, 200, BF16, 6)
    outs = []
    for _ in range(2):
        h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
        outs.append((h, *ext.gated_linear_backward(dh, x, wg, wu, gate, up)))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:  # two at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
            outs.append((h, *ext.gated_linear_backward(dh, x, wg, wu, gate, up)))
    torch.cuda.synchronize()
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert torch.equal(a, b)


def _replays(work, changes):
    """work() captured, replayed after each of `changes`, against its eager results; eager work in between."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for change in changes:
        change()
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_gated_in_a_graph(ext):
    x, wg, wu, bg, bu, dh = _gated(300, 77, 90, F32, 7)

    def work():
        h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
        return (h, *ext.gated_linear_backward(dh, x, wg, wu, gate, up))

    _replays(work, [lambda i=i: x.copy_(_randn(x.shape, 50 + i)) for i in range(3)])


def test_gated_autograd(ext):
    """Gradients through autograd, against differences of the forward pass in float32."""
    from hive_neuralnet_amd.training import gated_linear
    x, wg, wu, bg, bu, dh = _gated(6, 10, 7, F32, 8)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    for act in ("sigmoid", "silu", "gelu"):
        def loss():
            return (gated_linear(*leaves, activation=act).double() * dh.double()).sum()

        grads = torch.autograd.grad(loss(), leaves)
        for leaf, grad in zip(leaves, grads):
            step = _randn(leaf.shape, 11)
            size = 2.0 ** -6
            with torch.no_grad():
                leaf += size * step
                more = loss()
                leaf -= 2 * size * step
                less = loss()
                leaf += size * step
            slope = float((more - less) / (2 * size))
            # the third derivative's part, size^2 / 6 |step|^3 times it, and the forward pass's own rounding
            assert abs(slope - float((grad.double() * step.double()).sum())) < 2e-2 * float(step.norm()) ** 3 * size ** 2 + 1e-4
    y = gated_linear(leaves[0], *[t.detach() for t in leaves[1:]])
    assert torch.autograd.grad(y.sum(), leaves[0])[0].shape == x.shape  # a broadcast gradient, one leaf alone
    both = torch.autograd.grad(gated_linear(x.detach(), leaves[1], leaves[1]).sum(), leaves[1])[0]
    one, two = torch.autograd.grad(gated_linear(x.detach(), leaves[1], leaves[1].detach().clone().requires_grad_()).sum(),
                                   leaves[1])[0], None
    assert both.shape == one.shape and not torch.equal(both, one)
    with torch.no_grad():
        assert not gated_linear(*leaves).requires_grad


def test_gated_refusals(ext):
    x, wg, wu, bg, bu, dh = _gated(4, 16, 8, BF16, 1)
    h, gate, up = ext.gated_linear_forward(x, wg, wu, bg, bu)
    for call in (lambda: ext.gated_linear(x.float(), wg, wu), lambda: ext.gated_linear(x, wg, wu.float()),
                 lambda: ext.gated_linear(x, wg, wu[:4]), lambda: ext.gated_linear(x[:, :8], wg, wu),
                 lambda: ext.gated_linear(x.t().contiguous().t(), wg, wu), lambda: ext.gated_linear(x, wg.cpu(), wu),
                 lambda: ext.gated_linear(x, wg, wu, bg.float()), lambda: ext.gated_linear(x, wg, wu, bg[:4]),
                 lambda: ext.gated_linear(x, wg, wu, activation="tanh"), lambda: ext.gated_linear(x.double(), wg, wu),
                 lambda: ext.gated_linear(x, _randn((16, 8), 1, 1.0, BF16).t(), wu),
                 lambda: ext.gated_linear(x, wg[:0], wu[:0]), lambda: ext.gated_linear(x.long(), wg, wu),
                 lambda: ext.gated_linear_backward(dh[:2], x, wg, wu, gate, up),
                 lambda: ext.gated_linear_backward(dh.float(), x, wg, wu, gate, up),
                 lambda: ext.gated_linear_backward(dh, x, wg, wu, gate[:2], up),
                 lambda: ext.gated_linear_backward(dh, x, wg, wu, gate, up.half())):
        with pytest.raises(ValueError):
            call()


# ---- orthogonalised updates --------------------------------------------------

ABC = (3.4445, -4.7750, 2.0315)


def _iteration(u, steps=5, coefficients=ABC, eps=1e-7, kind=torch.float64):
    """The definition, and in 64 bits a bound on the error of the kernels' rounding in the Frobenius norm.

    A step takes an error of X up by at most the largest slope of s -> a s + b s^3 + c s^5 over the singular values and
    the largest of its chords through the origin (the divided differences of an odd function of the singular values
    lie between them).  A step's own error: X, A and P are held in 22 bits (2^-23 relative, 2^-38 absolute a value), sums of
    K terms as at the top of this file, in three products of parts, whose last one is left out (2^-22)."""
    x = u.to(kind)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (x.square().sum().sqrt() + eps)
    m, n = x.shape
    error = 2.0 ** -21 * float(x.norm()) + 2.0 ** -38 * math.sqrt(m * n)
    for i in range(steps):
        a, b, c = coefficients[min(i, len(coefficients) - 1)] if isinstance(coefficients[0], (list, tuple)) else coefficients
        if kind == torch.float64:
            s = torch.linalg.svdvals(x)
            grid = torch.linspace(float(s.min()), float(s.max()), 400, dtype=kind)
            slope = float((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max())
            chord = float((a + b * grid ** 2 + c * grid ** 4).abs().max())
            top, f, g = float(s.max()), float(x.norm()), float((x @ x.mT).norm())
            sum_m, sum_n = ((3 * k / 16 + 80) * U + 2.0 ** -21 for k in (m, n))
            grow = abs(b) + 2 * abs(c) * top ** 2
            own = sum_n * f * f * grow * top + abs(c) * sum_m * g * g * top + 4 * U * (abs(b) + abs(c)) * g * top \
                + sum_m * f * (abs(b) * top ** 2 + abs(c) * top ** 4 + abs(a)) + 2.0 ** -38 * m * (grow + 2)
            error = 1.01 * max(slope, chord) * error + own
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if tall else x), error


def _check_orthogonal(got, u, *args, **kwargs):
    for g, one in zip(got.reshape(-1, *got.shape[-2:]), u.reshape(-1, *u.shape[-2:])):
        want, error = _iteration(one, *args, **kwargs)
        off = float((g.double() - want).norm())
        most = error + HALF_ULP[got.dtype] * float(want.norm()) * 1.01 + TINY[got.dtype] * math.sqrt(want.numel())
        assert off <= most, (off, most, error, tuple(one.shape))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (40, 1), (2, 2), (3, 64), (64, 122), (64, 64), (65, 33), (128, 64),
                                       (31, 200), (129, 130), (257, 64), (100, 500), (600, 90), (300, 300)])
def test_orthogonalize(ext, rows, cols, t):
    u = _randn((rows, cols), rows + cols, 0.03, t)
    got = ext.orthogonalize(u)
    assert got.shape == u.shape and got.dtype == t and got.is_contiguous()
    _check_orthogonal(got, u)


@pytest.mark.parametrize("shape", [(7, 40, 33), (2, 3, 70, 20), (1, 1, 300, 129), (200, 8, 8), (3, 1100, 260)])
def test_orthogonalize_batches(ext, shape):
    u = _randn(shape, 3)
    u *= torch.logspace(-6, 6, u[..., 0, 0].numel(), device="cuda").view(*shape[:-2], 1, 1)
    got = ext.orthogonalize(u)
    _check_orthogonal(got, u)
    assert torch.equal(got.reshape(-1, *shape[-2:])[0], ext.orthogonalize(u.reshape(-1, *shape[-2:])[0])) or \
        u[..., 0, 0].numel() > 1  # a batch may take other tiles


def test_orthogonalize_every_tile(ext):
    """Enough tiles for the largest, enough for the middle ones; no worse than eight times float32 products' error: each
    rounding here is to 22 bits where theirs is to 24."""
    for shape in ((4, 1040, 2056), (9, 700, 700)):
        u = _randn(shape, 4)
        got = ext.orthogonalize(u)
        for g, one in zip(got, u):
            want, error = _iteration(one)
            plain, _ = _iteration(one, kind=F32)
            off = float((g.double() - want).norm())
            assert off <= error and off <= 8 * float((plain.double() - want).norm())


def test_orthogonalize_strides(ext):
    """Rows cut from wider ones, every other matrix, a broadcast batch, odd addresses."""
    for t in TYPES:
        wide = _randn((6, 50, 90), 5, 1.0, t)
        for u in (wide[:, :, 3:60], wide[::2, 1:40, :77], wide[1, ::3, 5:], wide[:1].expand(4, 50, 90), wide[:, :, :1]):
            _check_orthogonal(ext.orthogonalize(u), u)
            assert torch.equal(ext.orthogonalize(u), ext.orthogonalize(u.contiguous()))


def test_orthogonalize_settings(ext):
    u = _randn((48, 70), 6)
    for steps in (1, 2, 3, 10):
        _check_orthogonal(ext.orthogonalize(u, steps=steps), u, steps)
    schedule = [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375)]
    _check_orthogonal(ext.orthogonalize(u, steps=4, coefficients=schedule), u, 4, schedule)
    _check_orthogonal(ext.orthogonalize(u, eps=1.0), u, eps=1.0)
    # a schedule whose first steps lift small singular values most: a is past X's own range
    lifting = [(8.2, -23.0, 16.8), (4.1, -2.9, 0.55), (3.9, -2.85, 0.53), (2.0, -1.5, 0.5)]
    _check_orthogonal(ext.orthogonalize(u, steps=4, coefficients=lifting), u, 4, lifting)
    big = _randn((130, 400), 61)
    _check_orthogonal(ext.orthogonalize(big, steps=4, coefficients=lifting), big, 4, lifting)
    quintic = (1.875, -1.25, 0.375)  # converges: the result is orthogonal
    q = ext.orthogonalize(u, steps=30, coefficients=quintic).double()
    assert float((q @ q.t() - torch.eye(48, device="cuda")).abs().max()) < 1e-5


def test_orthogonalize_zero_large_small_and_bad(ext):
    """Zeros stay zeros; sizes near float's ends are those of their matrix; NaN stays in its matrix."""
    u = torch.zeros((3, 20, 30), device="cuda")
    assert not ext.orthogonalize(u).any()
    for scale in (1e30, 1e-18):
        one = scale * _randn((40, 30), 7)
        _check_orthogonal(ext.orthogonalize(one, eps=0.0), one, eps=0.0)
    batch = _randn((3, 40, 30), 8)
    clean = ext.orthogonalize(batch)
    batch[1, 3, 4] = float("nan")
    got = ext.orthogonalize(batch)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    spiked = torch.zeros((64, 64), device="cuda")
    spiked[5, 9] = -3.0  # one entry of size 1
    _check_orthogonal(ext.orthogonalize(spiked), spiked)
    assert ext.orthogonalize(torch.empty((0, 5, 6), device="cuda")).shape == (0, 5, 6)


def test_orthogonalize_streams_and_graph(ext):
    u = _randn((3, 200, 130), 9)
    want = ext.orthogonalize(u)
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(ext.orthogonalize(u))
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in outs)
    _replays(lambda: [ext.orthogonalize(u)], [lambda i=i: u.copy_(_randn(u.shape, 60 + i)) for i in range(3)])


def test_orthogonalize_refusals(ext):
    u = _randn((6, 8), 1)
    for call in (lambda: ext.orthogonalize(u[0]), lambda: ext.orthogonalize(u.double()), lambda: ext.orthogonalize(u.cpu()),
                 lambda: ext.orthogonalize(u.t()), lambda: ext.orthogonalize(u[:, :0]), lambda: ext.orthogonalize(u, steps=0),
                 lambda: ext.orthogonalize(u, eps=-1.0), lambda: ext.orthogonalize(u, coefficients=(1.0, 2.0)),
                 lambda: ext.orthogonalize(u, coefficients=[(1.0, 2.0, 3.0), (1.0,)]),
                 lambda: ext.orthogonalize(u, coefficients=[]),
                 lambda: ext.orthogonalize(_randn((4, 3, 6, 8), 1).transpose(0, 1))):
        with pytest.raises(ValueError):
            call()


def _muon_reference(p, g, m, lr, mu, nesterov, decay, scale, steps=5):
    g = g.double()
    m = mu * m.double() + g
    rows, cols = p.shape
    s = math.sqrt(max(1.0, rows / cols)) if scale == "spectral" else 0.2 * math.sqrt(max(rows, cols))
    x, error = _iteration(g + mu * m if nesterov else m, steps)
    return p.double() * (1 - lr * decay) - lr * s * x, m, lr * s * error


@pytest.mark.parametrize("scale", ["spectral", "rms"])
@pytest.mark.parametrize("pt,gt", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)], ids=str)
def test_muon_step(ext, pt, gt, scale):
    """Three steps of matrices of all kinds of shapes, more of them than a launch takes; one without a gradient."""
    shapes = [(64, 122), (64, 64), (64, 128), (200, 30), (1, 50), (50, 1), (129, 257)] + [(20 + i, 40 - i) for i in range(25)]
    params = [_randn(s, i, 0.1, pt) for i, s in enumerate(shapes)]
    plan = ext.prepare_muon(params, scale=scale)
    moms = [torch.zeros(s, device="cuda") for s in shapes]
    for step in range(3):
        grads = [_randn(s, 100 * step + i, 1e-3, gt) for i, s in enumerate(shapes)]
        skip = (2, 30)[step % 2]
        grads[skip] = None
        before = [p.clone() for p in params]
        versions = [p._version for p in params]
        plan.step(grads, lr=0.05, momentum=0.9, nesterov=step != 1, weight_decay=0.1)
        for i, (p, g, b) in enumerate(zip(params, grads, before)):
            if g is None:
                assert torch.equal(p, b) and torch.equal(plan.momentum[i], moms[i]) and p._version == versions[i]
                continue
            assert p._version > versions[i]
            want, m, error = _muon_reference(b, g, moms[i], 0.05, 0.9, step != 1, 0.1, scale)
            # 0.9 is rounded to float32, which the old momentum meets before the sum: u |0.9 m|, however small the sum is
            _close(plan.momentum[i], m, 2 * U * m.abs() + U * 0.9 * moms[i].double().abs(), "momentum")
            off = float((p.double() - want).norm())
            assert off <= error * 1.1 + (HALF_ULP[pt] + 4 * U) * float(want.norm()) + 4 * U * 0.05 * float(want.norm() + 8) + \
                TINY[pt] * math.sqrt(want.numel()), (i, off, error)
            moms[i] = plan.momentum[i].clone()


def test_muon_step_workspace_with_gradients_left_out(ext):
    """Whichever matrices have a gradient, a step stays within its workspace: the first twelve have none, and as many as a
    launch takes of large ones follow."""
    shapes = [(10, 12)] * 12 + [(140, 190)] * 24 + [(12, 10)] * 12
    params = [_randn(s, i) for i, s in enumerate(shapes)]
    grads = [None if i < 12 else _randn(s, 90 + i) for i, s in enumerate(shapes)]
    plan = ext.prepare_muon(params)
    need = ext._lib.hg_muon_step_workspace(plan._table, len(shapes))
    assert need == ext._lib.hg_muon_step_workspace(plan._table, 24)  # twelve large ones and twelve small ones
    ws = torch.full((need + (1 << 24),), 0x5A, dtype=torch.uint8, device="cuda")
    for t, g in zip(plan._table, grads):
        t.grad = None if g is None else g.data_ptr()
    before = [p.clone() for p in params]
    coefficients = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)
    assert ext._lib.hg_muon_step(plan._table, len(shapes), 0, 0, 0.02, 0.95, 1, 0.0, 5, coefficients, 1, 1e-7, ws.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0x5A).all())
    for i, (p, g, b) in enumerate(zip(params, grads, before)):
        if g is None:
            assert torch.equal(p, b)
        else:
            want, _, error = _muon_reference(b, g, torch.zeros_like(b), 0.02, 0.95, True, 0.0, "spectral")
            assert float((p.double() - want).norm()) <= error * 1.1 + 5 * U * float(want.norm()) + 4 * U * 0.02 * 40


def test_muon_step_in_a_graph(ext):
    params = [_randn(s, i) for i, s in enumerate([(64, 122), (90, 30)])]
    grads = [_randn(p.shape, 9 + i) for i, p in enumerate(params)]
    start, moms = [p.clone() for p in params], [torch.zeros_like(p) for p in params]
    plan = ext.prepare_muon(params, momentum=moms)

    def restore():
        for t, s in zip(params, start):
            t.copy_(s)
        for t in moms:
            t.zero_()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan.step(grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.step(grads)
    for i in range(3):
        for g in grads:
            g.copy_(_randn(g.shape, 70 + i))
        restore()
        plan.step(grads)
        want = [t.clone() for t in params + moms]
        restore()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params + moms, want))


def test_muon_refusals(ext):
    p, q = _randn((8, 6), 1), _randn((8, 6), 2)
    both = _randn((16, 6), 3)
    for call in (lambda: ext.prepare_muon([p.double()]), lambda: ext.prepare_muon([p, q.half()]),
                 lambda: ext.prepare_muon([p[0]]), lambda: ext.prepare_muon([p[:, :3]]), lambda: ext.prepare_muon([p, p]),
                 lambda: ext.prepare_muon([both[:9], both[8:]]), lambda: ext.prepare_muon([p], momentum=[p]),
                 lambda: ext.prepare_muon([p], momentum=[q, q]), lambda: ext.prepare_muon([p], momentum=[q.half()]),
                 lambda: ext.prepare_muon([p], momentum=[q[:4]]), lambda: ext.prepare_muon([p], scale="row"),
                 lambda: ext.prepare_muon([p.cpu()])):
        with pytest.raises(ValueError):
            call()
    plan = ext.prepare_muon([p, q])
    g = _randn((8, 6), 4)
    before = [p.clone(), q.clone(), *[m.clone() for m in plan.momentum]]
    for grads, kw in (([g], {}), ([g, g.half()], {}), ([g, g.t()], {}), ([g, g.cpu()], {}), ([g, p], {}), ([q, g], {}),
                      ([g, plan.momentum[0]], {}), ([g, g], dict(steps=0)), ([g, g], dict(eps=-1.0)),
                      ([g.long(), g.long()], {}), ([g, g], dict(coefficients=(1.0,)))):
        with pytest.raises(ValueError):
            plan.step(grads, **kw)
    assert all(torch.equal(a, b) for a, b in zip([p, q, *plan.momentum], before))
    plan.step([g, g])  # one gradient for two parameters
    plan.step([None, None])


def test_muon_optimizer(ext):
    """Groups, types, closures, copies, the state's way out and back in; settings out of range."""
    import copy
    import pickle

    from hive_neuralnet_amd.training import Muon
    def made():
        return [_randn((20, 12), 1).requires_grad_(), _randn((9, 30), 2, 1.0, BF16).requires_grad_(),
                _randn((5, 5), 3).requires_grad_()]

    a, b = made(), made()
    opts = [Muon([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.1}], weight_decay=0.1) for ps in (a, b)]

    def steps(ps, opt, seeds):
        for s in seeds:
            for i, p in enumerate(ps):
                p.grad = _randn(p.shape, 10 * s + i, 1.0, p.dtype)
            opt.step()

    steps(a, opts[0], range(4))
    steps(b, opts[1], range(2))
    saved = pickle.loads(pickle.dumps(opts[1].state_dict()))
    c = [p.detach().clone().requires_grad_() for p in b]
    opt = Muon([{"params": c[:2]}, {"params": c[2:]}])
    opt.load_state_dict(saved)
    assert opt.param_groups[1]["lr"] == 0.1
    steps(c, opt, range(2, 4))
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    d = copy.deepcopy(opts[1])
    steps(d.param_groups[0]["params"] + d.param_groups[1]["params"], d, range(2, 4))
    assert all(torch.equal(p, q) for p, q in zip(a, d.param_groups[0]["params"] + d.param_groups[1]["params"]))
    assert opts[1].step(lambda: torch.tensor(2.0)) == 2.0
    a[0].grad = a[1].grad = a[2].grad = None
    before = [p.clone() for p in a]
    opts[0].step()
    assert all(torch.equal(p, q) for p, q in zip(a, before))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(steps=0), dict(scale="x")):
        with pytest.raises(ValueError):
            Muon(made()[:1], **kw)
    with pytest.raises(ValueError):
        opts[0].add_param_group({"params": [_randn((3, 3), 1)]})
    for state in ({**saved, "scale": "rms"}, {**saved, "momentum": saved["momentum"][:1]},
                  {**saved, "param_groups": saved["param_groups"][:1]}):
        with pytest.raises(ValueError):
            opts[0].load_state_dict(state)
    with pytest.raises(ValueError):
        Muon([_randn((4,), 1).requires_grad_()])


# ---- a slot of each row --------------------------------------------------------


def _draw(row, n, u, t, k, p, min_p):
    """(slot, log probability) of a list of Python floats, sums exact to 64 bits."""
    kept = sorted((i for i in range(n) if row[i] > -math.inf), key=lambda i: (-row[i], i))
    if not kept:
        return -1, 0.0
    if not t > 0:
        return kept[0], 0.0
    top = row[kept[0]]
    if 0 < k < len(kept):
        kept = kept[:k]

    def weight(i):
        return 1.0 if row[i] == top else math.exp((row[i] - top) / t) if row[i] - top > -math.inf else 0.0

    w = {i: weight(i) for i in kept}
    if p < 1.0:
        want, held, fewest = p * math.fsum(w.values()), 0.0, []
        for i in kept:
            if fewest and held >= want:
                break
            fewest.append(i)
            held += w[i]
        kept = fewest
    kept = sorted(i for i in kept if w[i] >= min(min_p, 1.0))
    total, running = math.fsum(w[i] for i in kept), 0.0
    kept = [i for i in kept if w[i] > 0]
    for i in kept:
        running += w[i]
        if running > u * total:
            break
    return i, (0.0 if row[i] == top else (row[i] - top) / t) - math.log(total)


def _check_sample(ext, logits, u, n=None, t=1.0, k=0, p=1.0, min_p=0.0):
    got, log_prob = ext.sample_actions(logits, u, n, t, k, p, min_p)
    B, K = logits.shape
    assert got.dtype == torch.int64 and log_prob.dtype == F32 and got.shape == log_prob.shape == (B,)

    def each(v):
        return v.flatten().tolist() if isinstance(v, torch.Tensor) else [v] * B

    rows = logits.double().tolist()
    rows = [[-math.inf if v != v else v for v in row] for row in rows]
    counts = [K] * B if n is None else [min(max(v, 0), K) for v in each(n)]
    want = [_draw(*a) for a in zip(rows, counts, each(u.double()), each(t), each(k), each(p), each(min_p))]
    assert got.tolist() == [w[0] for w in want]
    # weights are rounded to 2^-43, at most 2^20 of them: under 2^-23 of the whole's 1 and more; then to float32
    for g, w in zip(log_prob.tolist(), want):
        assert abs(g - w[1]) <= 2.0 ** -22 + 2.0 ** -23 * abs(w[1]), (g, w)


def _logits(B, K, seed, t=F32, scale=2.5):
    return _randn((B, K), seed, scale, t)


def _uniforms(B, seed):
    return torch.rand((B,), generator=_gen(seed), device="cuda")


SETTINGS = [dict(), dict(k=1), dict(k=5), dict(p=0.9), dict(p=0.3, t=0.7), dict(min_p=0.1), dict(k=20, p=0.8, min_p=0.05, t=1.7),
            dict(t=0.0), dict(t=0.01), dict(t=100.0, p=0.5), dict(p=0.0), dict(min_p=1.0), dict(k=10 ** 9, p=2.0)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("B,K", [(1, 1), (3, 2), (5, 63), (9, 64), (40, 255), (70, 256), (6, 257), (7, 1000), (5, 1024),
                                 (4, 1025), (3, 5000), (2, 12345)])
def test_sample(ext, B, K, t, kw):
    _check_sample(ext, _logits(B, K, B + K, t), _uniforms(B, K), **kw)


@pytest.mark.parametrize("K", [30, 256, 700, 3000])
def test_sample_ragged_rows_and_their_own_settings(ext, K):
    """Lists of every length, an empty one, counts past the row and below zero; a setting of its own for each row."""
    B = 64
    g = _gen(K)
    n = torch.randint(-2, K + 3, (B,), generator=g, device="cuda")
    n[0], n[1], n[2], n[3] = 0, 1, K, K + 100
    t = torch.rand((B,), generator=g, device="cuda") * 2
    t[5:12] = 0.0
    k = torch.randint(0, 30, (B,), generator=g, device="cuda")
    p = torch.rand((B,), generator=g, device="cuda") * 1.2
    m = torch.rand((B,), generator=g, device="cuda") * 0.2
    logits = _logits(B, K, 3)
    u = _uniforms(B, 4)
    _check_sample(ext, logits, u, n, t, k, p, m)
    _check_sample(ext, logits, u.unsqueeze(1), n.unsqueeze(1), t.unsqueeze(1), 7, p.unsqueeze(1), 0.0)


@pytest.mark.parametrize("K", [256, 900, 4000])
def test_sample_masks(ext, K):
    """-inf, NaN, the type's lowest value, inf, rows with nothing left, of one slot, of equal slots."""
    for t in TYPES:
        x = _logits(12, K, 5, t)
        x[0] = -math.inf
        x[1] = float("nan")
        x[2] = torch.finfo(t).min
        x[3, : K - 1] = -math.inf
        x[4, 1:] = torch.finfo(t).min
        x[5, 7], x[5, 9] = math.inf, math.inf
        x[6, ::2] = -math.inf
        x[7, ::3] = float("nan")
        x[8] = 1.25
        x[9] = 0.0
        x[9, ::2] = -0.0
        x[10, : K // 2] = 3.0
        for kw in (dict(), dict(k=6), dict(p=0.5), dict(p=0.7, k=11), dict(min_p=0.5), dict(t=0.0), dict(t=2.0, p=0.25)):
            _check_sample(ext, x, _uniforms(12, 6), **kw)


@pytest.mark.parametrize("K", [200, 1024, 2000])
def test_sample_the_ends_of_the_numbers(ext, K):
    """u of 0, just below 1, 1 and more, NaN: the first and the last slot kept."""
    x = _logits(1, K, 7).expand(6, K)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, float("nan")], device="cuda")
    kept = sorted(x[0].topk(9).indices.tolist())
    got, _ = ext.sample_actions(x, u, top_k=9)
    assert got.tolist() == [kept[0], kept[-1], kept[-1], kept[-1], kept[0], kept[0]]


@pytest.mark.parametrize("K", [256, 600, 6000])
def test_sample_sorted_rows(ext, K):
    """Rising, falling and equal runs, where pivots and digits are at their worst."""
    up = torch.linspace(-4, 4, K, device="cuda")
    x = torch.stack([up, up.flip(0), up.round(), up.abs(), torch.cat([up[::2], up[::2].flip(0)])[:K]])
    for kw in (dict(k=17), dict(p=0.6), dict(k=K - 1, p=0.99), dict(min_p=0.3)):
        _check_sample(ext, x, _uniforms(len(x), 8), **kw)


@pytest.mark.parametrize("t", [F32, BF16], ids=str)
@pytest.mark.parametrize("K", [1025, 2300, 4097, 9000])
def test_sample_the_largest_of_a_long_row(ext, K, t):
    """As many as there are threads, fewer and more, than a wave holds, and than there are: at random, in order, all but alike,
    with most of the row masked."""
    x = _logits(4, K, K, t)
    x[1] = x[1].sort().values
    x[2] = (x[2] * 0.5).round()
    x[3, torch.randperm(K, generator=_gen(5), device="cuda")[: K * 7 // 8]] = float("-inf")
    for k in (1, 50, 256, 257, 575, 576, 1023, 1024, 1025, 1200, K - 1, K):
        _check_sample(ext, x, _uniforms(4, k), k=k)
    _check_sample(ext, x, _uniforms(4, 3), k=300, p=0.9, min_p=0.01, t=2.0)


def test_sample_strides_and_types(ext):
    """Rows cut from wider ones, every other row, a broadcast row, odd addresses."""
    for t in TYPES:
        wide = _logits(20, 1500, 9, t)
        for x in (wide[:, 3:250], wide[::2, 1:1300], wide[:1].expand(11, 1500), wide[:, 7:8]):
            _check_sample(ext, x, _uniforms(x.shape[0], 10), p=0.8, k=40)
    assert ext.sample_actions(torch.empty((0, 8), device="cuda"), torch.empty((0,), device="cuda"))[0].shape == (0,)


def test_sample_draws_by_the_probabilities(ext):
    """Evenly spaced numbers: each slot as often as its probability says, to one."""
    x = _logits(1, 50, 11)
    n = 20000
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5).div(n).float()
    got, log_prob = ext.sample_actions(x.expand(n, 50), u)
    p = torch.softmax(x[0].double(), 0)
    counts = torch.bincount(got, minlength=50).double()
    assert float((counts - n * p).abs().max()) <= 1.01 + n * 2.0 ** -24
    assert torch.allclose(log_prob.double(), p.log()[got], atol=1e-6)


def test_sample_large_and_streams_and_graph(ext):
    x, u = _logits(300, 20000, 12, BF16), _uniforms(300, 13)
    y, v = _logits(5000, 256, 14), _uniforms(5000, 15)
    want = [*ext.sample_actions(x, u, top_p=0.9), *ext.sample_actions(y, v, top_k=30)]
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([*ext.sample_actions(x, u, top_p=0.9), *ext.sample_actions(y, v, top_k=30)])
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, o))
    small, w = _logits(9, 3000, 16), _uniforms(9, 17)
    _replays(lambda: [*ext.sample_actions(small, w, top_p=0.7), *ext.sample_actions(y, v, temperature=0.5, top_p=0.8)],
             [lambda i=i: (small.copy_(_logits(9, 3000, 80 + i)), y.copy_(_logits(5000, 256, 90 + i))) for i in range(3)])


def test_sample_refusals(ext):
    x, u = _logits(4, 10, 1), _uniforms(4, 2)
    for call in (lambda: ext.sample_actions(x[0], u), lambda: ext.sample_actions(x.double(), u),
                 lambda: ext.sample_actions(x, u[:3]), lambda: ext.sample_actions(x, u.double()),
                 lambda: ext.sample_actions(x, u.cpu()), lambda: ext.sample_actions(x.cpu(), u),
                 lambda: ext.sample_actions(x.t(), u), lambda: ext.sample_actions(x[:, :0], u),
                 lambda: ext.sample_actions(x, u, torch.ones(4, device="cuda")),
                 lambda: ext.sample_actions(x, u, torch.ones(3, dtype=torch.int64, device="cuda")),
                 lambda: ext.sample_actions(x, u, temperature=-1.0), lambda: ext.sample_actions(x, u, top_k=-1),
                 lambda: ext.sample_actions(x, u, top_p=-0.1), lambda: ext.sample_actions(x, u, min_p=1.5),
                 lambda: ext.sample_actions(x, u, temperature=float("nan")),
                 lambda: ext.sample_actions(x, u, temperature=u.double()),
                 lambda: ext.sample_actions(x, u, top_k=2.5), lambda: ext.sample_actions(x, u, top_p=None),
                 lambda: ext.sample_actions(x, u, top_k=u), lambda: ext.sample_actions(x, u, top_p=u[:2])):
        with pytest.raises(ValueError):
            call()


# ---- together ------------------------------------------------------------------


def test_a_wider_network_trains_and_plays(ext):
    """The operators as they are used: a policy and value network with a gated block on the framework's own positions, one
    step of its matrices by their orthogonalised momentum and of the rest by AdamW, then a move for each game."""
    from hive_neuralnet_amd import hive_gpu
    from hive_neuralnet_amd.training import AdamW, Muon, gated_linear, layer_norm, matrices, policy_value_loss
    B, width = 48, 96
    states, _ = hive_gpu.random_positions(B, 0, 40, 3)
    legal, n, features = ext.generate_legal_moves_and_fnn_features_batch(states, B)

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate, self.up = torch.nn.Linear(122, width), torch.nn.Linear(122, width)
            self.norm = torch.nn.LayerNorm(width)
            self.policy, self.value = torch.nn.Linear(width, 256), torch.nn.Linear(width, 1)

        def forward(self, x, native=True):
            w = (self.gate.weight, self.up.weight, self.gate.bias, self.up.bias)
            if native:
                h = layer_norm(gated_linear(x, *w), self.norm.weight, self.norm.bias)
            else:
                h = self.norm(torch.nn.functional.silu(self.gate(x)) * self.up(x))
            return self.policy(h), torch.tanh(self.value(h))

    torch.manual_seed(0)
    net = Net().cuda()
    plain = Net().cuda().double()
    plain.load_state_dict(net.state_dict())
    live = torch.arange(256, device="cuda") < n.unsqueeze(1)
    targets = torch.rand((B, 256), generator=_gen(1), device="cuda") * live
    targets /= targets.sum(1, keepdim=True).clamp(min=1e-30)
    results = torch.randint(-1, 2, (B,), generator=_gen(2), device="cuda").float()
    ones = torch.ones((B,), device="cuda")
    rows, values = net(features)
    total, _, _ = policy_value_loss(rows[live], values.squeeze(1), n.long(), targets, ones, results, ones)
    total.backward()
    prow, pval = plain(features.double(), native=False)
    masked = prow.masked_fill(~live, -math.inf)
    some = n > 0
    ce = -(targets.double() * torch.log_softmax(masked[some], 1).masked_fill(~live[some], 0.0)
           if bool(some.all()) else targets[some].double() * torch.log_softmax(masked[some], 1).masked_fill(~live[some], 0.0)).sum()
    ((ce / B) + (pval.squeeze(1) - results.double()).square().mean()).backward()
    for (name, p), q in zip(net.named_parameters(), plain.parameters()):
        # float32 through four layers of at most 256 terms: a few hundred roundings of the gradient's size
        assert float((p.grad.double() - q.grad).norm()) <= 512 * U * float(q.grad.norm()) + 1e-7, name
    taken, others = matrices(net)
    assert {tuple(p.shape) for p in taken} == {(width, 122), (256, width)}
    before = {k: v.clone() for k, v in net.state_dict().items()}
    for o in (Muon(taken, lr=0.02), AdamW(others, lr=1e-3)):
        o.step()
    for p, q in zip(taken, (before["gate.weight"], before["up.weight"], before["policy.weight"])):
        want, _, error = _muon_reference(q, p.grad, torch.zeros_like(q), 0.02, 0.95, True, 0.0, "spectral")
        assert float((p.detach().double() - want).norm()) <= error + 4 * U * float(want.norm())
    with torch.no_grad():
        rows, _ = net(features)
        u = _uniforms(B, 5)
        moves, log_prob = ext.sample_actions(rows, u, n.long(), temperature=0.8, top_p=0.95)
        _check_sample(ext, rows, u, n.long(), t=0.8, p=0.95)
    has = n > 0
    assert torch.equal(moves >= 0, has) and bool((moves < n)[has].all())
    chosen = legal[torch.arange(B, device="cuda"), moves.clamp(min=0)].contiguous()
    ext.apply_moves_batch(states, chosen, B)


def test_training_step_with_muon(ext):
    """train_batch with two optimizers that share the network's weights out."""
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import AdamW, Muon, matrices, synthetic_batch, train_batch
    torch.manual_seed(1)
    net = HiveFNN(FNNConfig.large()).cuda()
    taken, others = matrices(net)
    assert {tuple(p.shape) for p in taken} == {(64, 122), (64, 64), (64, 128)}
    before = [p.detach().clone() for p in net.parameters()]
    losses = train_batch(net, [Muon(taken, lr=0.02), AdamW(others, lr=1e-3)], synthetic_batch(64))
    assert torch.isfinite(losses).all() and all(not torch.equal(p, q) for p, q in zip(net.parameters(), before))
    for p, q in zip(net.parameters(), before):
        if any(p is t for t in taken):
            want, _, error = _muon_reference(q, p.grad, torch.zeros_like(q), 0.02, 0.95, True, 0.0, "spectral")
            assert float((p.detach().double() - want).norm()) <= error + 4 * U * float(want.norm())
