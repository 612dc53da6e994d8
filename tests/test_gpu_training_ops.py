"""The training operators against plain implementations in 64 bits: layer norm
and its gradients, the policy and value loss with its gradient, the AdamW step
with moments in 32 and in 8 bits, at the sizes and masks where they can go
wrong, and what they refuse.

Tolerances are bounds on the rounding of float32 sums.  u = 2^-24 is half a
unit in the last place of 1; a sum whose longest chain of additions is n terms
is at most n u sum |terms| off.  The kernels add a row of C values in chains of
at most C / 64 + 16, R rows in chains of at most R / 64 + 400; a value rounded
to 16 bits is off by half a unit of its type besides."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ext():
    from hive_neuralnet_amd import hive_gpu
    return hive_gpu.load_extension()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, seed, scale=1.0, dtype=F32):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dtype)


def _close(got, want, bound, what):
    """|got - want| <= bound + the rounding to got's type, element by element; NaN and inf in the same places."""
    g, w = got.double(), want.double()
    assert g.shape == w.shape, what
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    fine = torch.isfinite(w)
    assert torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), what
    b = torch.as_tensor(bound, dtype=torch.float64, device=g.device).expand_as(w)
    over = ((g - w).abs() - b - HALF_ULP[got.dtype] * w.abs() - TINY[got.dtype])[fine]
    assert over.numel() == 0 or float(over.max()) <= 0.0, (what, float(over.max()), float(b.max()))


# ---- layer norm -------------------------------------------------------------


def _norm_reference(x, w, b, eps, sigmoid, dy=None):
    """y, mean, rstd, dx, dw, db in 64 bits, from the formulas."""
    x = x.double()
    a = torch.sigmoid(x) if sigmoid else x
    mean = a.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((a - mean).square().mean(-1, keepdim=True) + eps)
    h = (a - mean) * rstd
    y = h * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    out = {"y": y, "mean": mean.squeeze(-1), "rstd": rstd.squeeze(-1), "a": a, "h": h}
    if dy is not None:
        dy = dy.double()
        dh = dy * (1.0 if w is None else w.double())
        da = rstd * (dh - dh.mean(-1, keepdim=True) - h * (dh * h).mean(-1, keepdim=True))
        rows = tuple(range(x.dim() - 1))
        out.update(dx=da * a * (1.0 - a) if sigmoid else da, dw=(dy * h).sum(rows), db=dy.sum(rows), dh=dh)
    return out


def _check_norm(ext, x, w, b, dy, eps=1e-5, sigmoid=False):
    act = "sigmoid" if sigmoid else None
    y, mean, rstd = ext.layer_norm_forward(x, w, b, eps, act)
    dx, dw, db = ext.layer_norm_backward(dy, x, mean, rstd, w, b, act)
    ref = _norm_reference(x, w, b, eps, sigmoid, dy)
    C, R = x.shape[-1], max(1, x.numel() // x.shape[-1])
    chain = C / 64 + 16
    big = ref["a"].abs().amax(-1, keepdim=True)
    # an error of the mean or of a moves h by as much times rstd, one of rstd by its own share of h
    d_mean = chain * U * big + 4 * U * big
    d_h = 2 * d_mean * ref["rstd"].unsqueeze(-1) + (chain + 16) * U * ref["h"].abs()
    wmax = 1.0 if w is None else w.double().abs()
    _close(mean, ref["mean"], d_mean.squeeze(-1), "mean")
    _close(rstd, ref["rstd"], (2 * d_h.amax(-1) + (chain + 8) * U) * ref["rstd"], "rstd")
    _close(y, ref["y"], d_h * wmax + 4 * U * ref["y"].abs(), "y")
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    dh_big = ref["dh"].abs().amax(-1, keepdim=True)
    h_big = ref["h"].abs().amax(-1, keepdim=True)
    d_h_big = d_h.amax(-1, keepdim=True)
    d_da = ref["rstd"].unsqueeze(-1) * dh_big * ((chain + 16) * U * (2 + 2 * h_big.square()) + 4 * h_big * d_h_big)
    _close(dx, ref["dx"], d_da * (1.0 if not sigmoid else 0.25) + 8 * U * ref["dx"].abs(), "dx")
    rows = tuple(range(x.dim() - 1))
    sums = R / 64 + 400
    if w is not None:
        terms = dy.double().abs() * (sums * U * ref["h"].abs() + d_h)
        _close(dw, ref["dw"], terms.sum(rows), "dw")
        assert dw.dtype == w.dtype
    else:
        assert dw is None
    if b is not None:
        _close(db, ref["db"], sums * U * dy.double().abs().sum(rows), "db")
    else:
        assert db is None


@pytest.mark.parametrize("sigmoid", [False, True], ids=["plain", "sigmoid"])
@pytest.mark.parametrize("xt,wt", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, BF16)],
                         ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (5, 2), (3, 63), (700, 8), (1033, 32), (257, 64), (64, 65),
                                       (130, 122), (31, 255), (16, 256), (9, 1000), (7, 2047), (6, 2050), (5, 4096),
                                       (3, 4103), (4, 8192), (3, 12289), (2, 16384), (2, 40001)])
def test_layer_norm(ext, rows, cols, xt, wt, sigmoid):
    x = _randn((rows, cols), rows + cols, 2.0, xt) + 0.5
    w = (1.0 + _randn((cols,), cols + 1, 0.2)).to(wt)
    b = _randn((cols,), cols + 2, 0.2, wt)
    _check_norm(ext, x, w, b, _randn((rows, cols), cols + 3, 1.0, xt), sigmoid=sigmoid)


@pytest.mark.parametrize("cols", [64, 513, 4096])
def test_layer_norm_without_weight_or_bias(ext, cols):
    x, dy = _randn((37, cols), 1), _randn((37, cols), 2)
    w, b = _randn((cols,), 3), _randn((cols,), 4)
    for weight, bias in ((None, None), (w, None), (None, b)):
        _check_norm(ext, x, weight, bias, dy)


@pytest.mark.parametrize("xt", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,cols,pad,first", [(33, 64, 7, 1), (10, 1000, 3, 2), (5, 4096, 64, 5), (65, 17, 1, 0)])
def test_layer_norm_of_rows_cut_from_a_wider_tensor(ext, rows, cols, pad, first, xt):
    """Row strides, and rows that begin at any element: only the elements' own alignment is given."""
    wide = _randn((rows, cols + pad + first), 5, 1.0, xt)
    wide_dy = _randn((rows, cols + 2 * pad + first), 6, 1.0, xt)
    whole = _randn((cols + 3,), 7, 1.0, xt)
    _check_norm(ext, wide[:, first: first + cols], whole[1: 1 + cols], whole[3: 3 + cols],
                wide_dy[:, first: first + cols])


def test_layer_norm_shapes(ext):
    """Leading dimensions, a broadcast row, a single dimension, no rows."""
    _check_norm(ext, _randn((3, 4, 5, 64), 1), _randn((64,), 2), None, _randn((3, 4, 5, 64), 3))
    _check_norm(ext, _randn((1, 96), 1).expand(21, 96), _randn((96,), 2), None, _randn((1, 96), 3).expand(21, 96))
    x = _randn((300,), 4)
    y, mean, rstd = ext.layer_norm_forward(x)
    assert mean.shape == rstd.shape == () and torch.equal(y, ext.layer_norm_forward(x.unsqueeze(0))[0][0])
    x = torch.empty((0, 64), device="cuda")
    y, mean, rstd = ext.layer_norm_forward(x)
    assert y.shape == (0, 64) and mean.shape == (0,)
    w = _randn((64,), 5)
    dx, dw, db = ext.layer_norm_backward(x, x, mean, rstd, w, w)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    assert ext.layer_norm_backward(x, x, mean, rstd, need_dx=False) == (None, None, None)


def test_layer_norm_far_from_zero_and_constant(ext):
    """A mean far from zero costs no more than its own rounding (the variance is a sum of squared distances);
    a constant row has a variance of 0."""
    x = _randn((40, 1000), 1) + 1000.0
    _check_norm(ext, x, None, None, _randn((40, 1000), 2))
    y, mean, rstd = ext.layer_norm_forward(torch.full((3, 200), 0.75, device="cuda"))
    assert not y.any() and torch.all(mean == 0.75) and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))


def test_layer_norm_nan_and_inf_stay_in_their_row(ext):
    x, dy = _randn((9, 300), 1), _randn((9, 300), 2)
    x[2, 7], x[5, 299] = float("nan"), float("inf")
    w = _randn((300,), 3)
    y, mean, rstd = ext.layer_norm_forward(x, w, w)
    dx, _, db = ext.layer_norm_backward(dy, x, mean, rstd, w, w)
    bad = torch.tensor([2, 5], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).all() and torch.isfinite(db).all()
    rest = torch.tensor([0, 1, 3, 4, 6, 7, 8], device="cuda")
    y2, m2, r2 = ext.layer_norm_forward(x[rest], w, w)
    assert torch.equal(y[rest], y2)
    assert torch.equal(dx[rest], ext.layer_norm_backward(dy[rest], x[rest], m2, r2, w, w)[0])
    big = torch.tensor([[200.0, -200.0, 0.0, 88.8]], device="cuda")  # sigmoid at both ends
    _check_norm(ext, big, None, None, _randn((1, 4), 4), sigmoid=True)


@pytest.mark.parametrize("rows,cols,sigmoid", [(50000, 64, True), (9000, 200, False), (2500, 1024, False),
                                               (600, 8000, False)])
def test_layer_norm_weight_gradient_over_many_rows(ext, rows, cols, sigmoid):
    """Sums over many rows, the same bits on every call and on another stream."""
    x, dy = _randn((rows, cols), 1), _randn((rows, cols), 2)
    w, b = _randn((cols,), 3), _randn((cols,), 4)
    _check_norm(ext, x, w, b, dy, sigmoid=sigmoid)
    _, mean, rstd = ext.layer_norm_forward(x, w, b)
    once = ext.layer_norm_backward(dy, x, mean, rstd, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ext.layer_norm_backward(dy, x, mean, rstd, w, b)
    side.synchronize()
    for p, q in zip(once, again):
        assert torch.equal(p, q)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 16384), (700, 16384), (1100, 9001), (600, 12290)])
def test_layer_norm_widest_rows_of_a_block(ext, t, rows, cols):
    """Several rows a block, its sums of the weights' gradients beside its registers."""
    _check_norm(ext, _randn((rows, cols), 1).to(t), _randn((cols,), 3).to(t), _randn((cols,), 4).to(t),
                _randn((rows, cols), 2).to(t), sigmoid=rows == 600)


@pytest.mark.parametrize("sigmoid", [False, True], ids=["plain", "sigmoid"])
def test_layer_norm_gradient_against_differences(ext, sigmoid):
    """<gradient, direction> against the difference of the forward pass on both sides.  The forward pass is
    about 30 u off per value: over the difference of 2e-2 of 1,500 random values that is 30 u sqrt(1500) / 2e-2
    < 4e-3; the third derivative adds about (1e-2)^2 of the slope's size (10)."""
    act = "sigmoid" if sigmoid else None
    x, dy = _randn((50, 30), 1), _randn((50, 30), 2)
    w, b = _randn((30,), 3), _randn((30,), 4)
    _, mean, rstd = ext.layer_norm_forward(x, w, b, 1e-5, act)
    grads = ext.layer_norm_backward(dy, x, mean, rstd, w, b, act)
    h = 1e-2
    for i in range(3):
        v = _randn((x, w, b)[i].shape, 5 + i)
        v = v / v.norm()

        def at(step):
            args = [t.clone() for t in (x, w, b)]
            args[i] += step * v
            return float((ext.layer_norm_forward(*args, 1e-5, act)[0].double() * dy.double()).sum())

        slope = (at(h) - at(-h)) / (2 * h)
        assert abs(slope - float((grads[i].double() * v.double()).sum())) < 2e-2, i


def test_layer_norm_over_2_to_the_32_elements(ext):
    """The last rows of a tensor whose offsets pass 32 bits."""
    rows, cols = (1 << 20) + 5, 4099
    x = torch.zeros((rows, cols), dtype=BF16, device="cuda")
    tail = _randn((70, cols), 1, 1.0, BF16)
    x[-70:] = tail
    w = _randn((cols,), 2, 1.0, BF16)
    y, mean, rstd = ext.layer_norm_forward(x, w, w)
    want, wm, wr = ext.layer_norm_forward(tail, w, w)
    assert torch.equal(y[-70:], want) and torch.equal(mean[-70:], wm) and torch.equal(rstd[-70:], wr)
    del y
    dy = torch.zeros_like(x)
    dy[-70:] = tail.flip(0)
    dx, dw, db = ext.layer_norm_backward(dy, x, mean, rstd, w, w)
    wx, ww, wb = ext.layer_norm_backward(tail.flip(0).contiguous(), tail, wm, wr, w, w)
    assert torch.equal(dx[-70:], wx) and not dx[: rows - 70].any()
    ref = _norm_reference(tail, w, w, 1e-5, False, tail.flip(0))
    _close(dw, ref["dw"], 1e-4 * ref["h"].abs().sum(0), "dw")
    _close(db, ref["db"], 1e-4 * tail.double().abs().sum(0), "db")


def test_layer_norm_refusals(ext):
    x = _randn((8, 16), 1)
    _, m, r = ext.layer_norm_forward(x)
    w = _randn((16,), 2)
    for args, word in (
            ((x.cpu(),), "GPU tensor"), ((x.double(),), "float32, float16 or bfloat16"), ((x.t(),), "contiguous"),
            ((x[0, 0],), "dimension"), ((x.view(2, 4, 16).transpose(0, 1),), "evenly spaced"), ((x[:, :0],), "column"),
            ((x, w[:15]), "shape"), ((x, w, w.half()), "one type"), ((x, w.int()), "float32"),
            ((x, torch.stack([w, w], 1)[:, 0]), "contiguous"), ((x, w, w, -1.0), "eps"),
            ((x, w, w, 1e-5, "gelu"), "activation")):
        with pytest.raises(ValueError, match=word):
            ext.layer_norm_forward(*args)
    for args, word in (((x[:4], x, m, r), "dy must be"), ((x.half(), x, m, r), "dy must be"),
                       ((x, x, m[:4], r), "mean"), ((x, x, m, r.double()), "rstd"), ((x, x, m.cpu(), r), "mean"),
                       ((x, x, m, r, w[:3]), "shape")):
        with pytest.raises(ValueError, match=word):
            ext.layer_norm_backward(*args)


# ---- the loss ---------------------------------------------------------------


def _loss_reference(logits, values, counts, targets, pw, vt, vw, coef, scale):
    """Position by position in 64 bits on the host."""
    x, pi = logits.double().cpu().numpy(), targets.double().cpu().numpy()
    v, pw, vt, vw = (t.double().cpu().numpy().reshape(-1) for t in (values, pw, vt, vw))
    n = np.clip(counts.cpu().numpy(), 0, pi.shape[1])
    W, U_ = pw.sum() or 1.0, vw.sum() or 1.0
    dx, row, at = np.zeros_like(x), np.zeros(len(n)), 0
    with np.errstate(all="ignore"):
        for b, k in enumerate(n):
            k = max(0, min(int(k), len(x) - at))
            z, q = x[at: at + k], pi[b, :k]
            if pw[b] != 0 and k and not np.all(z == -np.inf):
                lse = z.max() + np.log(np.exp(z - z.max()).sum())
                row[b] = pw[b] / W * (q * (lse - z))[q != 0].sum()
                dx[at: at + k] = scale * pw[b] / W * (np.exp(z - lse) * q.sum() - q)
            at += int(n[b])
        off = np.where(vw != 0, v - vt, 0.0)
        value = (vw / U_ * off * off).sum()
    total = row.sum() + coef * value
    t = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    return t([total, row.sum(), value]), t(dx), t(2.0 * scale * coef * vw / U_ * off)


def _loss_inputs(B, width, longest, xt, pt, seed, full=False):
    g = np.random.default_rng(seed)
    n = np.full(B, longest) if full else g.integers(0, longest + 1, B)
    if B and not full:
        n[g.integers(0, B)] = longest
    pi = g.random((B, width)).astype(np.float32) ** 8
    live = np.arange(width) < n[:, None]
    pi = np.where(live & (g.random((B, width)) < max(0.2, 1.5 / max(1, longest))), pi, 0)
    pi = pi / np.maximum(pi.sum(1, keepdims=True), 1e-6)
    pi[~live] = np.nan  # what lies past a position's moves is not read
    cuda = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    return [cuda(2.0 * g.standard_normal(int(n.sum())).astype(np.float32)).to(xt),
            cuda(np.tanh(g.standard_normal(B)).astype(np.float32)).to(xt), cuda(n.astype(np.int64)), cuda(pi.astype(
                np.float32)).to(pt), cuda((g.random(B) < 0.8).astype(np.float32)),
            cuda(g.integers(-1, 2, B).astype(np.float32)), cuda(g.integers(0, 4, B).astype(np.float32))]


def _check_loss(ext, args, coef=0.5, scale=1.0, longest=None):
    losses, dx, dv = ext.policy_value_loss(*args, value_coef=coef, loss_scale=scale)
    want, wdx, wdv = _loss_reference(*args, coef, scale)
    longest = longest or args[3].shape[1]
    B = max(1, args[1].numel())
    # a probability: its exponent's rounding (|z| < 32: 32 u) and a sum over the row; a loss: the same
    # relative to the terms' size (at most 64), and a sum over the positions
    chain = longest / 64 + 64
    w = args[4].double().reshape(-1)
    share = float(w.abs().max() / (w.sum() if w.sum() > 0 else 1.0)) if w.numel() else 0.0
    _close(dx, wdx, scale * share * chain * U * 4, "dlogits")
    _close(dv, wdv, 8 * U * wdv.abs(), "dvalues")
    bound = (chain + B / 64 + 64) * U * torch.tensor([64.0 + 4 * coef, 64.0, 4.0], dtype=torch.float64, device="cuda")
    _close(losses, want, bound, "losses")
    return losses, dx, dv


@pytest.mark.parametrize("xt,pt", [(F32, F32), (F32, F16), (BF16, F32), (F16, F16), (F16, BF16)],
                         ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("B,width,longest", [(1, 1, 1), (1, 256, 256), (3, 256, 1), (16, 256, 60), (65, 256, 256),
                                             (1000, 256, 180), (2049, 64, 64), (5000, 7, 7), (40, 300, 300),
                                             (9, 1025, 1025), (33, 2000, 1500), (5, 9001, 9001), (3, 85834, 85834)])
def test_policy_value_loss(ext, B, width, longest, xt, pt):
    _check_loss(ext, _loss_inputs(B, width, longest, xt, pt, B + width), longest=longest,
                scale=1.0 if xt == F32 else float(B))


@pytest.mark.parametrize("B,width", [(1, 85834), (7, 30000), (300, 4096), (1100, 1024)])
def test_policy_value_loss_dense(ext, B, width):
    """Every position has every action: the dense action space."""
    _check_loss(ext, _loss_inputs(B, width, width, F32, F32, 3, full=True))


def test_policy_value_loss_sums_many_positions(ext):
    """Counts of all sizes over several planning ranges, most of them small."""
    for B in (2047, 2048, 2049, 4096, 70001):
        _check_loss(ext, _loss_inputs(B, 16, 16, F32, F32, B))


@pytest.mark.parametrize("B,width,longest", [(4097, 3, 3), (24 * 1024, 5, 5), (24 * 1024 + 1, 2, 2), (262145, 2, 2),
                                             (530001, 2, 1), (4200, 1100, 20)])
def test_policy_value_loss_finds_its_logits(ext, B, width, longest):
    """Each way to a position's first logit: ranges of 256 positions and of more, by each block and by a launch."""
    _check_loss(ext, _loss_inputs(B, width, longest, F32, F32, B), longest=longest)


@pytest.mark.parametrize("width", [200, 900, 9000])
def test_policy_value_loss_of_fewer_logits_than_counts(ext, width):
    """Lists that the logits' end cuts, at every step of the ways lists are read, and no logits at all."""
    args = _loss_inputs(5, width, width, F32, F32, width, full=True)
    for left in (0, 1, 3, width - 1, width, width + 1, 2 * width + 4099 % width, 5 * width - 1):
        _check_loss(ext, [args[0][:left].contiguous(), *args[1:]], longest=width)


@pytest.mark.parametrize("longest", [40, 700, 20000])
def test_policy_value_loss_masked_logits(ext, longest):
    """-inf at moves that are masked, whole positions of them, the type's lowest value, positions of weight 0
    that hold inf or NaN, and an inf loss where the target wants a masked move."""
    args = _loss_inputs(30, longest, longest, F32, F32, 11)
    logits, values, n, pi, pw, vt, vw = args
    ends = torch.cumsum(n, 0).tolist()
    row = lambda b: slice(ends[b] - int(n[b]), ends[b])  # noqa: E731
    pw.fill_(1.0)
    g = np.random.default_rng(5)
    for b in range(30):
        k = int(n[b])
        hide = torch.from_numpy(g.random(k) < 0.5).cuda()
        logits[row(b)] = torch.where(hide, torch.full((k,), -math.inf, device="cuda"), logits[row(b)])
        pi[b, :k][hide] = 0.0
    logits[row(3)] = -math.inf  # nothing left
    pi[3, : int(n[3])] = 0.25
    logits[row(4)] = torch.finfo(F32).min  # all the lowest value: equal, so uniform
    pi[4, : int(n[4])] = 0.0
    logits[row(5)] = math.nan  # not used
    pw[5] = 0.0
    logits[row(6)] = math.inf
    pw[6] = 0.0
    vw[7], values[7] = 0.0, math.nan
    losses, dx, dv = _check_loss(ext, args)
    assert torch.isfinite(losses).all() and torch.isfinite(dx).all() and torch.isfinite(dv).all()
    assert not dx[row(3)].any() and not dx[row(5)].any()
    n2 = int(n.argmax())
    logits[row(n2)] = torch.linspace(-1, 1, int(n[n2]), device="cuda")
    logits[row(n2)][0] = -math.inf
    pi[n2, : int(n[n2])] = 0.0
    pi[n2, 0] = 1.0
    losses, dx, _ = ext.policy_value_loss(*args)
    assert float(losses[1]) == math.inf and torch.isfinite(dx).all() and float(dx[row(n2)][0]) < 0.0
    logits[row(n2)][1] = math.nan  # a NaN that is used stays in its position's gradient
    losses, dx, _ = ext.policy_value_loss(*args)
    assert torch.isnan(losses[:2]).all() and torch.isfinite(losses[2]) and torch.isnan(dx[row(n2)]).all()
    rest = torch.ones_like(dx, dtype=torch.bool)
    rest[row(n2)] = False
    assert torch.isfinite(dx[rest]).all()


def test_policy_value_loss_weights_and_counts(ext):
    """No weight at all, counts outside [0, width], logits past the positions' own and too few of them."""
    args = _loss_inputs(50, 30, 30, F32, F32, 2)
    logits, values, n, pi, pw, vt, vw = args
    losses, dx, dv = ext.policy_value_loss(logits, values, n, pi, 0 * pw, vt, 0 * vw)
    assert not losses.any() and not dx.any() and not dv.any()
    odd = n.clone()
    odd[odd == 0] = -5
    odd[odd == 30] = 1000
    for p, q in zip(ext.policy_value_loss(logits, values, odd, pi, pw, vt, vw),
                    ext.policy_value_loss(*args)):
        assert torch.equal(p, q)
    more = torch.cat([logits, torch.full((333,), math.nan, device="cuda")])
    _, dx2, _ = ext.policy_value_loss(more, values, n, pi, pw, vt, vw)
    assert torch.equal(dx2[: len(logits)], ext.policy_value_loss(*args)[1]) and not dx2[len(logits):].any()
    short = logits[: len(logits) - 100].contiguous()
    _check_loss(ext, [short, *args[1:]])
    two = [t.unsqueeze(1) for t in (values, pw, vt, vw)]  # the replay buffer's [B, 1] columns
    losses, dx, dv = ext.policy_value_loss(logits, two[0], n, pi, *two[1:])
    assert dv.shape == (50, 1) and torch.equal(losses, ext.policy_value_loss(*args)[0])
    none = [torch.empty((0,), device="cuda")] * 2 + [torch.empty((0,), dtype=torch.int64, device="cuda"),
                                                     torch.empty((0, 256), device="cuda")]
    none += [torch.empty((0,), device="cuda")] * 3
    losses, dx, dv = ext.policy_value_loss(*none)
    assert not losses.any() and dx.shape == dv.shape == (0,)


def test_policy_value_loss_repeats_its_bits(ext):
    args = _loss_inputs(3000, 256, 200, BF16, F16, 4)
    once = ext.policy_value_loss(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ext.policy_value_loss(*args)
    side.synchronize()
    for p, q in zip(once, again):
        assert torch.equal(p, q)


def test_policy_value_loss_gradient_against_differences(ext):
    """The loss is near 4 and 60 u off: over a difference of 2e-1 that is 1e-5; the third derivative of a step
    of 1e-1 spread over 400 logits adds under 1e-4 of the slope's size (1e-2)."""
    args = _loss_inputs(20, 64, 64, F32, F32, 8)
    _, dx, dv = ext.policy_value_loss(*args, value_coef=0.7)
    for i, grad in ((0, dx), (1, dv)):
        v = _randn(args[i].shape, 3 + i)
        v = v / v.norm()

        def at(step):
            moved = list(args)
            moved[i] = moved[i] + step * v
            return float(ext.policy_value_loss(*moved, value_coef=0.7)[0][0])

        slope = (at(0.1) - at(-0.1)) / 0.2
        assert abs(slope - float((grad.double() * v.double()).sum())) < 3e-5, i


def test_policy_value_loss_over_2_to_the_32_logits(ext):
    B, width = 50063, 85834
    logits = torch.zeros((B * width,), dtype=BF16, device="cuda")
    targets = torch.zeros((B, width), dtype=F16, device="cuda")
    small = _loss_inputs(3, width, width, BF16, F16, 6, full=True)
    small[4].fill_(1.0)
    logits[-3 * width:] = small[0]
    targets[-3:] = small[3]
    cut = [torch.zeros((B,), dtype=t.dtype, device="cuda") for t in small[4:]]
    for whole, part in zip(cut, small[4:]):
        whole[-3:] = part
    values = torch.zeros((B,), dtype=BF16, device="cuda")
    values[-3:] = small[1]
    n = torch.full((B,), width, dtype=torch.int64, device="cuda")
    losses, dx, dv = ext.policy_value_loss(logits, values, n, targets, *cut)
    del logits, targets
    want, wdx, wdv = ext.policy_value_loss(*small)
    assert torch.equal(dx[-3 * width:], wdx) and torch.equal(dv[-3:], wdv)
    _close(losses, want, 1e-6 * want.double().abs(), "losses")
    assert not dx[: -3 * width].any()


def test_policy_value_loss_refusals(ext):
    args = _loss_inputs(8, 16, 16, F32, F32, 1)

    def refused(i, t, word):
        bad = list(args)
        bad[i] = t
        with pytest.raises(ValueError, match=word):
            ext.policy_value_loss(*bad)

    refused(0, args[0].cpu(), "GPU tensor")
    refused(0, args[0].double(), "float32, float16 or bfloat16")
    refused(0, args[0][: len(args[0]) // 2 * 2].view(-1, 2), "one contiguous row")
    refused(0, args[0][::2], "one contiguous row")
    refused(1, args[1].half(), "values must be")
    refused(1, args[1][:5], "shape")
    refused(2, args[2].int(), "num_actions must be")
    refused(3, args[3].view(-1), "contiguous")
    refused(3, args[3].t().contiguous().t(), "contiguous")
    refused(4, args[4][:3], "policy_weights")
    refused(5, args[5].half(), "value_targets")
    refused(6, args[6].cpu(), "value_weights")
    refused(3, torch.empty((0, 16), device="cuda"), "no position")


# ---- AdamW ------------------------------------------------------------------


HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SHAPES = [(64, 122), (64,), (1,), (1, 64), (257,), (300, 7), (0,), (255,), (1024, 33), (4096,), (5,)]


def _adamw_reference(p, g, m, v, step):
    """One step in 64 bits."""
    b1, b2 = HYPER["betas"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + HYPER["eps"])
    return p - HYPER["lr"] * (HYPER["weight_decay"] * p + update), m, v


@pytest.mark.parametrize("pt,gt", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F32),
                                   (F16, BF16), (BF16, F16), (F16, F32)],
                         ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_step(ext, bits, pt, gt):
    """Four steps of tensors of all sizes, each step against 64 bits from the state before it.  m and v: two
    products and a sum (3 u); the update: at most 12 u of itself, m being off by 3 u of its larger term."""
    params = [_randn(s, i, 0.5, pt) for i, s in enumerate(SHAPES)]
    plan = ext.prepare_adamw(params, state_bits=bits)
    scale = torch.full((1,), 0.25, device="cuda")
    for step in range(1, 5):
        grads = [_randn(s, 100 * step + i, 1.0, gt) for i, s in enumerate(SHAPES)]
        before = [p.clone() for p in params]
        state = {k: t.clone() for k, t in plan.state.items()}
        plan.step(grads, step, grad_scale=scale if step % 2 else None, seed=step, **HYPER)
        for i, (p, g, b, at) in enumerate(zip(params, grads, before, plan.places)):
            n = p.numel()
            m, v = _moments(state, at, n)
            g = g.double().view(-1) * (0.25 if step % 2 else 1.0)
            wp, wm, wv = _adamw_reference(b.double().view(-1), g, m, v, step)
            terms = (0.9 * m).abs() + (0.1 * g).abs()
            root = torch.sqrt(wv / (1 - 0.99 ** step)) + 1e-8
            slack = 4 * U * b.double().view(-1).abs() + HYPER["lr"] * 16 * U * terms / (1 - 0.9 ** step) / root
            _close(p.view(-1), wp, slack, (i, step, "params"))
            if bits == 32:
                _close(plan.state["exp_avg"][at: at + n], wm, 3 * U * terms, (i, step, "exp_avg"))
                _close(plan.state["exp_avg_sq"][at: at + n], wv, 4 * U * wv, (i, step, "exp_avg_sq"))
            else:
                b1, b2 = HYPER["betas"]
                g = g.float()  # the new moments in float32, operation by operation
                m = m.float() * b1 + g * (1 - b1)
                r = torch.sqrt(v.sqrt().float().square() * b2 + (g * g) * (1 - b2))
                _close(m, wm, 3 * U * terms, (i, step, "exp_avg"))
                _close(r, torch.sqrt(wv), 8 * U * torch.sqrt(wv), (i, step, "exp_avg_sq"))
                _check_codes(plan, at, n, m, r, (i, step))


def _moments(state, at, n):
    """The two moments that a state stands for, in 64 bits."""
    m, v = state["exp_avg"][at: at + n].double(), state["exp_avg_sq"][at: at + n].double()
    if "exp_avg_scale" in state:
        block = torch.arange(at, at + n, device="cuda") // 256
        m = m * state["exp_avg_scale"].double()[block]
        v = (v * state["exp_avg_sq_scale"].double()[block]).square()
    return m, v


CODES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 ... 448


def _check_codes(plan, at, n, m, r, what):
    """The scale is the largest float32 moment over 448, to the bit; every code is one of the two that hold its
    value between them (10 u of slack); what lies past a tensor's end is zero."""
    codes = CODES.cuda()
    for key, x in (("exp_avg", m), ("exp_avg_sq", r)):
        if n == 0:
            continue
        end = -(-n // 256) * 256
        got = plan.state[key][at: at + end].double()
        scale = plan.state[key + "_scale"][at // 256: (at + end) // 256]
        assert not got[n:].any(), what
        top = torch.zeros((end,), device="cuda")
        top[:n] = x.abs()
        assert torch.equal(scale, top.view(-1, 256).amax(1).div(448.0).clamp(min=2.0 ** -110)), what
        x = x.double()
        y = x.abs() / scale.double().repeat_interleave(256)[:n]
        below = codes[(torch.searchsorted(codes, y * (1 - 10 * U), right=True) - 1).clamp(min=0)]
        above = codes[torch.searchsorted(codes, y * (1 + 10 * U)).clamp(max=126)]
        a = got[:n].abs()
        ok = (a >= below) & (a <= above) & ((a == 0) | (torch.sign(got[:n]) == torch.sign(x)))
        if key == "exp_avg_sq":
            ok &= (a > 0) | (x == 0)
            ok |= (a == 2.0 ** -9) & (y > 0) & (y < 2.0 ** -9)
        assert ok.all(), (what, key, int((~ok).sum()))


def test_adamw_8_bit_rounding_is_unbiased(ext):
    """The mean of many steps' codes from one state.  A code is off by less than a spacing, 1/8 of its value or
    2^-9; over 4,000 seeds the mean's standard deviation is at most half a spacing / sqrt(4000) and six of them
    are under 5% of a spacing (512 values: a chance under 1e-6 of a false alarm)."""
    n, seeds = 512, 4000
    g = torch.exp(_randn((n,), 1, 1.5)) * torch.sign(_randn((n,), 2))
    sums = torch.zeros((2, n), dtype=torch.float64, device="cuda")
    for seed in range(seeds):
        plan = ext.prepare_adamw([torch.zeros((n,), device="cuda")], state_bits=8)
        plan.step([g], 1, seed=seed, **HYPER)
        m, v = _moments(plan.state, 0, n)
        sums[0] += m
        sums[1] += v.sqrt()
    for mean, x, key in ((sums[0] / seeds, 0.1 * g.double(), "exp_avg"),
                         (sums[1] / seeds, 0.1 * g.double().abs(), "exp_avg_sq")):
        scale = plan.state[key + "_scale"].double().repeat_interleave(256)
        spacing = torch.maximum(x.abs() / 8, 2.0 ** -9 * scale)
        assert float(((mean - x).abs() / spacing).max()) < 0.05, key


def test_adamw_8_bit_bits_depend_on_seed_and_place_alone(ext):
    """The same seed gives the same codes whatever launches beside it; a tensor cut in two at a multiple of 256
    elements is stepped like the whole; another seed rounds otherwise."""
    g = _randn((4096,), 1)

    def codes(splits, seed):
        params = [torch.zeros((n,), device="cuda") for n in splits]
        plan = ext.prepare_adamw(params, state_bits=8)
        plan.step(list(torch.split(g, splits)), 1, seed=seed)
        return plan.state["exp_avg"].view(torch.uint8), plan.state["exp_avg_sq"].view(torch.uint8)

    whole = codes([4096], 7)
    for again in (codes([4096], 7), codes([256, 1024, 2816], 7)):
        assert torch.equal(whole[0], again[0]) and torch.equal(whole[1], again[1])
    other = codes([4096], 8)
    assert 0.1 < float((whole[0] != other[0]).float().mean()) < 0.9
    assert not torch.equal(whole[0] == other[0], whole[1] == other[1])


def test_adamw_8_bit_range(ext):
    """Gradients of zero, the smallest and the largest, one block of each kind; a second moment above zero is
    never held as zero; inf and NaN stay in their block."""
    g = torch.zeros((8 * 256,), device="cuda")
    g[256:512] = 1e-30
    g[512:768] = 1e18
    g[768:1024] = torch.logspace(-12, 3, 256, device="cuda")
    g[1024] = 1e-38
    g[1300] = math.inf
    g[1600] = math.nan
    g[1792:] = 1.0
    p = torch.zeros_like(g)
    plan = ext.prepare_adamw([p], state_bits=8)
    plan.step([g], 1, **HYPER)
    m, v = _moments(plan.state, 0, g.numel())
    assert not m[:256].any() and not v[:256].any() and not p[:256].any()
    assert (v[768:1024] > 0).all()
    assert torch.allclose(m[512:768], torch.full_like(m[512:768], 1e17), rtol=1e-5)
    assert torch.allclose(m[1792:], torch.full_like(m[1792:], 0.1), rtol=1e-6)
    assert torch.isfinite(p[:1300]).all() and torch.isnan(p[1600]) and torch.isfinite(p[1601:]).all()
    for i in (5, 6):  # the blocks of the inf and of the NaN
        assert not torch.isfinite(plan.state["exp_avg_scale"][i])
    assert torch.isfinite(plan.state["exp_avg_scale"][[0, 1, 2, 3, 4, 7]]).all()


def test_adamw_many_tensors_and_places(ext):
    """Hundreds of tensors (several launches), views at any element of a flat buffer, and no write outside."""
    g = np.random.default_rng(3)
    sizes = g.integers(1, 700, 301).tolist()
    for pt, bits in ((F32, 32), (BF16, 32), (F32, 8), (F16, 8)):
        flat = _randn((sum(sizes) + 2 * len(sizes),), 1, 1.0, pt)
        flat_g = _randn((sum(sizes) + 2 * len(sizes),), 2, 1.0, pt)
        cuts, at = [], 1
        for n in sizes:
            cuts.append((at, n))
            at += n + 2 - (n % 3 == 0)
        before = flat.clone()
        params = [flat[a: a + n] for a, n in cuts]
        plan = ext.prepare_adamw(params, state_bits=bits)
        plan.step([flat_g[a: a + n] for a, n in cuts], 1, **HYPER)
        inside = torch.zeros_like(flat, dtype=torch.bool)
        for a, n in cuts:
            inside[a: a + n] = True
        assert torch.equal(flat[~inside], before[~inside])
        zero = torch.zeros((1,), dtype=torch.float64, device="cuda")
        want, _, _ = _adamw_reference(before.double(), flat_g.double(), zero, zero, 1)
        _close(flat[inside], want[inside], 4 * U * before.double()[inside].abs() + HYPER["lr"] * 32 * U, (pt, bits))


def test_adamw_state_comes_back(ext):
    """A plan made from another's state goes on where that one stopped."""
    for bits in (32, 8):
        a = [_randn((300, 7), 1), _randn((65,), 2)]
        b = [t.clone() for t in a]
        grads = [[_randn(t.shape, 10 * k + i) for i, t in enumerate(a)] for k in range(4)]
        plan = ext.prepare_adamw(a, state_bits=bits)
        for k in range(4):
            plan.step(grads[k], k + 1, seed=k)
        plan = ext.prepare_adamw(b, state_bits=bits)
        for k in range(2):
            plan.step(grads[k], k + 1, seed=k)
        saved = {k: t.cpu() for k, t in plan.state.items()}
        plan = ext.prepare_adamw(b, state_bits=bits, state={k: t.cuda() for k, t in saved.items()})
        for k in range(2, 4):
            plan.step(grads[k], k + 1, seed=k)
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_adamw_over_2_to_the_32_elements(ext):
    n = (1 << 32) + 4099
    p = torch.zeros((n,), dtype=BF16, device="cuda")
    g = torch.zeros((n,), dtype=BF16, device="cuda")
    p[-5000:], g[-5000:] = _randn((5000,), 1, 1.0, BF16), _randn((5000,), 2, 1.0, BF16)
    small, small_g = p[-5000:].clone(), g[-5000:].clone()
    for bits in (32, 8):
        plan = ext.prepare_adamw([p], state_bits=bits)
        plan.step([g], 1, **HYPER)
        one = ext.prepare_adamw([small], state_bits=32)
        one.step([small_g], 1, **HYPER)
        assert torch.equal(p[-5000:], small) and not p[:-5000].any()
        m, _ = _moments(plan.state, n - 5000, 5000)
        assert float((m - 0.1 * small_g.double()).abs().max()) < 0.1 * 4.0 * (1e-6 if bits == 32 else 0.125)
        del plan, m


def test_adamw_refusals(ext):
    p = [_randn((8, 4), 1), _randn((3,), 2)]
    for args, word in ((([],), "at least one"), (([p[0].cpu()],), "GPU tensor"),
                       (([p[0], p[1].half()],), "one type"), (([p[0].t()],), "contiguous"),
                       (([p[0].double()],), "float32, float16 or bfloat16"), ((p, 16), "32 or 8"),
                       ((p, 32, {"exp_avg": p[0]}), "must hold"),
                       ((p, 32, {"exp_avg": p[0], "exp_avg_sq": p[0]}), "contiguous torch.float32 tensor of 512")):
        with pytest.raises(ValueError, match=word):
            ext.prepare_adamw(*args)
    plan = ext.prepare_adamw(p)
    g = [_randn((8, 4), 3), _randn((3,), 4)]
    before = [t.clone() for t in p]
    for grads, kw, word in ((g[:1], {}, "1 gradients"), ([g[0], g[1].half()], {}, "contiguous"),
                            ([g[0].t().contiguous().t(), g[1]], {}, "contiguous"), ([g[0], g[0]], {}, "contiguous"),
                            ([t.double() for t in g], {}, "float32, float16 or bfloat16"),
                            ([t.cpu() for t in g], {}, "contiguous"), (g, {"step": 0}, "count from 1"),
                            (g, {"betas": (1.0, 0.9)}, "betas"), (g, {"eps": -1.0}, "eps"),
                            (g, {"grad_scale": torch.ones((2,), device="cuda")}, "grad_scale"),
                            (g, {"grad_scale": torch.ones((1,))}, "grad_scale")):
        kw = {"step": 1, **kw}
        with pytest.raises(ValueError, match=word):
            plan.step(grads, **kw)
    p[1].data = p[1].data.clone()
    with pytest.raises(ValueError, match="new plan"):
        plan.step(g, 1)
    assert all(torch.equal(a, b) for a, b in zip(p, before))


# ---- the two ways of a call ---------------------------------------------------


def _each_entry_point(ext):
    """What every entry point gives for plain arguments, as a list of tensors."""
    out = []
    for t, w_type, sigmoid in ((F32, F32, None), (BF16, F32, "sigmoid"), (F16, F16, None)):
        wide = _randn((300, 200), 1).to(t)
        x, dy = wide[:, 3:180], _randn((300, 177), 2).to(t)
        w, b = _randn((177,), 3).to(w_type), _randn((177,), 4).to(w_type)
        for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
            y, mean, rstd = ext.layer_norm_forward(x, weight, bias, 1e-5, sigmoid)
            out += [y, mean, rstd, *ext.layer_norm_backward(dy, x, mean, rstd, weight, bias, sigmoid)]
            out += ext.layer_norm_backward(dy, x, mean, rstd, weight, bias, sigmoid, need_dx=False)
        deep = dy.contiguous().view(3, 100, 177)
        out += ext.layer_norm_forward(deep, w, b)
        out += ext.policy_value_loss(*_loss_inputs(50, 30, 30, t, F32, 2), value_coef=0.5, loss_scale=3.0)
        args = _loss_inputs(50, 30, 30, t, F16, 2)
        out += ext.policy_value_loss(args[0], args[1].unsqueeze(1), args[2], args[3],
                                     *[a.unsqueeze(1) for a in args[4:]])
        for bits in (32, 8):
            params = [_randn((n,), n).to(t) for n in (1, 300, 4097)]
            plan = ext.prepare_adamw(params, bits)
            grads = [_randn((p.numel(),), 7).to(w_type) for p in params]
            scale = torch.full((1,), 0.25, device="cuda")
            plan.step(grads, 1, 1e-2, seed=5)
            plan.step([grads[0], None, grads[2]], 2, 1e-2, seed=6)
            plan.step(grads, 3, 1e-2, grad_scale=scale, seed=(1 << 40) - 3)
            plan.step(tuple(grads), 4, 1e-2, betas=(0.5, 0.9), eps=1e-3, weight_decay=0.1, seed=8)
            out += params + [v.float() for v in plan.state.values()]
    return [v for v in out if v is not None], [v is None for v in out]


def test_native_calls_give_what_python_gives(ext, monkeypatch):
    from hive_neuralnet_amd import training_ops
    assert training_ops._calls is not None, "built with the library"
    native, gaps = _each_entry_point(ext)
    monkeypatch.setattr(training_ops, "_calls", None)
    alone, gaps_alone = _each_entry_point(ext)
    assert gaps == gaps_alone and len(native) == len(alone)
    for p, q in zip(native, alone):
        assert p.shape == q.shape and p.dtype == q.dtype and p.is_contiguous() and torch.equal(p, q)
        assert not p.requires_grad


def test_native_calls_serve_plain_arguments_and_leave_the_rest(ext):
    from hive_neuralnet_amd import training_ops
    calls = training_ops._calls
    x, w = _randn((40, 64), 1), _randn((64,), 2)
    assert calls.layer_norm_forward(x, w, w, 1e-5, None) is not None
    for bad in ((x.t(), w, w, 1e-5, None), (x, w[:3], w, 1e-5, None), (x, w, w.half(), 1e-5, None),
                (x.double(), None, None, 1e-5, None), (x, w.cpu(), None, 1e-5, None), (x, w, w, -1.0, None),
                (x, w, w, float("nan"), None), (x, w, w, 1e-5, "tanh"), (x[:, :0], None, None, 1e-5, None),
                (x[0, 0], None, None, 1e-5, None), (x, _randn((128,), 1)[::2], None, 1e-5, None)):
        assert calls.layer_norm_forward(*bad) is None
    _, mean, rstd = ext.layer_norm_forward(x)
    assert calls.layer_norm_backward(x, x, mean, rstd, w, w, None, True) is not None
    for bad in ((x[:4], x, mean, rstd), (x.half(), x, mean, rstd), (x, x, mean[:4], rstd), (x, x, mean, rstd.double()),
                (x, x, mean.cpu(), rstd), (x.t().contiguous().t(), x, mean, rstd)):
        assert calls.layer_norm_backward(*bad, w, w, None, True) is None
    args = _loss_inputs(10, 30, 30, F32, F32, 2)
    assert calls.policy_value_loss(*args, 1.0, 1.0) is not None
    for i, bad in ((0, args[0].double()), (0, args[0].unsqueeze(0)), (1, args[1][:3]), (1, args[1].half()),
                   (2, args[2].int()), (3, args[3][:, ::2]), (3, args[3].double()), (4, args[4].double()),
                   (5, args[5].cpu()), (6, args[6].unsqueeze(0)), (6, None)):
        assert calls.policy_value_loss(*[bad if k == i else a for k, a in enumerate(args)], 1.0, 1.0) is None, i
    p, g = [_randn((64,), 1)], [_randn((64,), 2)]
    plan = ext.prepare_adamw(p)
    before = p[0].clone()

    def step(params=p, grads=g, number=1, beta1=0.9, eps=1e-8, scale=None):
        return calls.adamw_step(params, grads, plan._table_ptr, 0, 32, number, 1e-3, beta1, 0.999, eps, 0.0, scale, 0)

    for bad in (dict(grads=[None]), dict(grads=[g[0][:3]]), dict(grads=[g[0].double()]), dict(grads=[g[0].cpu()]),
                dict(grads=g + g), dict(number=0), dict(number=1.5), dict(beta1=1.0), dict(eps=-1.0),
                dict(scale=torch.ones((2,), device="cuda")), dict(scale=1.0), dict(params=[before])):
        assert step(**bad) is None, bad
    assert torch.equal(p[0], before) and step() is True and not torch.equal(p[0], before)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_adamw_refuses_memory_that_a_step_writes_twice(ext, native, monkeypatch):
    """The same weight twice, slices that overlap, one tensor as both moments, moments in a weight's memory, and
    gradients or a scale that lie in what the step writes; nothing is launched.  Slices side by side are served, and a
    gradient that is its own weight's memory."""
    from hive_neuralnet_amd import training_ops
    if not native:
        monkeypatch.setattr(training_ops, "_calls", None)
    flat = _randn((1024,), 1)
    other = _randn((256,), 2)
    zeros = torch.zeros((512,), device="cuda")
    inside = torch.zeros((1024,), device="cuda")
    for params, state, word in (
            ([other, other], None, r"params\[0\] and params\[1\]"), ([flat[:300], flat[299:]], None, "share memory"),
            ([flat[100:200], flat], None, "share memory"), ([flat, other, flat[5:6]], None, "share memory"),
            ([flat[:300]], {"exp_avg": zeros, "exp_avg_sq": zeros}, "exp_avg_sq"),
            ([inside[700:1000]], {"exp_avg": inside[:512], "exp_avg_sq": inside[256:768]}, "share memory"),
            ([inside[500:800]], {"exp_avg": inside[:512], "exp_avg_sq": zeros}, r"exp_avg and params\[0\]")):
        with pytest.raises(ValueError, match=word):
            ext.prepare_adamw(params, 32, state)
    p = [flat[:300], flat[300:], torch.empty((0,), device="cuda"), other]
    plan = ext.prepare_adamw(p)
    before = flat.clone()
    g = [torch.ones_like(t) for t in p]
    for grads, kw in (([flat[1:301], *g[1:]], {}), ([*g[:3], flat[:256]], {}), ([*g[:3], flat[768:]], {}),
                      ([*g[:3], plan.state["exp_avg"][5:261]], {}), (g, {"grad_scale": flat[300:301]}),
                      (g, {"grad_scale": plan.state["exp_avg_sq"][:1]})):
        with pytest.raises(ValueError, match="memory"):
            plan.step(grads, 1, **kw)
    with pytest.raises(ValueError, match="memory"):  # at its weight's address, but not element for element
        ext.prepare_adamw([flat]).step([flat[:512].view(BF16)], 1)
    assert torch.equal(flat, before)
    plan.step([p[0], g[1], g[2], p[3]], 1, **HYPER)  # a gradient that is the weight itself
    zero = torch.zeros((1,), dtype=torch.float64, device="cuda")
    want, _, _ = _adamw_reference(before[:300].double(), before[:300].double(), zero, zero, 1)
    _close(p[0], want, 4 * U * before[:300].double().abs() + HYPER["lr"] * 16 * U, "own memory")


@pytest.mark.parametrize("t", [F32, BF16], ids=str)
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_a_square_past_float32(ext, bits, t):
    """A finite gradient whose square is inf: the formula's update is m / inf = 0, the weight only decays; the
    others of its 256 are stepped as ever (the terms of test_adamw_step)."""
    p, g = _randn((600,), 1, 0.5), _randn((600,), 2).to(t)
    g[[7, 300, 599]] = torch.tensor([1e20, -3e38, 2e19], device="cuda").to(t)
    before = p.clone()
    plan = ext.prepare_adamw([p], state_bits=bits)
    plan.step([g], 1, **HYPER)
    zero = torch.zeros((1,), dtype=torch.float64, device="cuda")
    want, _, _ = _adamw_reference(before.double(), g.double(), zero, zero, 1)
    keep = before.double() * (1.0 - HYPER["lr"] * HYPER["weight_decay"])
    want = torch.where(torch.isinf(g.float() * g.float()), keep, want)
    _close(p, want, 4 * U * before.double().abs() + HYPER["lr"] * 16 * U, "params")
    _, v = _moments(plan.state, 0, 600)
    assert not torch.isfinite(v[[7, 300, 599]]).any()
    assert bits == 8 or torch.isfinite(v[[0, 6, 8, 301, 598]]).all()


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("cols", [7, 15, 30, 60, 61, 63, 122, 1001, 2047])
def test_layer_norm_constant_rows(ext, cols, t):
    """Rows of one value whose sum float32 holds exactly (a multiple of 16 below 2^28): their mean is that value,
    so y is the bias, and what the backward pass takes from h, the weight's gradient, is 0."""
    x = torch.tensor([10000.0, -30000.0, 16.0], device="cuda").to(t).unsqueeze(1).repeat(1, cols)
    w, b, dy = _randn((cols,), 1), _randn((cols,), 2), _randn((3, cols), 3, 1.0, t)
    y, mean, rstd = ext.layer_norm_forward(x, w, b)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, b.to(t).expand(3, cols))
    _close(rstd, torch.full((3,), 1e-5, dtype=torch.float64, device="cuda").rsqrt(), 4 * U * 317, "rstd")
    dx, dw, db = ext.layer_norm_backward(dy, x, mean, rstd, w, b)
    assert not dw.any()
    dh = dy.double() * w.double()
    want = rstd.double().unsqueeze(1) * (dh - dh.mean(1, keepdim=True))
    bound = rstd.double().unsqueeze(1) * (dh.abs() + dh.abs().mean(1, keepdim=True)) * (cols / 64 + 24) * U
    _close(dx, want, bound, "dx")


@pytest.mark.parametrize("cols", [60, 1001, 4096])
def test_layer_norm_backward_far_from_zero(ext, cols):
    """h as the distance from the mean over the deviation, which far from zero the rounding of mean * rstd is not
    part of.  Against 64 bits from the same mean and rstd: h is 3 u off, a sum of R rows (R + 6) u of its terms, a
    row's sums (C / 64 + 24) u of theirs; dy goes along with h, so that dx has its share of h."""
    x = _randn((3, cols), 1) + 1000.0
    _, mean, rstd = ext.layer_norm_forward(x)
    h = (x.double() - mean.double().unsqueeze(1)) * rstd.double().unsqueeze(1)
    dy, w = (h + _randn((3, cols), 2, 0.1)).float(), _randn((cols,), 3, 0.1) + 1.0
    dx, dw, _ = ext.layer_norm_backward(dy, x, mean, rstd, w, w)
    _close(dw, (dy.double() * h).sum(0), 9 * U * (dy.double() * h).abs().sum(0), "dw")
    dh = dy.double() * w.double()
    s1, s2 = dh.mean(1, keepdim=True), (dh * h).mean(1, keepdim=True)
    size = dh.abs() + dh.abs().mean(1, keepdim=True) + h.abs() * (dh * h).abs().mean(1, keepdim=True)
    _close(dx, rstd.double().unsqueeze(1) * (dh - s1 - h * s2),
           rstd.double().unsqueeze(1) * size * (cols / 64 + 24) * U, "dx")


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_adamw_step_raises_the_weights_versions(ext, native, monkeypatch):
    """A weight that autograd saved before a step of the plan is known to have changed; one left out has not."""
    from hive_neuralnet_amd import training_ops
    if not native:
        monkeypatch.setattr(training_ops, "_calls", None)
    a, b = _randn((8, 8), 1), _randn((5,), 2)
    plan = ext.prepare_adamw([a, b])
    x = _randn((8, 8), 3).requires_grad_()
    y, z = (x @ a).sum(), (x[0, :5] * b).sum()
    versions = a._version, b._version
    plan.step([torch.ones_like(a), None], 1)
    assert a._version > versions[0] and b._version == versions[1]
    z.backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    versions = a._version, b._version
    plan.step([torch.ones_like(a), torch.ones_like(b)], 2)
    plan.step([torch.ones_like(a), torch.ones_like(b)], 3)
    assert a._version >= versions[0] + 2 and b._version >= versions[1] + 2
    with torch.inference_mode():  # tensors without a version
        c = _randn((5,), 4)
        before = c.clone()
        ext.prepare_adamw([c]).step([torch.ones_like(c)], 1)
        assert not torch.equal(c, before)


def test_native_step_enters_no_gradient_of_a_list_it_leaves(ext):
    """A call that is given back to Python has changed nothing, the plan's table among it."""
    from hive_neuralnet_amd import training_ops
    p, g = [_randn((64,), 1), _randn((9,), 2)], [_randn((64,), 3), _randn((9,), 4)]
    plan = ext.prepare_adamw(p)
    plan.step(g, 1)
    held = plan._table.copy()
    for bad in (g[1].double(), g[1].half(), g[1][:4], g[1].cpu(), None):
        assert training_ops._calls.adamw_step(p, [g[0].clone(), bad], plan._table_ptr, 0, 32, 2, 1e-3, 0.9, 0.999, 1e-8,
                                              0.0, None, 0) is None
        assert (plan._table == held).all()


def test_adamw_refuses_codes_at_odd_addresses(ext):
    """Codes are read four at a time: a state of another alignment is refused when the plan is made."""
    p = [_randn((300,), 1)]
    state = ext.prepare_adamw(p, state_bits=8).state
    for key in ("exp_avg", "exp_avg_sq"):
        odd = torch.zeros((513,), dtype=torch.float8_e4m3fn, device="cuda")[1:]
        with pytest.raises(ValueError, match="4-byte aligned"):
            ext.prepare_adamw(p, 8, {**state, key: odd})


# ---- loops that only the widest rows and longest lists take --------------------


@pytest.mark.parametrize("xt,wt,sigmoid", [(F32, F32, False), (BF16, F32, True), (F16, F16, False)],
                         ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("rows,cols,pad", [(130, 16385, 0), (200, 20001, 7)])
def test_layer_norm_many_rows_past_a_block(ext, rows, cols, pad, xt, wt, sigmoid):
    """More rows than there are row ranges, whole and cut from a wider tensor, with and without weight, bias and dx."""
    x = (_randn((rows, cols + pad), 1, 2.0) + 0.5).to(xt)[:, :cols]
    dy = _randn((rows, cols + 2 * pad), 2, 1.0, xt)[:, pad: pad + cols]
    w, b = (1.0 + _randn((cols,), 3, 0.2)).to(wt), _randn((cols,), 4, 0.2, wt)
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        _check_norm(ext, x, weight, bias, dy, sigmoid=sigmoid)
        act = "sigmoid" if sigmoid else None
        _, mean, rstd = ext.layer_norm_forward(x, weight, bias, 1e-5, act)
        _, dw, db = ext.layer_norm_backward(dy, x, mean, rstd, weight, bias, act)
        none, dw2, db2 = ext.layer_norm_backward(dy, x, mean, rstd, weight, bias, act, need_dx=False)
        assert none is None and (dw is None or torch.equal(dw, dw2)) and (db is None or torch.equal(db, db2))


@pytest.mark.parametrize("xt,pt", [(F32, F32), (BF16, F16), (F16, F32)], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("width", [300001, 1200007])
def test_policy_value_loss_longest_lists(ext, width, xt, pt):
    """More slices than a wave has lanes, and slices of two pieces: logits that rise over the list, so that every piece
    has a larger one than those before, lists that the logits' end cuts, and long runs of masked moves.  Element by
    element: a probability is 2 |z| + 4 u of itself off (|z| < 60), sums in chains of under 100 additions."""
    def check(args):
        losses, dx, _ = _check_loss(ext, args)
        _, want, _ = _loss_reference(*args, 0.5, 1.0)
        pi = args[3].double().view(-1)[: len(want)]
        _close(dx, want, 300 * U * (want.abs() + pi), "dlogits")
        return losses, dx

    args = _loss_inputs(2, width, width, xt, pt, 3, full=True)
    args[4].fill_(1.0)
    rise = torch.linspace(-20.0, 20.0, width, device="cuda")
    args[0] = (args[0].float().view(2, width) * 0.1 + torch.stack([rise, rise.flip(0)])).view(-1).to(xt)
    check(args)
    for left in (width + 1, 2 * width - 5000, 2 * width - 100):
        check([args[0][:left].contiguous(), *args[1:]])
    place = torch.arange(width, device="cuda")
    for hide in (place % 4700 < 4200, place < width - 3, place != 5):
        logits, pi = args[0].clone().view(2, width), args[3].clone()
        logits[:, hide] = -math.inf
        pi[:, hide] = 0.0
        losses, dx = check([logits.view(-1), args[1], args[2], pi, *args[4:]])
        assert torch.isfinite(losses).all() and not dx.view(2, width)[:, hide].any()
