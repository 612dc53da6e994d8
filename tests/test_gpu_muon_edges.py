"""Orthogonalised updates of matrices far smaller than eps, and of float32's
smallest, coefficients that shrink, the optimizer's settings.  Definition and
tolerances: test_gpu_network_ops.py."""
import math

import pytest
import torch

from test_gpu_network_ops import ABC, F32, U, _check_orthogonal, _iteration, _muon_reference, _randn, ext  # noqa: F401

pytestmark = pytest.mark.gpu


def _relative(rows, cols, steps):
    """Where |X| stays far below 1, a step is X <- a X but for what rounds: X, A and P held in 22 bits (2^-22 each of the
    value, 2^-38 of 1 a value, |X| being held at 1/8 and more), the sum of P's and X's products ((3 K / 16 + 80) u, K the
    shorter side), and X and the result in float32 at both ends."""
    short, long = min(rows, cols), max(rows, cols)
    return steps * ((3 * short / 16 + 80) * U + 3 * 2.0 ** -22 + 2.0 ** -35 * math.sqrt(short * long) + 2.0 ** -35 * short) + 8 * U


@pytest.mark.parametrize("size", [1e-9, 1e-11, 1e-12, 1e-14, 1e-16, 1e-22])
@pytest.mark.parametrize("rows,cols", [(1, 1), (40, 33), (64, 200), (300, 129), (500, 700)])
def test_far_below_eps(ext, rows, cols, size):  # noqa: F811
    """X = U / (|U| + eps) is held as exactly where |U| is far below eps as where it is not."""
    u = _randn((rows, cols), rows, size / math.sqrt(rows * cols))
    want, _ = _iteration(u)
    got = ext.orthogonalize(u)
    # X grows 3.4445 times a step: to 485 |U| / eps in five
    assert 300 * size / 1e-7 < float(want.norm()) < 700 * size / 1e-7 or size > 1e-10 or rows * cols == 1
    assert float((got.double() - want).norm()) <= _relative(rows, cols, 5) * float(want.norm())


@pytest.mark.parametrize("rows,cols", [(40, 33), (300, 129)])
def test_between_eps_and_one(ext, rows, cols):  # noqa: F811
    """Sizes at which the iteration leaves its straight part after one, two, ... steps; more steps; other coefficients."""
    for i in range(12):
        u = _randn((rows, cols), i, 10.0 ** (-10 + 0.5 * i) / math.sqrt(rows * cols))
        _check_orthogonal(ext.orthogonalize(u), u)
    u = _randn((rows, cols), 20, 1e-13 / math.sqrt(rows * cols))
    for steps in (1, 2, 9, 14):
        _check_orthogonal(ext.orthogonalize(u, steps=steps), u, steps)
    want, _ = _iteration(u, 3, (0.25, 0.5, 0.1))  # shrinks
    got = ext.orthogonalize(u, steps=3, coefficients=(0.25, 0.5, 0.1))
    assert float((got.double() - want).norm()) <= _relative(rows, cols, 3) * float(want.norm())


def test_a_batch_of_all_sizes(ext):  # noqa: F811
    """Each matrix by its own size."""
    for shape in ((9, 30, 50), (9, 130, 300)):
        sizes = torch.logspace(-18, 0, 9, device="cuda")
        u = _randn(shape, 4, 1.0 / math.sqrt(shape[1] * shape[2])) * sizes.view(-1, 1, 1)
        got = ext.orthogonalize(u)
        for one, g, size in zip(u, got, sizes.tolist()):
            if size < 1e-10:
                want, _ = _iteration(one)
                assert float((g.double() - want).norm()) <= _relative(*shape[1:], 5) * float(want.norm())
            else:
                _check_orthogonal(g, one)


@pytest.mark.parametrize("rows,cols", [(20, 30), (200, 300)])
def test_the_smallest_floats(ext, rows, cols):  # noqa: F811
    """Matrices whose size is under 2^13 / float's largest, and of subnormal values, with an eps of 0."""
    for size in (1e-36, 1e-38, 1e-42):
        u = _randn((rows, cols), 3, size)
        assert bool(u.any())
        _check_orthogonal(ext.orthogonalize(u, eps=0.0), u, eps=0.0)
    u = _randn((rows, cols), 3, 1e37)
    _check_orthogonal(ext.orthogonalize(u, eps=0.0), u, eps=0.0)


def test_a_step_with_gradients_far_below_eps(ext):  # noqa: F811
    params = [_randn(s, i, 1e-6) for i, s in enumerate([(64, 122), (200, 300)])]
    before = [p.clone() for p in params]
    grads = [_randn(p.shape, 9 + i, 1e-15 / math.sqrt(p.numel())) for i, p in enumerate(params)]
    ext.prepare_muon(params).step(grads, lr=1.0, momentum=0.0)
    for p, b, g in zip(params, before, grads):
        want, _, _ = _muon_reference(b, g, torch.zeros_like(b), 1.0, 0.0, True, 0.0, "spectral")
        moved = float((want - b.double()).norm())
        off = float((p.double() - want).norm())
        assert off <= 1.01 * _relative(*p.shape, 5) * moved + U * float(want.norm()) + 2 * U * float(b.norm()), (off, moved)


def test_a_saved_state_with_settings_out_of_range(ext):  # noqa: F811
    """load_state_dict refuses what the constructor does, and leaves the optimizer as it was."""
    from hive_neuralnet_amd.training import Muon
    p = _randn((20, 12), 1).requires_grad_()
    opt = Muon([p], lr=0.1)
    p.grad = _randn((20, 12), 2)
    opt.step()
    saved = opt.state_dict()
    held = [m.clone() for m in saved["momentum"][0]]
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(steps=0), dict(steps=101), dict(eps=float("nan")), dict(weight_decay=-1)):
        state = {**saved, "momentum": [[torch.zeros_like(m) for m in held]],
                 "param_groups": [{**saved["param_groups"][0], "lr": 0.5, **bad}]}
        with pytest.raises(ValueError):
            opt.load_state_dict(state)
        assert opt.param_groups[0]["lr"] == 0.1 and all(torch.equal(a, b) for a, b in zip(opt.state_dict()["momentum"][0], held))
    opt.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], "lr": 0.5}]})
    assert opt.param_groups[0]["lr"] == 0.5


def test_an_optimizer_with_coefficients_of_its_own(ext):  # noqa: F811
    """A group's coefficients are those of MuonPlan.step, and go through a saved state; a state saved without them leaves them."""
    from hive_neuralnet_amd.training import Muon
    schedule = [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375)]
    p, q = (_randn((20, 12), 1).requires_grad_() for _ in range(2))
    opt = Muon([{"params": [p], "coefficients": schedule}], lr=0.1)
    plan = ext.prepare_muon([q.detach()])
    p.grad = _randn((20, 12), 2)
    for _ in range(2):
        opt.step()
        plan.step([p.grad], lr=0.1, coefficients=schedule)
    assert torch.equal(p.detach(), q.detach())
    saved = opt.state_dict()
    other = Muon([_randn((20, 12), 1).requires_grad_()])
    other.load_state_dict(saved)
    assert other.param_groups[0]["coefficients"] == schedule
    older = {**saved, "param_groups": [{k: v for k, v in g.items() if k != "coefficients"} for g in saved["param_groups"]]}
    other = Muon([_randn((20, 12), 1).requires_grad_()])
    other.load_state_dict(older)
    assert other.param_groups[0]["coefficients"] == ABC
    for bad in ((1.0, 2.0), [], "abc", [(1.0, 2.0, 3.0), (1.0,)]):
        with pytest.raises(ValueError):
            Muon([_randn((20, 12), 1).requires_grad_()], coefficients=bad)


@pytest.mark.parametrize("rows,cols", [(40, 33), (300, 129)])
@pytest.mark.parametrize("size", [1.0, 1e-12])
def test_coefficients_that_shrink(ext, rows, cols, size):  # noqa: F811
    """Steps that take X down tenfold each: it is held to its own size on the way, and given at it."""
    u = _randn((rows, cols), 5, size / math.sqrt(rows * cols))
    for triple in ((0.1, 0.05, 0.01), (0.1, 0.0, 0.0), (1e-5, 0.0, 0.0)):
        want, _ = _iteration(u, 6, triple)
        got = ext.orthogonalize(u, steps=6, coefficients=triple)
        assert float(want.norm()) < 1e-5
        # X's rounding is passed on by each step; b A + c A A is a tenth of P at most: half more than where it is next to none
        assert float((got.double() - want).norm()) <= 1.5 * _relative(rows, cols, 6) * float(want.norm())
    assert not ext.orthogonalize(u, steps=3, coefficients=(0.0, 0.0, 0.0)).any()
    many = [(0.1, 0.05, 0.01)] * 20  # more of them than the kernel of small matrices takes
    want, _ = _iteration(u, 20, many)
    got = ext.orthogonalize(u, steps=20, coefficients=many)
    assert float((got.double() - want).norm()) <= 1.5 * _relative(rows, cols, 20) * float(want.norm())


def test_a_pickle_without_coefficients(ext):  # noqa: F811
    """One made before they were a setting steps as it did."""
    from hive_neuralnet_amd.training import Muon
    p = _randn((20, 12), 1).requires_grad_()
    opt = Muon([p], lr=0.1)
    state = opt.__getstate__()
    state["param_groups"] = [{k: v for k, v in g.items() if k != "coefficients"} for g in state["param_groups"]]
    other = Muon.__new__(Muon)
    other.__setstate__(state)
    p.grad = _randn((20, 12), 2)
    before = p.detach().clone()
    other.step()
    want, _, error = _muon_reference(before, p.grad, torch.zeros_like(before), 0.1, 0.95, True, 0.0, "spectral")
    assert float((p.detach().double() - want).norm()) <= error + 4 * U * float(want.norm() + 8)


def test_gradients_of_other_kinds(ext):  # noqa: F811
    """Any sequence of them is taken; what is no dense tensor is refused before anything is written."""
    params = [_randn((20, 12), i) for i in range(2)]
    plan = ext.prepare_muon(params)
    before = [p.clone() for p in params]
    g = _randn((20, 12), 5)
    for bad in (1.0, "g", g.tolist(), g.cpu().numpy(), g.to_sparse()):
        with pytest.raises(ValueError):
            plan.step([g, bad])
        with pytest.raises(ValueError):
            plan.step([bad, None])
    assert all(torch.equal(a, b) for a, b in zip(params, before)) and not any(m.any() for m in plan.momentum)
    plan.step(x for x in (g, None))
    assert not torch.equal(params[0], before[0]) and torch.equal(params[1], before[1])
