"""The kinds of numbers that a wider network's operators take as settings, the
same whether the native call module takes the call or Python does."""
import decimal
import fractions

import numpy as np
import pytest
import torch

from hive_neuralnet_amd import network_ops
from test_gpu_network_ops import _logits, _randn, _uniforms, ext  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def calls(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(network_ops, "_calls", None)
    elif network_ops._calls is None:
        pytest.skip("_train_calls.so is not built")


def test_draws_take_any_kind_of_number(ext, calls):  # noqa: F811
    x, u = _logits(7, 60, 1), _uniforms(7, 2)
    want = ext.sample_actions(x, u, temperature=0.5, top_k=9, top_p=0.75, min_p=0.125)
    for real, whole in ((np.float32, np.int32), (np.float64, np.int64), (np.float16, np.uint8), (fractions.Fraction, int)):
        got = ext.sample_actions(x, u, temperature=real(0.5), top_k=whole(9), top_p=real(0.75), min_p=real(0.125))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), real
    assert torch.equal(ext.sample_actions(x, u, temperature=1, top_p=1, min_p=0)[0], ext.sample_actions(x, u)[0])
    for name in ("temperature", "top_k", "top_p", "min_p"):
        for bad in ("1", None, [1.0], decimal.Decimal(1), np.ones(1), 1j, np.float32("nan") if name != "top_k" else 1.0, -1):
            with pytest.raises(ValueError):
                ext.sample_actions(x, u, **{name: bad})
    for name in ("temperature", "top_p"):
        with pytest.raises(ValueError):
            ext.sample_actions(x, u, **{name: 10 ** 400})
    assert torch.equal(ext.sample_actions(x, u, top_k=10 ** 400)[0], ext.sample_actions(x, u)[0])


def test_iterations_take_any_kind_of_number(ext):  # noqa: F811
    u = _randn((20, 30), 1)
    want = ext.orthogonalize(u, steps=3, coefficients=(2.0, -1.5, 0.5), eps=0.25)
    for triple in (np.array([2.0, -1.5, 0.5], dtype=np.float32), [np.float32(2.0), fractions.Fraction(-3, 2), 0.5],
                   np.array([[2.0, -1.5, 0.5]]), (t for t in [(2, -1.5, 0.5)])):
        assert torch.equal(ext.orthogonalize(u, steps=np.int64(3), coefficients=triple, eps=np.float32(0.25)), want)
    for kw in (dict(steps=2.5), dict(steps="3"), dict(steps=None), dict(eps="x"), dict(eps=None), dict(coefficients=None),
               dict(coefficients=3.0), dict(coefficients=("a", "b", "c")), dict(coefficients=[(1.0, 2.0, None)]),
               dict(coefficients=[1.0, 2.0, (3.0,)])):
        with pytest.raises(ValueError):
            ext.orthogonalize(u, **kw)
    params = [_randn((20, 30), 2) for _ in range(2)]
    plans = [ext.prepare_muon([p]) for p in params]
    plans[0].step([u], lr=0.5, momentum=0.25, weight_decay=0.125)
    plans[1].step([u], lr=np.float32(0.5), momentum=np.float16(0.25), weight_decay=fractions.Fraction(1, 8))
    assert not torch.equal(params[0], _randn((20, 30), 2)) and torch.equal(*params)
    for kw in (dict(lr=None), dict(momentum="1"), dict(weight_decay=torch.ones(2, device="cuda"))):
        with pytest.raises(ValueError):
            plans[0].step([u], **kw)
    assert torch.equal(*params)
