"""Slots drawn from rows of logits, at the ends of their settings: NaN among a
row's own.
References and tolerances: test_gpu_network_ops.py."""
import math

import pytest
import torch

from test_gpu_network_ops import TYPES, _check_sample, _logits, _uniforms, ext  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("K", [200, 1024, 5000])
def test_nan_in_the_settings_of_a_row(ext, K, t):  # noqa: F811
    """A NaN temperature takes the largest, a NaN top_p or min_p leaves all, with the first slot masked."""
    B = 6
    x, u = _logits(B, K, 3, t), _uniforms(B, 4)
    x[:, 0] = -math.inf
    nan = torch.tensor([float("nan"), 0.7, float("nan"), 0.9, float("nan"), 0.2], device="cuda")

    def settled(value):
        return torch.where(nan.isnan(), torch.full_like(nan, value), nan)

    for kw in (dict(), dict(k=9), dict(p=0.8)):
        _same(ext, x, u, {**kw, "t": nan}, {**kw, "t": settled(0.0)})
        _same(ext, x, u, {**kw, "min_p": nan}, {**kw, "min_p": settled(0.0)})
    for kw in (dict(), dict(k=1200), dict(min_p=0.01)):
        _same(ext, x, u, {**kw, "p": nan}, {**kw, "p": settled(1.0)})


def _same(ext, x, u, settings, meaning):  # noqa: F811
    """The draw by `settings` is what `meaning` says, which is checked against the definition."""
    names = {"t": "temperature", "k": "top_k", "p": "top_p", "min_p": "min_p"}
    got, want = (ext.sample_actions(x, u, **{names[k]: v for k, v in kw.items()}) for kw in (settings, meaning))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check_sample(ext, x, u, **meaning)
