"""What a wider network's operators refuse at the ends of their sizes: a
ValueError that names the limit, before anything is allocated or launched."""
import pytest
import torch

from test_gpu_network_ops import ext  # noqa: F401

pytestmark = pytest.mark.gpu


def _wide(rows, cols, dtype=torch.bfloat16):
    """rows x cols of which one row is held."""
    return torch.zeros((1, cols), dtype=dtype, device="cuda").expand(rows, cols)


def test_more_matrices_than_a_launch_takes(ext):  # noqa: F811
    u = torch.ones((1, 8, 8), device="cuda")
    for count, rows, cols in ((65537, 8, 8), (70000, 8, 8), (2, 1 << 17, 1 << 17), (65000, 64, 2100)):
        wide = torch.zeros((1, 1, cols), device="cuda").expand(count, rows, cols)
        with pytest.raises(ValueError, match="at most 65536 matrices"):
            ext.orthogonalize(wide)
    out = ext.orthogonalize(u.expand(65536, 8, 8))
    assert torch.equal(out[0], ext.orthogonalize(u)[0]) and bool((out == out[0]).all())


def test_gated_blocks_past_a_launch(ext):  # noqa: F811
    one = _wide(1, 1).contiguous()
    for rows, cols, hidden in ((1 << 20, (1 << 15) + 8, 1), (1 << 18, 8, (1 << 17) + 1)):
        x = _wide(rows, cols)
        w = torch.zeros((hidden, cols), dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match="each two of them"):
            ext.gated_linear(x, w, w)
        with pytest.raises(ValueError, match="each two of them"):
            ext.gated_linear_forward(x, w, w)
        with pytest.raises(ValueError, match="each two of them"):
            ext.gated_linear_backward(one, x, w, w, one, one)


def test_more_rows_than_a_launch_draws_from(ext):  # noqa: F811
    u = torch.zeros((1,), device="cuda")
    for rows, width in (((1 << 25) + 1, 4), ((1 << 21) + 1, 1025)):
        x, numbers = _wide(rows, width), torch.zeros((rows,), device="cuda")
        with pytest.raises(ValueError, match="at most"):
            ext.sample_actions(x, numbers)
    assert ext.sample_actions(_wide(1, 1025), u)[0].item() == 0
