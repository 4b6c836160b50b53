"""Calls of the long-sequence operators at the edge of what they take: refused on the host, or right on the GPU."""
import pytest
import torch


def test_weight_gradients_of_too_many_columns_are_refused_by_the_launchers():
    """A tile's column number is 16 bits: past 32767 tiles of 128 columns it would wrap around to addresses before the gradient."""
    from mitune.ops import lib as L
    so = L.load()
    for wide in (32767 * 128 + 8, 5_000_000):
        assert so.mt_linear_wgrad_launch(16, 16, 16, None, 8, 8, wide, 8, wide, 1, 1, None) == -2
        assert so.mt_wgrad_single_launch(16, 16, 16, None, 8, 8, wide, 1, 8 * wide + 8, None) == -2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_of_too_many_features_are_refused_before_they_run(dtype):
    from mitune.ops import linear as M
    from mitune.ops.linear import _fused_linear
    wide = M.MAX_FUSED_WIDTH + 8
    new = lambda *s: torch.empty(*s, device="meta", dtype=dtype)          # noqa: E731
    with pytest.raises(ValueError, match="features"):
        _fused_linear(new(4, 8), new(wide, 8), None, None, None)
    with pytest.raises(ValueError, match="features"):
        _fused_linear(new(4, wide).requires_grad_(), new(8, wide), None, "relu", None)
    if dtype == torch.bfloat16:
        wide = M.MAX_BF16_DW_WIDTH + 8
        with pytest.raises(ValueError, match="features"):
            _fused_linear(new(4, wide), new(8, wide).requires_grad_(), None, "relu", None)
