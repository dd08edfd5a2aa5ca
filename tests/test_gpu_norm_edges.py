"""GPU tests of `rms_norm` at the edges of its shapes and values.  Expectations and tolerances: those of test_gpu_norm.py."""
import pytest
import torch

from test_gpu_norm import ops

pytestmark = pytest.mark.gpu


def test_scale_of_no_rows():
    """The scale of a tensor without rows is that of one of zeros, whatever its memory held before; a given one stays."""
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        junk = torch.full((), float("nan"), device="cuda")
        del junk
        q, sf, scale, h = ops().rms_norm(x, residual=x, precision="nvfp4")
        assert q.shape == (0, 32) and sf.shape == (1, 0, 4) and scale.item() == 0 and h.shape == (0, 64)
    given = torch.tensor(0.5, device="cuda")
    assert ops().rms_norm(x, precision="nvfp4", global_scale=given)[2].item() == 0.5
    assert ops().dequantize(q, sf, scale).shape == (0, 64)
