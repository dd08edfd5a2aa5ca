"""Arguments of another kind or rank than the operators take: a RuntimeError that says so, as for every other refusal."""
import pytest
import torch


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def test_grouped_linear_without_an_output():
    x, sf, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(())
    w, wsf, off = torch.zeros((1, 8, 32), dtype=torch.uint8), torch.zeros((1, 1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(weight=w[0]), dict(weight=w[0, 0]), dict(weight=w.tolist()), dict(x=x[0]), dict(x=x.tolist()), dict(x=None),
                dict(rows=torch.zeros((), dtype=torch.int32)), dict(rows=[0, 1, 2, 3])):
        args = dict(x=x, x_scale=sf, x_global_scale=s, weight=w, weight_scale=wsf, weight_global_scale=s, offsets=off)
        with pytest.raises(RuntimeError):
            ops().grouped_linear(**{**args, **bad})


def test_residual_that_is_no_tensor():
    with pytest.raises(RuntimeError, match="residual"):
        ops().rms_norm(torch.zeros((4, 64), dtype=torch.bfloat16), residual=1.0)


@pytest.mark.gpu
def test_norm_operands_that_are_no_tensors():
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    for kw in (dict(precision="nvfp4", global_scale=0.01), dict(out=[1.0]), dict(residual=x, residual_out=1.0), dict(weight=[1.0] * 64),
               dict(precision="nvfp4", global_scale=torch.zeros((), device="cuda", dtype=torch.float64))):
        with pytest.raises(RuntimeError):
            ops().rms_norm(x, **kw)
