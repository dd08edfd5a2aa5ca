"""GPU tests of `rms_norm` at the edges of its shapes and values.  Expectations and tolerances: those of test_gpu_norm.py."""
import pytest
import torch

from test_gpu_norm import DTYPES, EPS, check_plain, check_quantized, data, ops, reference

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


@pytest.mark.parametrize("rows,k", [(1, 16385), (3, 20000), (40, 32768), (300, 24581)])
@pytest.mark.parametrize("dtype,w32,residual", [("bf16", False, True), ("fp16", True, False), ("fp32", True, True)])
def test_rows_of_sixteen_to_thirty_two_thousand(rows, k, dtype, w32, residual):
    """Rows of which a lane holds three and four vectors: every output."""
    x, w = data((rows, k), DTYPES[dtype], rows + k), (data((k,), torch.float32, 3, 0.2) + 1).to(torch.float32 if w32 else DTYPES[dtype])
    r = data((rows, k), DTYPES[dtype], 7, 3.0) if residual else None
    h, exact, y32 = reference(x, w, r)
    for precision in (None, "nvfp4", "fp8e4m3", "int8"):
        got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, residual=None if r is None else r.cuda(), precision=precision)
        if residual:
            assert torch.equal(got[-1].cpu(), h)
        if precision is None:
            check_plain(got[0] if residual else got, exact)
        else:
            check_quantized(got, y32, precision)


@pytest.mark.parametrize("rows,k", [(8, 300), (40, 300), (600, 1040)])
def test_rows_that_are_not_finite_to_nvfp4(rows, k):
    """One scale for all rows: a row with an infinite or a NaN element makes a found one NaN, and with it every row.  With a given scale the rows without
    such elements keep their bits; of the others, NaN rows are NaN, and rows with an infinite element have NaN in its block and zeros elsewhere."""
    x = data((rows, k), torch.bfloat16, 1)
    given = ops().rms_norm(x.cuda(), precision="nvfp4")
    bad = x.clone()
    bad[5, 39] = float("inf")
    bad[6, k - 1] = float("nan")
    q, sf, scale = ops().rms_norm(bad.cuda(), precision="nvfp4")
    assert torch.isnan(scale) and torch.isnan(ops().dequantize(q, sf, scale, cols=k)).all()
    q, sf, scale = ops().rms_norm(bad.cuda(), precision="nvfp4", global_scale=given[2])
    keep = torch.tensor([i for i in range(rows) if i not in (5, 6)], device="cuda")
    assert torch.equal(q[keep], given[0][keep])
    assert torch.equal(sf.view(torch.uint8)[:, keep], given[1].view(torch.uint8)[:, keep])
    d = ops().dequantize(q, sf, scale, cols=k)
    assert torch.isnan(d[6]).all() and torch.isnan(d[5, 32:48]).all()
    assert (d[5, :32] == 0).all() and (d[5, 48:] == 0).all() and torch.isfinite(d[keep]).all()
