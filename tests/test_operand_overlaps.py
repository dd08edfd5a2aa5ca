"""Outputs that share memory with an operand: refused where another workgroup could still read what one has overwritten, accepted where they only touch.
Operands are laid into a buffer of bytes, the output over their first or last ones, or right beside them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
AT = 4096  # of the operand in its buffer


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def laid(t):
    """(buffer of bytes, copy of t at AT in it, bytes of t)"""
    n = t.numel() * t.element_size()
    buf = torch.zeros(3 * AT + n, dtype=torch.uint8, device="cuda")
    copy = buf[AT:AT + n].view(t.dtype).reshape(t.shape)
    copy.copy_(t)
    return buf, copy, n


def at(buf, first, shape, dtype):
    n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    return buf[first:first + n].view(dtype).reshape(shape)


def around(t, shape, dtype):
    """Copy of t, outputs of shape over its first and its last element, and outputs right in front of it and behind it."""
    buf, copy, n = laid(t)
    size = torch.empty((), dtype=dtype).element_size()
    out = math.prod(shape) * size
    step = -(-n // size) * size
    meet = [at(buf, AT + size - out, shape, dtype), at(buf, AT + (n - 1) // size * size, shape, dtype)]
    return copy, meet, [at(buf, AT - out, shape, dtype), at(buf, AT + step, shape, dtype)]


def test_grouped_linear():
    x = ops().quantize(torch.ones((6, 64), dtype=torch.bfloat16, device="cuda"), 0, 1)
    w = ops().quantize(torch.ones((2, 4, 64), dtype=torch.bfloat16, device="cuda"), 1, 2)
    args = {"x": x[0], "x_scale": x[1], "x_global_scale": x[2], "weight": w[0], "weight_scale": w[1], "weight_global_scale": w[2],
            "offsets": torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda"), "rows": torch.arange(6, dtype=torch.int32, device="cuda"),
            "bias": torch.ones((2, 4), dtype=torch.bfloat16, device="cuda")}
    want = ops().grouped_linear(**args)
    for name, t in args.items():
        copy, meet, beside = around(t, (6, 4), torch.bfloat16)
        for out in meet:
            with pytest.raises(RuntimeError, match="overlap"):
                ops().grouped_linear(**{**args, name: copy}, out=out)
        for out in beside:
            assert torch.equal(ops().grouped_linear(**{**args, name: copy}, out=out), want)


def test_rope():
    table, pos = ops().rope_table(8, 12), torch.arange(10, dtype=torch.int32, device="cuda").reshape(1, 2, 5)
    for dtype in (torch.bfloat16, torch.float32):
        q, k = (torch.ones((2, 5, h, 16), dtype=dtype, device="cuda") for h in (3, 1))
        want = ops().rope((q, k), table, positions=pos)
        for name, t in (("table", table), ("positions", pos), ("positions", pos.long())):
            args = {"table": table, "positions": pos}
            for x, y in ((q, want[0]), (k, want[1])):
                copy, meet, beside = around(t, x.shape, dtype)
                for out in meet:
                    with pytest.raises(RuntimeError, match="overlap"):
                        ops().rope(x, **{**args, name: copy}, out=out)
                    with pytest.raises(RuntimeError, match="overlap"):  # the second of a pair
                        ops().rope((q, x), **{**args, name: copy}, out=(torch.empty_like(q), out))
                for out in beside:
                    assert torch.equal(ops().rope(x, **{**args, name: copy}, out=out), y)


@pytest.mark.parametrize("precision", ["nvfp4", "fp8e4m3", "int8"])
def test_dequantize(precision):
    quantized = ops().rms_norm(torch.ones((5, 64), dtype=torch.bfloat16, device="cuda"), precision=precision)
    want = ops().dequantize(*quantized)
    for i, t in enumerate(quantized):
        copy, meet, beside = around(t, want.shape, want.dtype)
        operands = [copy if j == i else u for j, u in enumerate(quantized)]
        for out in meet:
            with pytest.raises(RuntimeError, match="overlap"):
                ops().dequantize(*operands, out=out)
        for out in beside:
            assert torch.equal(ops().dequantize(*operands, out=out), want)


def test_norm_with_a_given_scale():
    x = torch.ones((5, 64), dtype=torch.bfloat16, device="cuda")
    scale = torch.tensor(0.01, device="cuda")
    want = ops().rms_norm(x, residual=x, precision="nvfp4", global_scale=scale)
    copy, meet, beside = around(scale, x.shape, x.dtype)
    for out in meet:
        with pytest.raises(RuntimeError, match="overlap"):
            ops().rms_norm(x, residual=x, residual_out=out, precision="nvfp4", global_scale=copy)
    for out in beside:
        got = ops().rms_norm(x, residual=x, residual_out=out, precision="nvfp4", global_scale=copy)
        assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


def test_columns_of_one_buffer():
    """Inputs and outputs that are slices of the same rows share nothing and are taken."""
    wide = torch.randn((33, 5, 3, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    rows = wide.reshape(165, 192)
    x, y, z = rows[:, :64], rows[:, 64:128], rows[:, 128:]
    want = ops().rms_norm(x.clone(), residual=z.clone())
    assert ops().rms_norm(x, residual=z, residual_out=z, out=y)[0] is y
    assert torch.equal(y, want[0]) and torch.equal(z, want[1])
    table = ops().rope_table(32, 8)
    turned = ops().rope(x.clone().reshape(33, 5, 1, 64), table)
    assert torch.equal(ops().rope(wide[:, :, :1], table, out=wide[:, :, 1:2]), turned)
    with pytest.raises(RuntimeError, match="overlap"):
        ops().rms_norm(x, out=rows[:, 63:127])


def test_outputs_without_elements():
    x, outs = torch.empty((2, 0, 64), device="cuda"), [torch.empty((2, 0, 64), device="cuda") for _ in range(2)]
    assert ops().rms_norm(x, residual=x, residual_out=outs[0], out=outs[1])[0] is outs[1]
