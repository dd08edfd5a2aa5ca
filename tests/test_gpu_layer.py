"""The operators of a transformer layer in a row, as a model calls them: norm with a quantized output, linear, rotary positions, attention,
linear, norm with the residual's addition, routing to experts."""
import pytest
import torch

from conftest import make_input

pytestmark = pytest.mark.gpu


def test_layer_with_experts():
    """Against the same layer in 64 bits on the values that the quantized tensors stand for, step by step: each step takes the kernels' own
    output of the step before, so that every comparison is that of one operator (tolerances: one bf16 rounding and sums in 32 bits)."""
    from ac4k_kernel_amd import ops
    tokens, heads, dim, hidden, experts, topk = 96, 4, 64, 256, 4, 2
    deq = lambda q, **kw: ops.dequantize(*q, dtype=torch.float32, **kw).double()
    weight = lambda *shape, seed: ops.quantize(make_input(shape, seed=seed, std=0.06).cuda(), len(shape) - 2, len(shape) - 1)
    x, res = make_input((tokens, hidden), seed=1).cuda(), make_input((tokens, hidden), seed=2).cuda()
    n1, n2 = ((1 + make_input((hidden,), seed=s, std=0.1)).cuda() for s in (3, 4))
    w_qkv, w_o = weight(3 * hidden, hidden, seed=5), weight(hidden, hidden, seed=6)
    w_up, w_down = weight(experts, 512, hidden, seed=7), weight(experts, hidden, 512, seed=8)

    def near(y, exact):
        assert ((y.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + exact.abs().max() * 2.0 ** -13).all()

    *xq, h = ops.rms_norm(x, n1, residual=res, precision="nvfp4")
    assert torch.equal(h, (x.float() + res.float()).bfloat16())
    qkv = ops.linear(*xq, *w_qkv)
    near(qkv, deq(xq) @ deq(w_qkv).t())
    q, k, v = qkv.reshape(1, tokens, 3, heads, dim).unbind(2)
    sections = (12, 10, 10)
    table = ops.rope_table(sections, 16)
    q, k = ops.rope((q, k), table, grid=(4, 4, 6), sections=sections)
    o = ops.attention(q, k, v.contiguous(), layout="BNHD")
    s = torch.einsum("bnhd,bmhd->bhnm", q.double(), k.double()) / dim ** 0.5
    exact = torch.matmul(s.softmax(-1), v.double().transpose(1, 2)).transpose(1, 2)
    assert (o.double() - exact).norm() <= 0.06 * exact.norm()  # 8-bit probabilities, keys, values: the precision of that operator
    a = ops.linear(*ops.quantize(o.reshape(tokens, hidden), 0, 1), *w_o)
    *xq, h = ops.rms_norm(a, n2, residual=h, residual_out=h, precision="nvfp4")
    scores = torch.randn((tokens, experts), generator=torch.Generator().manual_seed(9)).cuda()
    gate, chosen = scores.softmax(-1).topk(topk)
    order = chosen.reshape(-1).argsort(stable=True)
    rows = (order // topk).to(torch.int32)
    offsets = torch.nn.functional.pad(torch.bincount(chosen.reshape(-1), minlength=experts).cumsum(0), (1, 0)).to(torch.int32)
    up = ops.grouped_linear(*xq, *w_up, offsets, rows=rows)
    e = chosen.reshape(-1)[order]
    near(up, torch.bmm(deq(w_up)[e], deq(xq)[rows.long()].unsqueeze(2)).squeeze(2))
    act = ops.quantize(torch.nn.functional.silu(up), 0, 1)
    down = ops.grouped_linear(*act, *w_down, offsets)
    near(down, torch.bmm(deq(w_down)[e], deq(act).unsqueeze(2)).squeeze(2))
    y = torch.zeros((tokens, hidden), device="cuda").index_add_(0, rows.long(), down.float() * gate.reshape(-1)[order, None])
    assert torch.isfinite(y).all() and torch.isfinite(h.float()).all()
