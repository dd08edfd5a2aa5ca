"""The operators of the feed-forward half of a layer in a row, as a model calls them: with experts (norm of the attention block's output into the residual,
routing, linears grouped by expert, the rows back to their tokens, the norm in front of the next block) and dense (layer norm with modulation, linear with an
activation, linear with the residual), eager and captured."""
import pytest
import torch

from conftest import make_input

pytestmark = pytest.mark.gpu


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def deq(q):
    return ops().dequantize(*q, dtype=torch.float32).double()


def weight(*shape, seed):
    return ops().quantize(make_input(shape, seed=seed, std=0.06).cuda(), len(shape) - 2, len(shape) - 1)


def near(y, exact):
    """One bf16 rounding, and what sums in 32 bits lose next to the largest value."""
    assert ((y.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + exact.abs().max() * 2.0 ** -13).all()


def normed(h, kind="rms"):
    h = h.double()
    if kind == "layer":
        h = h - h.mean(-1, keepdim=True)
    return h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt()


@pytest.mark.parametrize("tokens", [1, 16, 96, 700])
def test_with_experts(tokens):
    """Step by step on the kernels' own output of the step before, so that every comparison is that of one operator."""
    hidden, experts, topk = 256, 16, 3
    o, x = make_input((tokens, hidden), seed=1).cuda(), make_input((tokens, hidden), seed=2).cuda()
    post, pre, gate = ((1 + make_input((hidden,), seed=s, std=0.1)).cuda() for s in (3, 4, 5))
    router, bias = (make_input((hidden, experts), seed=6, std=0.1).float().cuda(), make_input((experts,), seed=7, std=0.1).float().cuda())
    up, down = weight(experts, 512, hidden, seed=8), weight(experts, hidden, 512, seed=9)
    padded = tokens // 8   # tokens behind the sequence

    # the block's output, normed, gated, into the residual; its norm for the experts' linears, and once more as it is for the router
    *xq, h = ops().block_norm(o, x, pre, gate=gate, residual_scale=0.9, post_weight=post, precision="nvfp4")
    near(h, 0.9 * x.double() + normed(o) * post.double() * gate.double())
    z = ops().block_norm(h, weight=pre)
    near(z, normed(h) * pre.double())
    logits = z.float() @ router
    logits[tokens - padded:] = -torch.inf
    weights, chosen, offsets, rows, places = ops().route_experts(logits, topk, scoring="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2, scale=2.0)
    assert offsets[-1] == (tokens - padded) * topk and (chosen[tokens - padded:] == -1).all()
    e = torch.repeat_interleave(torch.arange(experts, device="cuda"), offsets.diff())
    met = e.numel()

    a = ops().grouped_linear(*xq, *up, offsets, rows=rows)
    near(a[:met], torch.bmm(deq(up)[e], deq(xq)[rows[:met].long()].unsqueeze(2)).squeeze(2))
    assert (a[met:] == 0).all()
    q = ops().quantize(torch.nn.functional.silu(a), 0, 1)
    y = ops().grouped_linear(*q, *down, offsets)
    near(y[:met], torch.bmm(deq(down)[e], deq(q)[:met].unsqueeze(2)).squeeze(2))
    out = ops().combine_experts(y, weights, places, residual=h)
    exact = h.double()
    for s in range(topk):
        part = y.double()[places[:, s].long().clamp(min=0)] * weights[:, s, None].double()
        exact = exact + torch.where(places[:, s, None] >= 0, part, 0.0)
    near(out, exact)
    assert torch.equal(out[tokens - padded:], h[tokens - padded:])
    assert torch.allclose(weights[:tokens - padded].sum(1), torch.full((tokens - padded,), 2.0, device="cuda"), rtol=1e-6)


@pytest.mark.parametrize("batch,tokens", [(1, 1), (2, 40), (3, 150)])
@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh"])
def test_dense(batch, tokens, activation):
    hidden, wide = 384, 1024
    x = make_input((batch, tokens, hidden), seed=1).cuda()
    attention = make_input((batch, tokens, hidden), seed=2).cuda()
    shift, scale, gate = make_input((batch, 3, hidden), seed=3, std=0.3).cuda().chunk(3, dim=1)
    up, down = weight(wide, hidden, seed=4), weight(hidden, wide, seed=5)
    b_up, b_down = make_input((wide,), seed=6).cuda(), make_input((hidden,), seed=7).cuda()
    *xq, h = ops().block_norm(attention, x, gate=gate, scale=scale, shift=shift, kind="layer", precision="nvfp4")
    near(h, x.double() + gate.double() * attention.double())
    z = normed(h, "layer") * (1 + scale.double()) + shift.double()
    assert (deq(xq).reshape(z.shape) - z).norm() <= 0.13 * z.norm()      # e2m1
    a = ops().linear(*xq, *up, bias=b_up, activation=activation)
    v = deq(xq) @ deq(up).t() + b_up.double()
    near(a, v * torch.special.ndtr(v) if activation == "gelu" else v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
    q = ops().quantize(a, 0, 1)
    flat = h.reshape(-1, hidden)
    y = ops().linear(*q, *down, bias=b_down, residual=flat)
    near(y, deq(q) @ deq(down).t() + b_down.double() + flat.double())


def test_captured_with_experts():
    tokens, hidden, experts, topk = 64, 256, 8, 2
    up, down = weight(experts, 512, hidden, seed=8), weight(experts, hidden, 512, seed=9)
    o, x, logits = make_input((tokens, hidden), seed=1).cuda(), make_input((tokens, hidden), seed=2).cuda(), torch.randn((tokens, experts), device="cuda")

    def layer():
        *xq, h = ops().block_norm(o, x, precision="nvfp4")
        weights, _, offsets, rows, places = ops().route_experts(logits, topk)
        a = ops().grouped_linear(*xq, *up, offsets, rows=rows)
        y = ops().grouped_linear(*ops().quantize(torch.nn.functional.silu(a), 0, 1), *down, offsets)
        return ops().combine_experts(y, weights, places, residual=h)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for seed in range(4):
        o.copy_(make_input((tokens, hidden), seed=seed + 20))
        logits.normal_()
        logits[5 * seed:5 * seed + 3] = -torch.inf
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, layer())
