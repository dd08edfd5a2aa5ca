"""GPU tests of routing, the return of the experts' rows, the block norm and the linear with an epilogue on operands of more than 2^32 elements: the last rows
against the same call on these rows alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    from ac4k_kernel_amd import ops as o
    return o


@pytest.fixture(autouse=True)
def release():
    yield
    torch.cuda.empty_cache()


def noise(shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))


def test_route():
    t, e, k = 35_000_000, 128, 2  # 4.5e9 logits
    x = noise((t, e))
    weights, experts, offsets, rows, places = ops().route_experts(x, k)
    last = ops().route_experts(x[-48:], k)
    assert torch.equal(weights[-48:], last[0]) and torch.equal(experts[-48:], last[1])
    del x
    count = torch.bincount(experts.view(-1), minlength=e)
    assert torch.equal(offsets.long(), torch.nn.functional.pad(count.cumsum(0), (1, 0))) and offsets[-1] == t * k
    assert torch.equal(rows[places.long().view(-1)].view(t, k), torch.arange(t, device="cuda", dtype=torch.int32)[:, None].expand(t, k))
    for expert in (0, 77, e - 1):  # tokens of an expert in rising order
        assert (rows[offsets[expert]:offsets[expert + 1]].diff() > 0).all()
        assert (experts[rows[offsets[expert]:offsets[expert + 1]].long()] == expert).any(1).all()


def test_combine():
    m, n, k = 600_000, 8192, 8  # 4.9e9 elements
    y = noise((m, n))
    places = torch.randint(0, m, (64, k), device="cuda", dtype=torch.int32)
    places[:, 0] = m - 1 - torch.arange(64, device="cuda", dtype=torch.int32)
    weights = torch.rand((64, k), device="cuda")
    few = torch.arange(64 * k, device="cuda", dtype=torch.int32).view(64, k)
    want = ops().combine_experts(y[places.view(-1).long()], weights, few)
    assert torch.equal(ops().combine_experts(y, weights, places), want)
    one = torch.arange(m, device="cuda", dtype=torch.int32)[:, None]
    scale = torch.full((m, 1), 2.0, device="cuda")
    out = ops().combine_experts(y, scale, one, residual=y)
    assert torch.equal(out[-40:], (y[-40:].float() * 3).to(torch.bfloat16))


def test_block_norm():
    rows, k = 600_000, 8192  # 4.9e9 elements
    x, r, w = noise((rows, k)), noise((rows, k)), noise((k,))
    last = slice(rows - 32, rows)
    args = dict(weight=w, gate=w, kind="layer")
    want = ops().block_norm(x[last], r[last], scale=x[last], shift=r[last], **args)
    got = ops().block_norm(x, r, scale=x, shift=r, **args)
    assert torch.equal(got[0][last], want[0]) and torch.equal(got[1][last], want[1])
    del got
    small = ops().block_norm(x[last].clone(), r[last].clone(), precision="int8", **args)
    q, sf, _ = ops().block_norm(x, r, residual_out=r, precision="int8", **args)
    assert torch.equal(q[last], small[0]) and torch.equal(sf[last], small[1]) and torch.equal(r[last], small[2])
    del q, sf
    q, sf, gs = ops().block_norm(r, precision="nvfp4", **dict(args, gate=None))
    p, pf, _ = ops().block_norm(r[last], precision="nvfp4", global_scale=gs, **dict(args, gate=None))
    assert torch.equal(q[last], p) and torch.equal(sf[:, last].view(torch.uint8), pf.view(torch.uint8))


def test_linear_with_epilogue():
    m, n, k = 280_000, 16384, 128  # 4.6e9 outputs
    x = torch.randint(0, 256, (m, k // 2), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    sf = torch.full((k // 64, m, 4), 1.0, device="cuda").to(torch.float8_e4m3fn)
    gs = torch.full((), 0.01, device="cuda")
    w = ops().quantize(noise((n, k)), 0, 1)
    r = noise((m, n))
    want = ops().linear(x[-64:].contiguous(), sf[:, -64:].contiguous(), gs, *w, activation="gelu", residual=r[-64:], out=torch.empty((64, n), dtype=torch.bfloat16, device="cuda"))
    got = ops().linear(x, sf, gs, *w, activation="gelu", residual=r, out=r)
    # two tile shapes may add in another order: one bf16 rounding apart at the most
    assert ((got[-64:].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -13).all()
