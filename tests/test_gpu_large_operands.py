"""GPU tests of `rms_norm`, `dequantize`, `rope` and `grouped_linear` on operands of more than 2^32 elements or bytes: the last rows against
the same call on these rows alone."""
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


def test_norm_and_dequantize():
    rows, k = 600_000, 8192  # 4.9e9 elements
    x, w = noise((rows, k)), noise((k,))
    last = slice(rows - 32, rows)
    assert torch.equal(ops().rms_norm(x, w, out=torch.empty_like(x))[last], ops().rms_norm(x[last], w))
    q, sf = ops().rms_norm(x, w, precision="int8")
    p, pf = ops().rms_norm(x[last], w, precision="int8")
    assert torch.equal(q[last], p) and torch.equal(sf[last], pf)
    del q, sf
    q, sf, gs = ops().rms_norm(x, w, precision="nvfp4")
    p, pf, _ = ops().rms_norm(x[last], w, precision="nvfp4", global_scale=gs)
    assert torch.equal(q[last], p) and torch.equal(sf[:, last].view(torch.uint8), pf.view(torch.uint8))
    del x
    assert torch.equal(ops().dequantize(q, sf, gs)[last], ops().dequantize(p, pf, gs))


def test_rope():
    n, heads = 700_000, 48  # 4.3e9 elements
    x = noise((1, n, heads, 128))
    table = ops().rope_table(64, 64)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)[None, None] % 64
    want = ops().rope(x[:, -40:], table, positions=pos[:, :, -40:])
    assert torch.equal(ops().rope(x, table, positions=pos, out=x)[:, -40:], want)


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_linear(gather):
    t, k, n, e = 1_100_000, 8192, 16, 2  # x of 4.5e9 bytes
    x = torch.randint(0, 256, (t, k // 2), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    sf = torch.full((k // 64, t, 4), 1.0, device="cuda").to(torch.float8_e4m3fn)
    gs = torch.full((), 0.01, device="cuda")
    w = ops().quantize(noise((e, n, k)), 1, 2)
    last = torch.arange(t - 64, t, device="cuda")
    small = (x[-64:].contiguous(), sf[:, -64:].contiguous(), gs)
    want = ops().grouped_linear(*small, *w, torch.tensor([0, 0, 64], dtype=torch.int32, device="cuda"))
    if gather:  # more bytes than a tile's lane offsets reach
        got = ops().grouped_linear(x, sf, gs, *w, torch.tensor([0, 0, 64], dtype=torch.int32, device="cuda"), rows=last.to(torch.int32))
    else:
        got = ops().grouped_linear(x, sf, gs, *w, torch.tensor([0, 100, t], dtype=torch.int32, device="cuda"))[-64:]
    # the order of the sums goes by the kernel: two bf16 roundings of 2^-8 each, and sums in fp32 whose errors are at most
    # k 2^-24 = 2^-11 of the terms' sum of sizes, about sqrt(k) = 90 standard deviations of a result: 0.044 of one, and the
    # largest of 1024 results is more than 3; a wrong row is off by whole standard deviations
    torch.testing.assert_close(got, want, atol=1.5e-2 * want.abs().max().item(), rtol=2.0 ** -7)
