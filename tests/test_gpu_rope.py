"""GPU tests of `rope` against the rotation in 64 bits with angles from its definition.

|out - exact| <= |exact| * eps/2 of the type + (|a| + |b|) * 6 * 2^-24 (+ half the smallest subnormal number): the rounding of the result
behind those of a cosine and a sine (2^-24 each), of two products and of a sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def data(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def exact(x, positions, sections, layout, interleaved, inverse=False, theta=10000.0):
    """positions [axes, B, N] (CPU int64, negative: as it is) -> (result, |a| + |b|) in 64 bits."""
    x = x.double()
    x = x if layout == "BNHD" else x.transpose(1, 2)
    pairs = sum(sections)
    y, size = x.clone(), torch.zeros_like(x)
    stay = (positions < 0).any(0)[..., None]
    first = 0
    for axis, n in enumerate(sections):
        for j in range(n):
            ang = positions[axis].double() * theta ** (-j / n)
            ang = torch.where(stay[..., 0], 0.0, -ang if inverse else ang)[..., None]
            p = first + j
            i, k = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
            a, b = x[..., i], x[..., k]
            y[..., i], y[..., k] = a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()
            size[..., i] = size[..., k] = a.abs() + b.abs()
        first += n
    return (y, size) if layout == "BNHD" else (y.transpose(1, 2), size.transpose(1, 2))


def check(out, ref):
    y, size = ref
    out = out.cpu()
    info = torch.finfo(out.dtype)
    bound = y.abs() * info.eps / 2 + size * 6 * 2.0 ** -24 + info.tiny * info.eps / 2
    assert ((out.double() - y).abs() <= bound).all()


CASES = [  # B, N, heads of q and k, D, sections
    (1, 1, 1, 1, 2, (1,)), (2, 3, 4, 2, 128, (64,)), (1, 17, 40, 8, 128, (64,)), (2, 33, 3, 3, 128, (22, 21, 21)), (1, 50, 2, 1, 96, (16, 16, 16)),
    (1, 9, 5, 5, 40, (8, 6, 6)), (1, 7, 2, 2, 36, (10, 8)), (3, 5, 3, 1, 64, (20,)), (1, 6, 2, 2, 50, (5, 0, 6)), (1, 4, 300, 3, 16, (4, 4)),
    (1, 5, 2, 2, 256, (128,)), (1, 3, 1, 1, 1024, (512,)), (1, 5, 2, 2, 13, (5,)), (2, 1, 40, 8, 128, (64,)),
]


@pytest.mark.parametrize("b,n,hq,hk,d,sections", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["BNHD", "BHND"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_positions(b, n, hq, hk, d, sections, dtype, layout, interleaved):
    length = 5000
    g = torch.Generator().manual_seed(n + d)
    pos = torch.randint(0, length, (len(sections), b, n), generator=g)
    if n > 2:
        pos[0, 0, n // 2] = -1  # padding along one axis is enough
    table = ops().rope_table(sections, length)
    shape = (lambda h: (b, n, h, d)) if layout == "BNHD" else (lambda h: (b, h, n, d))
    q, k = data(shape(hq), DTYPES[dtype], 1), data(shape(hk), DTYPES[dtype], 2)
    for t in (torch.int32, torch.int64):
        got = ops().rope((q.cuda(), k.cuda()), table, positions=pos.cuda().to(t), sections=sections, layout=layout, interleaved=interleaved)
        for x, y in zip((q, k), got):
            check(y, exact(x, pos, sections, layout, interleaved))
    alone = ops().rope(q.cuda(), table, positions=pos.cuda(), sections=sections, layout=layout, interleaved=interleaved)
    assert torch.equal(alone, got[0])
    back = ops().rope(got, table, positions=pos.cuda(), sections=sections, layout=layout, interleaved=interleaved, inverse=True)
    for x, y, z in zip(got, back, (q, k)):
        check(y, exact(x.cpu(), pos, sections, layout, interleaved, inverse=True))
        if dtype == "fp32":
            torch.testing.assert_close(y.cpu(), z, atol=2e-5, rtol=0)


@pytest.mark.parametrize("grid,n", [((2, 3, 4), 24), ((2, 3, 4), 31), ((3, 5, 7), 105), ((1, 1, 9), 9), ((7, 1, 1), 5)])
def test_grid(grid, n):
    """Row-major places; tokens behind the last one stay as they are, to the bit."""
    sections = (22, 21, 21)
    x = data((2, n, 3, 128), torch.bfloat16, n)
    i = torch.arange(n)
    pos = torch.stack((i // (grid[1] * grid[2]), i // grid[2] % grid[1], i % grid[2]))
    pos = torch.where(i < grid[0] * grid[1] * grid[2], pos, -1)[:, None].expand(-1, 2, -1)
    y = ops().rope(x.cuda(), ops().rope_table(sections, 16), grid=grid, sections=sections)
    check(y, exact(x, pos, sections, "BNHD", True))
    assert torch.equal(y[:, grid[0] * grid[1] * grid[2]:].cpu(), x[:, grid[0] * grid[1] * grid[2]:])


def test_default_positions_and_broadcast():
    x = data((3, 20, 2, 64), torch.float32, 1)
    table = ops().rope_table(32, 64)
    pos = torch.arange(20).expand(1, 3, -1)
    want = ops().rope(x.cuda(), table, positions=pos.cuda())
    for p in (None, torch.arange(20), torch.arange(20)[None], torch.arange(20).expand(3, 20)):
        assert torch.equal(ops().rope(x.cuda(), table, positions=None if p is None else p.cuda()), want)
    check(want, exact(x, pos, (32,), "BNHD", True))


def test_shared_series():
    sections = (16, 24, 24)
    table = ops().rope_table(sections, 100, shared=True).cpu().double()
    ang = torch.arange(100).double()[:, None] * 10000.0 ** (-torch.arange(64).double() / 64)
    assert (table[..., 0] - ang.cos()).abs().max() <= 2.0 ** -24 and (table[..., 1] - ang.sin()).abs().max() <= 2.0 ** -24


def test_far_positions():
    """Angles of far positions are those of 64 bits: position * frequency in 32 bits would be off by 0.03 here."""
    pos = torch.tensor([[[0, 1, 131071, 131070, 99999]]])
    x = data((1, 5, 2, 128), torch.float32, 1)
    check(ops().rope(x.cuda(), ops().rope_table(64, 131072), positions=pos.cuda()), exact(x, pos, (64,), "BNHD", True))


def test_positions_without_an_angle():
    """A position behind the table: NaN in the pairs of that axis only, the other axes, tokens and batches as they should be."""
    sections = (8, 8)
    pos = torch.zeros((2, 1, 4), dtype=torch.int64)
    pos[1, 0, 2] = 10
    pos[0, 0, 3] = 2 ** 31 + 1  # does not fit 32 bits
    y = ops().rope(data((1, 4, 2, 40), torch.bfloat16, 1).cuda(), ops().rope_table(sections, 10), positions=pos.cuda(), sections=sections)
    nan = torch.isnan(y)
    assert nan[0, 2, :, 16:32].all() and nan[0, 3, :, :16].all() and nan.sum() == 2 * 2 * 16


def test_views_in_place_and_packed_projection():
    """q and k as head slices of one projection, turned in place: the values between stay; views at odd places."""
    table = ops().rope_table(24, 100)
    pos = torch.randint(0, 100, (1, 2, 11), generator=torch.Generator().manual_seed(1))
    qkv = data((2, 11, 9, 50), torch.bfloat16, 1)
    want = qkv.clone()
    t = qkv.cuda()
    q, k = t[:, :, 0:4], t[:, :, 4:6]
    assert ops().rope((q, k), table, positions=pos.cuda(), out=(q, k))[0] is q
    fresh = ops().rope((qkv.cuda()[:, :, 0:4], qkv.cuda()[:, :, 4:6]), table, positions=pos.cuda())
    assert torch.equal(q, fresh[0]) and torch.equal(k, fresh[1]) and torch.equal(t[:, :, 6:].cpu(), want[:, :, 6:])
    check(q, exact(qkv[:, :, 0:4], pos, (24,), "BNHD", True))
    odd = data((2, 11, 3, 61), torch.float16, 2)[..., 5:54]  # heads of 49 elements at odd places
    check(ops().rope(odd.cuda(), table, positions=pos.cuda(), interleaved=False), exact(odd, pos, (24,), "BNHD", False))
    wide = odd.cuda()[..., ::2]  # copied first
    check(ops().rope(wide, ops().rope_table(12, 100), positions=pos.cuda()), exact(odd[..., ::2], pos, (12,), "BNHD", True))


@pytest.mark.parametrize("d,pairs", [(40, 20), (36, 18), (50, 20), (96, 44), (26, 9), (64, 30), (130, 60), (13, 5)])
def test_cut_vectors_in_place(d, pairs):
    """Widths that are no multiple of a vector: in place the same bits as into another tensor, one tensor and two."""
    table = ops().rope_table(pairs, 50)
    pos = torch.randint(0, 50, (1, 2, 33), generator=torch.Generator().manual_seed(1))
    for interleaved in (True, False):
        q, k = data((2, 33, 7, d), torch.bfloat16, d), data((2, 33, 3, d), torch.bfloat16, d + 1)
        fresh = ops().rope((q.cuda(), k.cuda()), table, positions=pos.cuda(), interleaved=interleaved)
        qc, kc = q.cuda(), k.cuda()
        ops().rope((qc, kc), table, positions=pos.cuda(), interleaved=interleaved, out=(qc, kc))
        alone = q.cuda()
        ops().rope(alone, table, positions=pos.cuda(), interleaved=interleaved, out=alone)
        check(fresh[0], exact(q, pos, (pairs,), "BNHD", interleaved))
        assert torch.equal(qc, fresh[0]) and torch.equal(kc, fresh[1]) and torch.equal(alone, fresh[0])


def test_gradient_by_differences():
    """<rope(x + d) - rope(x), g> = <d, inverse(g)> for a linear map, in fp32."""
    sections = (22, 21, 21)
    table = ops().rope_table(sections, 50)
    pos = torch.randint(0, 50, (3, 2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    x, d, g = (data((2, 9, 4, 128), torch.float32, i).cuda() for i in range(3))
    turn = lambda t, **kw: ops().rope(t, table, positions=pos, sections=sections, **kw).double()
    left = ((turn(x + d) - turn(x)) * g.double()).sum().item()
    right = (d.double() * turn(g, inverse=True)).sum().item()
    assert abs(left - right) <= 9216 * 4 * 2.0 ** -22  # elements, times their size and the roundings of four numbers


def test_one_tensor_of_a_pair_without_heads():
    q, k = data((2, 5, 3, 16), torch.bfloat16, 1).cuda(), torch.empty((2, 5, 0, 16), dtype=torch.bfloat16, device="cuda")
    table = ops().rope_table(8, 10)
    for pair in ((q, k), (k, q)):
        got = ops().rope(pair, table, sections=8)
        for x, y in zip(pair, got):
            assert y.shape == x.shape and torch.equal(y, ops().rope(x, table))


def test_many_tokens():
    """Workgroups of several tokens in both layouts, and batches whose last workgroup is not full."""
    for layout, shape in (("BNHD", (3, 3001, 2, 64)), ("BHND", (3, 5, 3001, 64)), ("BNHD", (1, 9001, 3, 40)), ("BHND", (1, 24, 2999, 128))):
        n = shape[1] if layout == "BNHD" else shape[2]
        x = data(shape, torch.bfloat16, n)
        pos = torch.randint(0, 50, (1, shape[0], n), generator=torch.Generator().manual_seed(1))
        pairs = shape[3] // 2
        y = ops().rope(x.cuda(), ops().rope_table(pairs, 50), positions=pos.cuda(), layout=layout, interleaved=layout == "BNHD")
        check(y, exact(x, pos, (pairs,), layout, layout == "BNHD"))


def test_empty():
    table = ops().rope_table(8, 10)
    assert ops().rope(torch.empty((0, 4, 2, 16), device="cuda"), table).shape == (0, 4, 2, 16)
    assert ops().rope(torch.empty((2, 0, 2, 16), device="cuda"), table).shape == (2, 0, 2, 16)


def test_outputs_stay_inside():
    pos = torch.randint(0, 10, (1, 1, 7), generator=torch.Generator().manual_seed(1)).cuda()
    for d, pairs in ((128, 64), (36, 18), (13, 5), (50, 20)):
        for interleaved in (True, False):
            x = data((1, 7, 3, d), torch.bfloat16, d).cuda()
            table = ops().rope_table(pairs, 10)
            buf = torch.full((x.numel() * 2 + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
            out = buf[4096:4096 + x.numel() * 2].view(torch.bfloat16).reshape(x.shape)
            ops().rope(x, table, positions=pos, interleaved=interleaved, out=out)
            assert torch.equal(out, ops().rope(x, table, positions=pos, interleaved=interleaved))
            assert (buf[:4096] == 0xA5).all() and (buf[4096 + x.numel() * 2:] == 0xA5).all()


def test_graph_and_streams():
    table = ops().rope_table(64, 4096)
    q, k = data((4, 1, 40, 128), torch.bfloat16, 1).cuda(), data((4, 1, 8, 128), torch.bfloat16, 2).cuda()
    pos = torch.zeros((1, 4, 1), dtype=torch.int32, device="cuda")
    call = lambda: ops().rope((q, k), table, positions=pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call()
    side.synchronize()
    assert torch.equal(first[0], call()[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for step in range(4):
        pos.fill_(1000 * step)
        q.copy_(data(q.shape, torch.bfloat16, 10 + step).cuda())
        g.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
