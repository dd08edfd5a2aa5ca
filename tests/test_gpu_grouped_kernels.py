"""GPU tests of each kernel of `grouped_linear`, by shapes that take it, with the kernel that ran asserted: the sizes that choose a kernel are those
known on the host (rows, N, K, experts), the sizes of the groups are free.  Tolerances: those of test_gpu_grouped.py."""
import pytest
import torch

from test_gpu_grouped import DTYPES, Problem, check, ops

pytestmark = pytest.mark.gpu

ROWS16, TILES_64_128, TILES_64_256, TILES_256 = 1, 2, 3, 4


def ran():
    from ac4k_kernel_amd import _lib
    return _lib.load().ac4k_debug_last_grouped_kernel()


# kernel, rows of each expert, N, K; `before` rows in front of the first group and `behind` rows behind the last one
SHAPES = [
    (ROWS16, [3, 0, 5], 1001, 2048), (ROWS16, [17, 0, 5, 1], 1001, 2112), (ROWS16, [2, 0, 1] * 30, 40, 320),
    (TILES_64_128, [30, 0, 66, 64], 2047, 512), (TILES_64_128, [30, 1, 65, 129], 2047, 448), (TILES_64_128, [20, 0, 70] * 24, 130, 320),
    (TILES_64_256, [1500, 0, 1, 1490], 1023, 256), (TILES_64_256, [63, 1, 2865, 62], 1023, 320), (TILES_64_256, [2, 1, 3, 0] * 18, 2047, 4032),
    (TILES_256, [9000, 0, 1, 22990], 257, 512), (TILES_256, [255, 20000, 3, 11733], 257, 448),
]
IDS = [f"{k}-{len(s)}x{sum(s)}-{n}-{kk}" for k, s, n, kk in SHAPES]


@pytest.mark.parametrize("kernel,sizes,n,k", SHAPES, ids=IDS)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out,bias", [("bf16", None), ("fp32", "bf16"), ("fp16", "fp32")])
def test_each_kernel(kernel, sizes, n, k, gather, out, bias):
    """Against the products in 64 bits; rows of no range and the memory around the output stay; the same bits again."""
    p = Problem(sizes, n, k, rows_of=97 if gather else None, seed=n + k, bias=bias, before=3, behind=5)
    buf = torch.full((p.m * n + 4097,), 7.0, dtype=DTYPES[out], device="cuda")
    y = buf[2049:2049 + p.m * n].reshape(p.m, n)  # rows at odd elements
    p.run(out=y)
    assert ran() == kernel
    check(p, y)
    assert (buf[:2049] == 7).all() and (buf[2049 + p.m * n:] == 7).all() and (y[:3] == 7).all() and (y[-5:] == 7).all()
    again = torch.full_like(y, 7.0)
    p.run(out=again)
    assert torch.equal(y, again)


def test_many_experts_on_the_largest_tiles():
    """More experts than a wave has lanes, groups that start anywhere, among them empty ones and single rows."""
    g = torch.Generator().manual_seed(3)
    for k in (448, 512):
        cuts = torch.randint(0, 87_990, (69,), generator=g).sort().values.tolist()
        cuts[10] = cuts[11] = cuts[12]
        cuts[20] = cuts[21] - 1
        ends = [0, *sorted(cuts), 87_990]
        p = Problem([b - a for a, b in zip(ends, ends[1:])], 431, k, rows_of=600, seed=k, bias="bf16", before=6, behind=4)
        y = p.run()
        assert ran() == TILES_256
        check(p, y)


TABLES = [(ROWS16, 8, 1000, 2048, 2), (TILES_64_128, 160, 2047, 512, 4), (TILES_64_256, 3000, 1023, 320, 4), (TILES_256, 32000, 257, 512, 4)]


@pytest.mark.parametrize("kernel,m,n,k,e", TABLES)
def test_wrong_tables_stay_in_range(kernel, m, n, k, e):
    """Indexes past x and in front of it: clamped, the rows of the others keep their bits; offsets past the rows, in front of them and falling:
    nothing outside of the output is touched."""
    sizes = [m // e] * (e - 1) + [m - m // e * (e - 1)]
    p = Problem(sizes, n, k, rows_of=50, seed=1)
    y = p.run()
    assert ran() == kernel
    check(p, y)
    rows = p.rows.clone()
    rows[::7] = 10 ** 9
    rows[3::7] = -5
    z = p.run(rows=rows.cuda())
    good = (rows == p.rows).cuda()
    assert torch.equal(z[good], y[good])
    p.rows = rows.clamp(0, 49)
    check(p, z)
    inner = [m // 4, m // 2] if e == 4 else []
    buf = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    for offsets in ([-3, *inner, m // 2, m + 1000], [m, *inner[::-1], m // 2, 0], [2 ** 31 - 1, *inner, -2 ** 31, 5], [0, *inner[:1], m, *inner[1:], m]):
        ops().grouped_linear(*p.x, *p.w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), rows=p.rows.cuda(),
                             out=buf[2048:2048 + m * n].reshape(m, n))
        assert ran() == kernel and (buf[:2048] == 7).all() and (buf[-2048:] == 7).all()


@pytest.mark.parametrize("kernel,m,n,k,e", TABLES)
def test_graph_replays_with_other_groups(kernel, m, n, k, e):
    """Two captured calls of every kernel (each with its own workspace, where there is one) replayed in turn on other routings, eager calls between."""
    p = Problem([m // e] * (e - 1) + [m - m // e * (e - 1)], n, k, rows_of=60, seed=3)
    rows, offsets = p.rows.cuda(), p.offsets.cuda()
    call = lambda: ops().grouped_linear(*p.x, *p.w, offsets, rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call()
    side.synchronize()
    assert torch.equal(first, call()) and ran() == kernel
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        assert ran() == kernel
        graphs.append((g, out))
    for turn in range(4):
        sizes = [0] * e
        sizes[turn % e] = m - (e - 1)
        sizes = [s or 1 for s in sizes]
        p.offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32)
        p.rows = torch.randint(0, 60, (m,), generator=torch.Generator().manual_seed(turn)).to(torch.int32)
        offsets.copy_(p.offsets.cuda())
        rows.copy_(p.rows.cuda())
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call())
        check(p, graphs[0][1])
        assert torch.equal(graphs[0][1], graphs[1][1])


@pytest.mark.parametrize("kernel,m,n,k,e", [(ROWS16, 28, 1000, 2048, 2), *TABLES[1:]])
@pytest.mark.parametrize("before,behind", [(0, 9), (6, 0), (5, 7)])
def test_rows_of_no_range_in_a_new_tensor_are_zero(kernel, m, n, k, e, before, behind):
    """Also where the memory of the new tensor held something else before; no range at all; no experts."""
    inner = m - before - behind
    p = Problem([inner // e] * (e - 1) + [inner - inner // e * (e - 1)], n, k, rows_of=60, seed=4, before=before, behind=behind)
    def run():
        junk = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
        del junk
        return p.run()
    y = run()
    assert ran() == kernel
    check(p, y)
    assert (y[:before] == 0).all() and (y[m - behind:] == 0).all()
    p.offsets = torch.full((e + 1,), m // 2, dtype=torch.int32)
    assert (run() == 0).all()
    none = ops().grouped_linear(*p.x, p.w[0][:0], p.w[1][:0], p.w[2][:0], torch.zeros(1, dtype=torch.int32, device="cuda"), rows=p.rows.cuda())
    assert none.shape == (m, n) and (none == 0).all()


@pytest.mark.parametrize("kernel,sizes,n", [(TILES_64_128, [30, 1, 65, 129], 2047), (TILES_64_256, [1500, 0, 1, 1490], 1023),
                                            (TILES_256, [9000, 0, 1, 22990], 257)])
@pytest.mark.parametrize("k", [128, 192])
@pytest.mark.parametrize("gather", [False, True])
def test_one_and_two_stages(kernel, sizes, n, k, gather):
    """A K of fewer stages than a kernel keeps under way, a whole one and one that starts in front of the row."""
    p = Problem(sizes, n, k, rows_of=97 if gather else None, seed=n + k, bias="fp32", before=2, behind=1)
    y = p.run()
    assert ran() == kernel
    check(p, y)
    assert (y[:2] == 0).all() and (y[-1:] == 0).all()


@pytest.mark.parametrize("kernel,m,n,k,e", [(ROWS16, 28, 1000, 2048, 2), *TABLES[1:]])
def test_graph_of_a_fixed_capacity(kernel, m, n, k, e):
    """One captured call for up to m rows: replayed with fewer, the rows behind the last range are zero, also where a replay before left values."""
    p = Problem([m // e] * (e - 1) + [m - m // e * (e - 1)], n, k, rows_of=60, seed=6)
    rows, offsets = p.rows.cuda(), p.offsets.cuda()
    call = lambda: ops().grouped_linear(*p.x, *p.w, offsets, rows=rows)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    assert ran() == kernel
    for used in (m, m // 3, 0, m - 1, 1):
        p.offsets = torch.tensor([used * i // e for i in range(e + 1)], dtype=torch.int32)
        offsets.copy_(p.offsets.cuda())
        g.replay()
        torch.cuda.synchronize()
        check(p, out)
        assert (out[used:] == 0).all() and torch.equal(out, call())
