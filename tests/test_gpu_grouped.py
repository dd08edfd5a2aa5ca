"""GPU tests of `grouped_linear` against the products in 64 bits of what the packed operands stand for.

|y - exact| <= |exact| * eps/2 of the output's type + (K + 8) * 2^-23 * gs * sum |a b| (+ the same rounding of the bias' sum): the products are
exact, every addition of a sum in 32 bits is off by a unit of its last place at the most."""
import pytest
import torch

from conftest import make_input
from oracle import nvfp4_oracle as T

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ops():
    from ac4k_kernel_amd import ops as o
    return o


class Problem:
    def __init__(self, sizes, n, k, rows_of=None, seed=0, bias=None, shared_scale=False, before=0, behind=0):
        """sizes: rows of each expert; rows_of: number of rows of x where rows are gathered; before / behind: rows in no range."""
        e, m = len(sizes), before + sum(sizes) + behind
        g = torch.Generator().manual_seed(seed)
        self.m, self.n, self.k, self.before = m, n, k, before
        self.offsets = torch.tensor([before + sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32)
        self.rows = None if rows_of is None else torch.randint(0, rows_of, (m,), generator=g).to(torch.int32)
        x = make_input((m if rows_of is None else rows_of, k), seed=seed, outliers=True)
        self.x = ops().quantize(x.cuda(), 0, 1)
        w = make_input((e, n, k), seed=seed + 1, std=0.05)
        if shared_scale:
            self.w = ops().quantize(w.cuda(), 1, 2)
        else:
            w = (w.float() * torch.linspace(0.5, 2.0, e)[:, None, None]).to(torch.bfloat16)
            parts = [ops().quantize(t.cuda(), 0, 1) for t in w]
            self.w = (torch.stack([p[0] for p in parts]), torch.stack([p[1].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn),
                      torch.stack([p[2] for p in parts]))
        self.bias = None if bias is None else make_input((e, n), seed=seed + 2).to(DTYPES[bias])

    def run(self, out=None, **kw):
        args = dict(rows=None if self.rows is None else self.rows.cuda(), bias=None if self.bias is None else self.bias.cuda(), out=out)
        return ops().grouped_linear(*self.x, *self.w, self.offsets.cuda(), **{**args, **kw})

    def exact(self):
        """(y, gs * sum |a b| + |bias|) in 64 bits on the GPU, zero in rows of no range; and which rows have a range."""
        def values(q, sf):
            v = T.e2m1_unpack(q.cpu()).reshape(q.shape[0], -1, 16) * T.sf_to_linear(sf.cpu().view(torch.uint8), q.shape[0]).unsqueeze(-1)
            return v.reshape(q.shape[0], -1).double().cuda()
        x = values(self.x[0], self.x[1])
        y = torch.zeros((self.m, self.n), dtype=torch.float64, device="cuda")
        size, met = torch.zeros_like(y), torch.zeros(self.m, dtype=torch.bool, device="cuda")
        for e in range(len(self.offsets) - 1):
            a, b = self.offsets[e].item(), self.offsets[e + 1].item()
            if a == b:
                continue
            src = x[a:b] if self.rows is None else x[self.rows[a:b].long().cuda()]
            w = values(self.w[0][e], self.w[1][e])
            gs = self.x[2].double() * (self.w[2].double() if self.w[2].dim() == 0 else self.w[2][e].double())
            y[a:b], size[a:b], met[a:b] = src @ w.t() * gs, src.abs() @ w.abs().t() * gs, True
            if self.bias is not None:
                y[a:b] += self.bias[e].double().cuda()
                size[a:b] += self.bias[e].abs().double().cuda()
        return y, size, met


def check(p, out):
    y, size, met = p.exact()
    info = torch.finfo(out.dtype)
    bound = y.abs() * info.eps / 2 + size * (p.k + 8) * 2.0 ** -23 + info.tiny
    assert ((out.double() - y).abs() <= bound)[met].all()


SIZES = [([1], 16, 64), ([5], 1, 64), ([0, 3, 0], 17, 128), ([16, 1, 31, 0, 7], 100, 192), ([2, 2, 2, 2], 33, 320), ([40, 0, 0, 90], 129, 256),
         ([300, 17, 1], 256, 448), ([128, 128], 128, 1024), ([257, 0, 255, 130], 300, 576), ([1] * 70, 48, 256), ([3, 0] * 100, 20, 64),
         ([700, 5], 1003, 2880), ([33] * 9, 512, 4096), ([1000], 130, 64), ([64, 65, 63], 257, 14336)]


@pytest.mark.parametrize("sizes,n,k", SIZES)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out,bias", [("bf16", None), ("fp32", "fp32"), ("fp16", "bf16"), ("bf16", "fp16")])
def test_against_exact(sizes, n, k, gather, out, bias):
    p = Problem(sizes, n, k, rows_of=max(1, sum(sizes) // 3) if gather else None, seed=n + k, bias=bias)
    y = p.run(out=torch.full((p.m, n), 7.0, dtype=DTYPES[out], device="cuda"))
    check(p, y)
    again = p.run(out=torch.full((p.m, n), 9.0, dtype=DTYPES[out], device="cuda"))
    assert torch.equal(y, again)  # the same bits for the same call


@pytest.mark.parametrize("sizes,n,k", [([3, 0, 9], 40, 128), ([200, 150], 300, 512), ([1, 2] * 40, 256, 256), ([600, 700], 512, 256)])
def test_rows_of_no_range_stay(sizes, n, k):
    """Rows in front of the first offset and behind the last one; a shared weight scale."""
    for gather in (None, 11):
        p = Problem(sizes, n, k, rows_of=gather, seed=5, shared_scale=True, before=6, behind=9)
        out = torch.full((p.m, n), 7.0, dtype=torch.bfloat16, device="cuda")
        p.run(out=out)
        check(p, out)
        assert (out[:6] == 7).all() and (out[-9:] == 7).all()


def test_every_kernel():
    """The four kernels by the shapes that take them: few rows on a long K, one tile of 64 rows an expert with narrow and wide weights, many rows;
    K with and without a half stage, gathered rows and rows in order."""
    for sizes, n, k in (([3, 0, 5], 4096, 2048), ([30] * 8, 2048, 512), ([20] * 40, 512, 320), ([1500, 900, 10, 1300], 1030, 320), ([1500, 900, 1, 1300], 1030, 512)):
        for gather in (None, 500):
            p = Problem(sizes, n, k, rows_of=gather, seed=n, bias="bf16", before=3)
            check(p, p.run())


@pytest.mark.parametrize("n", [1, 15, 16, 33, 64, 100, 127])
def test_narrow_weights_and_many_rows(n):
    """Fewer weight rows than a tile has, down to one: what lies behind the last one is neither read nor written."""
    for k in (128, 320):
        p = Problem([700, 0, 300, 65], n, k, rows_of=400, seed=n, bias="fp32", behind=2)
        buf = torch.full((p.m * n + 4096,), 7.0, dtype=torch.float32, device="cuda")
        out = buf[2048:2048 + p.m * n].reshape(p.m, n)
        p.run(out=out)
        check(p, out)
        assert (buf[:2048] == 7).all() and (out[-2:] == 7).all() and (buf[2048 + p.m * n:] == 7).all()


def test_one_expert_is_the_linear():
    """Up to the order of the fp32 sums: two bf16 roundings apart at the most."""
    for m, n, k in ((4, 512, 1024), (300, 640, 512)):
        p = Problem([m], n, k, seed=m)
        want = ops().linear(*p.x, p.w[0][0], p.w[1][0], p.w[2][0])
        torch.testing.assert_close(p.run(), want, atol=1e-3, rtol=2.0 ** -7)


@pytest.mark.parametrize("n,k,m", [(64, 128, 40), (300, 512, 900)])
def test_wrong_tables_stay_in_range(n, k, m):
    """Offsets past the rows or falling, indexes past x: clamped; what is in range of the others is right, nothing else is touched."""
    p = Problem([m // 2, m - m // 2], n, k, rows_of=50, seed=1)
    y = p.run()
    rows = p.rows.clone()
    rows[::7] = 10 ** 9
    rows[3::7] = -5
    z = p.run(rows=rows.cuda())
    good = (rows == p.rows).cuda()
    assert torch.equal(z[good], y[good]) and torch.isfinite(z.float()).all()
    buf = torch.full((m * n + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    for offsets in ([-3, m // 2, m + 1000], [m, m // 2, 0], [2 ** 31 - 1, -2 ** 31, 5]):
        ops().grouped_linear(*p.x, *p.w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), rows=p.rows.cuda(),
                             out=buf[2048:2048 + m * n].reshape(m, n))
        assert (buf[:2048] == 7).all() and (buf[-2048:] == 7).all()


def test_output_at_odd_elements():
    for sizes, n, k, dt in (([5, 9], 33, 128, torch.bfloat16), ([300, 200], 301, 256, torch.float32), ([300, 200], 301, 256, torch.bfloat16)):
        p = Problem(sizes, n, k, seed=2)
        buf = torch.full((p.m * n + 4097,), 7.0, dtype=dt, device="cuda")
        out = buf[2049:2049 + p.m * n].reshape(p.m, n)
        p.run(out=out)
        assert torch.equal(out, p.run(out=torch.empty((p.m, n), dtype=dt, device="cuda")))
        assert (buf[:2049] == 7).all() and (buf[2049 + p.m * n:] == 7).all()


def test_empty():
    p = Problem([0, 0], 32, 64, rows_of=4)
    assert p.run().shape == (0, 32)


@pytest.mark.parametrize("m,n,k", [(24, 256, 512), (600, 384, 512)])
def test_graph_replays_with_other_groups(m, n, k):
    """One captured call serves every routing of the same number of rows; two graphs, eager calls between the replays."""
    p = Problem([m // 4] * 4, n, k, rows_of=max(8, m // 4), seed=3)
    rows, offsets = p.rows.cuda(), p.offsets.cuda()
    call = lambda: ops().grouped_linear(*p.x, *p.w, offsets, rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call()
    side.synchronize()
    assert torch.equal(first, call())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for sizes in ([m, 0, 0, 0], [1, m - 3, 1, 1], [0, 0, m // 2, m - m // 2], [m // 3, m // 3, 0, m - 2 * (m // 3)]):
        p.offsets = torch.tensor([sum(sizes[:i]) for i in range(5)], dtype=torch.int32)
        offsets.copy_(p.offsets.cuda())
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            check(p, out)
            assert torch.equal(out, call())
