"""GPU tests of `linear` with an activation and a residual against the formula in 64 bits on what the packed operands stand for.

|y - exact| <= |exact| * eps/2 of the output's type (one rounding), and before it in 32 bits: the sum, off by a unit of the last place for each addition,
s = (K + 8) * 2^-23 * gs * sum |a b| + 2^-23 * |bias|, times the steepest slope of an activation (1.13); the activation itself, 2^-20 * min(|v|, 1) + 2^-22 of its value
(of |v| the part that the far side of the normal distribution or the sigmoid has: its factor is off by 7 units in the fit, by 2 and v^2 units in the exponent,
and |v|^3 times either tail is under 0.6); the residual's sum, 2^-24 of both."""
import pytest
import torch

from conftest import make_input
from oracle import nvfp4_oracle as T

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTIVATIONS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def activated(kind, v):
    """In 64 bits."""
    if kind == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if kind == "gelu":
        return 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
    if kind == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    return v * torch.sigmoid(v) if kind == "silu" else v


def values(q):
    v = T.e2m1_unpack(q[0].cpu()).reshape(q[0].shape[0], -1, 16) * T.sf_to_linear(q[1].cpu().view(torch.uint8), q[0].shape[0]).unsqueeze(-1)[:, :q[0].shape[1] // 8]
    return v.reshape(q[0].shape[0], -1).double().cuda()


class Problem:
    def __init__(self, m, n, k, bias=None, residual=False, out="bf16", seed=0, std=0.05):
        self.m, self.n, self.k, self.out = m, n, k, DTYPES[out]
        self.x = ops().quantize(make_input((m, k), seed=seed).cuda(), 0, 1)
        self.w = ops().quantize(make_input((n, k), seed=seed + 1, std=std).cuda(), 0, 1)
        self.bias = None if bias is None else make_input((n,), seed=seed + 2).to(DTYPES[bias]).cuda()
        self.residual = make_input((m, n), seed=seed + 3, std=3.0).to(self.out).cuda() if residual else None
        gs = self.x[2].double() * self.w[2].double()
        a, b = values(self.x), values(self.w)
        self.v, size = a @ b.t() * gs, a.abs() @ b.abs().t() * gs
        self.error = (k + 8) * 2.0 ** -23 * size
        if self.bias is not None:
            self.v = self.v + self.bias.double()
            self.error = self.error + 2.0 ** -23 * self.bias.double().abs()

    def run(self, activation, out=None, **kw):
        if out is None and self.out is not torch.bfloat16:
            out = torch.full((self.m, self.n), 7.0, dtype=self.out, device="cuda")
        return ops().linear(*self.x, *self.w, **{**dict(bias=self.bias, out=out, activation=activation, residual=self.residual), **kw})

    def check(self, got, activation):
        assert got.shape == (self.m, self.n) and got.dtype == self.out
        exact = activated(activation, self.v)
        error = 1.13 * self.error + 2.0 ** -20 * self.v.abs().clamp(max=1.0) + 2.0 ** -22 * exact.abs()
        if self.residual is not None:
            exact = exact + self.residual.double()
            error = error + 2.0 ** -24 * exact.abs()
        info = torch.finfo(self.out)
        bound = error + (exact.abs() + error) * info.eps / 2 + info.tiny * info.eps / 2
        diff = (got.double() - exact).abs()
        assert (diff <= bound).all(), ((diff - bound).max(), (diff > bound).sum())


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("out", list(DTYPES))
@pytest.mark.parametrize("bias", [None, "bf16", "fp16", "fp32"])
def test_types(activation, out, bias):
    for m, n, k in ((3, 65, 256), (100, 130, 320), (150, 200, 192), (40, 33, 48)):
        p = Problem(m, n, k, bias, residual=bias is not None, out=out, seed=m)
        p.check(p.run(activation), activation)


# every kernel: decode with rows in sixteens, in rings, in registers, split along K; all of M in one tile; tiles; K of odd multiples of 16
SHAPES = [(1, 1, 64), (1, 14336, 4096), (2, 512, 12288), (1, 24577, 8192), (5, 300, 14336), (16, 4096, 4096), (17, 1001, 1024), (32, 28672, 512), (32, 14336, 1024), (8, 24600, 2048),
          (33, 64, 256), (48, 1000, 4096), (64, 5003, 1024), (100, 4100, 2880), (128, 128, 14336), (128, 5008, 448), (129, 257, 192), (300, 1003, 4096), (1001, 517, 2880),
          (1000, 5003, 320), (2049, 4097, 256), (700, 3000, 384), (4096, 2048, 512), (200, 127, 512), (70, 130, 80), (5, 7, 48), (333, 444, 16)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(m, n, k):
    p = Problem(m, n, k, "fp32", residual=True, seed=n)
    for activation in ("gelu", "silu") if m * n > 1000000 else ACTIVATIONS:
        p.check(p.run(activation), activation)
    p.residual = None
    p.check(p.run("gelu_tanh"), "gelu_tanh")
    q = Problem(m, n, k, None, residual=True, out="fp32", seed=n)
    q.check(q.run("relu"), "relu")


@pytest.mark.parametrize("mi,nj,splits", [(2, 1, 1), (2, 2, 1), (2, 4, 1), (3, 2, 1), (3, 4, 1), (4, 2, 1), (4, 4, 1), (2, 2, 3), (4, 4, 2), (3, 4, 2)])
@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_tile_plans(mi, nj, splits, out, linear_tuning):
    linear_tuning(mi=mi, nj=nj, splits=splits)
    for m, n, k in ((300, 520, 1024), (261, 391, 2112)):
        p = Problem(m, n, k, "bf16", residual=True, out=out, seed=mi)
        for activation in ("gelu", "silu", "relu"):
            p.check(p.run(activation), activation)
        p.residual = None
        p.check(p.run("gelu"), "gelu")


@pytest.mark.parametrize("kind", [1, 2, 3])
@pytest.mark.parametrize("m", [1, 8, 16, 31, 32])
def test_decode_kernels(kind, m, linear_tuning):
    linear_tuning(decode_kernel=kind)
    for n, k in ((300, 1024), (2050, 768)):
        p = Problem(m, n, k, "fp16", residual=True, seed=m)
        for activation in ("gelu", "relu"):
            p.check(p.run(activation), activation)


@pytest.mark.parametrize("m,n,k", [(4, 4096, 1024), (100, 1000, 512), (500, 1030, 256), (40, 100, 80)])
def test_residual_rows_apart_and_in_place(m, n, k):
    for out in DTYPES:
        p = Problem(m, n, k, "bf16", residual=True, out=out)
        want = p.run("silu")
        wide = torch.full((m, n + 37), 5.0, dtype=p.out, device="cuda")
        wide[:, 5:n + 5] = p.residual
        assert torch.equal(p.run("silu", residual=wide[:, 5:n + 5]), want)
        assert torch.equal(p.run("silu", residual=p.residual.t().contiguous().t()), want)
        same = p.residual.clone()
        got = p.run("silu", residual=same, out=same)
        assert got is same and torch.equal(got, want)
        one = wide[:1, 5:n + 5].expand(m, n)     # one row for all
        p.residual = one
        p.check(p.run("silu"), "silu")


def test_no_activation_and_no_residual_is_the_linear():
    for m, n, k in ((3, 300, 512), (100, 300, 512), (300, 300, 512)):
        p = Problem(m, n, k, "bf16")
        assert torch.equal(p.run(None), ops().linear(*p.x, *p.w, p.bias))
        zero = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
        p.check(p.run(None, residual=zero), None)


def test_activations_far_out():
    """Each activation over its whole range: the bias alone, with a weight of zeros."""
    n = 4096
    bias = torch.cat((torch.linspace(-15, 15, n - 12), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 88.0, -88.0, 1000.0, -1000.0, 1e30, -1e30, 3e38, -3e38])))
    for m in (1, 64, 200):
        p = Problem(m, n, 256, out="fp32")
        p.w = (torch.zeros_like(p.w[0]), p.w[1], p.w[2])
        p.bias = bias.cuda()
        p.v, p.error = bias.double().cuda().expand(m, n), torch.zeros((m, n), dtype=torch.float64, device="cuda")
        for activation in ACTIVATIONS:
            got = p.run(activation)
            assert torch.isfinite(got).all()
            p.check(got, activation)


@pytest.mark.parametrize("m", [1, 64, 200])
def test_values_that_are_not_finite(m):
    p = Problem(m, 512, 256, "fp32", out="fp32")
    p.bias[3], p.bias[7], p.bias[11] = float("nan"), float("inf"), float("-inf")
    rest = [i for i in range(512) if i not in (3, 7, 11)]
    clean = Problem(m, 512, 256, "fp32", out="fp32")
    for activation in ACTIVATIONS:
        got = p.run(activation)
        assert got[:, 3].isnan().all() and (got[:, 7] == float("inf")).all()
        assert torch.equal(got[:, rest], clean.run(activation)[:, rest])
        if activation in (None, "relu"):
            assert (got[:, 11] == (0 if activation else float("-inf"))).all()


def test_captured_and_on_another_stream():
    for m, n, k in ((1, 512, 8192), (64, 1024, 4096), (300, 512, 4096), (600, 1024, 256)):
        p = Problem(m, n, k, "bf16", residual=True)
        p.run("gelu")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = p.run("gelu")
        for seed in range(3):
            q = Problem(m, n, k, "bf16", residual=True, seed=seed + 5)
            for dst, src in zip((*p.x, *p.w, p.bias, p.residual), (*q.x, *q.w, q.bias, q.residual)):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                want = q.run("gelu")
            stream.synchronize()
            assert torch.equal(got, want)


def test_no_rows_and_refusals():
    p = Problem(8, 64, 128, "bf16", residual=True)
    x, w = p.x, p.w
    empty = (x[0][:0], torch.empty((2, 0, 4), dtype=torch.float8_e4m3fn, device="cuda"), x[2])
    assert ops().linear(*empty, *w, activation="relu").shape == (0, 64)
    r = p.residual
    big = torch.zeros((9, 64), dtype=torch.bfloat16, device="cuda")
    for kw in (dict(activation="tanh"), dict(activation=1), dict(residual=r.float()), dict(residual=r[:4]), dict(residual=r[:, :32]), dict(residual=r.cpu()), dict(residual=1.0),
               dict(residual=r, out=r.float()), dict(residual=big[:8], out=big[1:]), dict(out=r[:4], activation="relu"), dict(bias=p.bias[:5], activation="relu"),
               dict(bias=1.0, activation="relu"), dict(out=torch.empty((8, 64), device="cuda"), residual=r), dict(x=x[0][0], activation="relu"), dict(weight=None, activation="relu"),
               dict(x_scale=None, activation="relu"), dict(weight_scale=w[1][:1], activation="relu"), dict(x_global_scale=1.0, activation="relu"), dict(weight=w[0][:, :32], activation="relu")):
        args = dict(x=x[0], x_scale=x[1], x_global_scale=x[2], weight=w[0], weight_scale=w[1], weight_global_scale=w[2])
        with pytest.raises(RuntimeError):
            ops().linear(**{**args, **kw})
    with pytest.raises(RuntimeError, match="overlap"):
        d = torch.zeros((8, 64), dtype=torch.bfloat16, device="cuda")
        ops().linear(x[0], x[1], x[2], w[0], w[1], w[2], bias=d[0], out=d, activation="relu")
