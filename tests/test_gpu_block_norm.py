"""GPU tests of `block_norm` against its formula in 64 bits and, where the output is quantized, bit for bit against the same order of fp32 operations: sums are
held in 64 bits, so that means and factors are the rounded ones, and everything behind them is a fixed order of products and sums.

Bounds.  h is off by one rounding to its type and six roundings in 32 bits of its two terms.  y, from the h that was kept, by one rounding to its type and, in
32 bits, two differences, the factor, its product, the weight's, 1 + scale, its product (8 * 2^-24 of the product, the last one of the sum), the second piece of the mean
(2^-48 of it)."""
import pytest
import torch

from oracle import nvfp4_oracle as T
from test_gpu_norm import DTYPES, check_quantized, data

pytestmark = pytest.mark.gpu
EPS = 1e-6
U = 2.0 ** -24


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def stats(v, kind, eps):
    """(mean, 1 / sqrt(..)) in 64 bits."""
    d = v.double()
    mean = d.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(d[..., :1])
    return mean, 1.0 / ((d - mean).square().mean(-1, keepdim=True) + eps).sqrt()


def normed32(v, kind, eps):
    mean, r = stats(v, kind, eps)
    m1 = mean.float()
    return ((v.float() - m1) - (mean - m1.double()).float()) * r.float()


def fma32(a, b, c):
    """a * b + c, rounded once (the product of two fp32 numbers is exact in 64 bits)."""
    return (a.double() * b.double() + c.double()).float()


class Reference:
    def __init__(self, x, residual=None, weight=None, gate=None, residual_scale=1.0, post_weight=None, scale=None, shift=None, kind="rms", eps=EPS):
        cpu = [None if t is None else t.cpu() for t in (x, residual, weight, gate, post_weight, scale, shift)]
        x, residual, weight, gate, post_weight, scale, shift = cpu
        self.h = x
        if residual is not None:
            u, u64 = x.float(), x.double()
            if post_weight is not None:
                mean, r = stats(x, kind, eps)
                u, u64 = normed32(x, kind, eps) * post_weight.float(), (x.double() - mean) * r * post_weight.double()
            a = torch.tensor(residual_scale, dtype=torch.float32)
            h = residual.float() * a
            if gate is not None:
                h, u64 = fma32(u, gate.float(), h), u64 * gate.double()
            else:
                h = h + u
            self.h = h.to(x.dtype)
            self.h64 = residual.double() * a.double() + u64
            self.h_size = (residual.double() * a.double()).abs() + u64.abs()
        mean, r = stats(self.h, kind, eps)
        self.y32, n64 = normed32(self.h, kind, eps), (self.h.double() - mean) * r
        size = n64.abs() + mean.abs() * r * 2.0 ** -24
        if weight is not None:
            self.y32, n64, size = self.y32 * weight.float(), n64 * weight.double(), size * weight.double().abs()
        if scale is not None:
            n64, size = n64 * (1.0 + scale.double()), size * (1.0 + scale.double()).abs()
            self.y32 = self.y32 * (1.0 + scale.float()) if shift is None else fma32(self.y32, 1.0 + scale.float(), shift.float())
        elif shift is not None:
            self.y32 = self.y32 + shift.float()
        if shift is not None:
            n64 = n64 + shift.double()
        self.y64, self.size = n64, size

    def check(self, got, precision=None, gs=None):
        got = got if isinstance(got, tuple) else (got,)
        k = self.h.shape[-1]
        if hasattr(self, "h64"):
            h = got[-1].cpu()
            assert h.dtype == self.h.dtype and h.shape == self.h.shape
            info = torch.finfo(h.dtype)
            assert ((h.double() - self.h64).abs() <= self.h64.abs() * info.eps / 2 + 7 * U * self.h_size + info.tiny * info.eps / 2).all()
            assert torch.equal(h, self.h)  # the same order of operations
        if precision is None:
            y = got[0].cpu()
            info = torch.finfo(y.dtype)
            assert y.dtype == self.h.dtype and y.shape == self.h.shape
            bound = self.y64.abs() * (info.eps / 2 + U) + 8 * U * self.size + info.tiny * info.eps / 2
            diff = (y.double() - self.y64).abs()
            assert (diff <= bound).all(), (diff - bound).max()
        else:
            check_quantized(got, self.y32.reshape(-1, k), precision, gs)


def problem(shape, dtype="bf16", vector="bf16", kind="rms", residual=True, weight=True, post=False, gate="none", modulate=False, alpha=1.0, seed=0, mean=0.0):
    """Arguments on the CPU.  gate: none, vector, batch (one a leading index) or row."""
    dt, vt, k = DTYPES[dtype], DTYPES[vector], shape[-1]
    g = torch.Generator().manual_seed(seed + 77)

    def vec(how, centre=0.0):
        s = {"vector": (k,), "batch": (shape[0], *[1] * (len(shape) - 2), k), "row": tuple(shape)}[how]
        return (torch.randn(s, generator=g) * 0.4 + centre).to(vt)
    a = dict(x=(data(shape, torch.float32, seed) + mean).to(dt), kind=kind)
    if residual:
        a["residual"], a["residual_scale"] = (data(shape, torch.float32, seed + 1, 3.0) + mean).to(dt), alpha
        if post:
            a["post_weight"] = vec("vector", 1.0)
        if gate != "none":
            a["gate"] = vec(gate)
    if weight:
        a["weight"] = vec("vector", 1.0)
    if modulate:
        a["scale"], a["shift"] = vec(modulate), vec(modulate)
    return a


def on_gpu(a):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in a.items()}


def run(a, precision=None, **kw):
    return ops().block_norm(**on_gpu(a), precision=precision, **kw)


PRECISIONS = [None, "fp8e4m3", "int8", "nvfp4"]
# the launch shapes: 16 lanes a row to 16 waves, vectors that are cut, rows of one element
COLS = [1, 7, 16, 100, 128, 130, 256, 300, 513, 1000, 1024, 2000, 4096, 5003, 6144, 8192, 10001, 16384, 20000, 32768]


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("k", COLS)
def test_widths(k, precision):
    for rows, kind, post, gate, modulate in ((1, "layer", True, "none", "vector"), (5, "rms", True, "vector", False), (37, "layer", False, "row", "row")):
        a = problem((rows, k), kind=kind, post=post, gate=gate, modulate=modulate, alpha=0.75, seed=k)
        Reference(**a).check(run(a, precision), precision)


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("dtype,vector", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_types(dtype, vector, kind, precision):
    for k in (200, 2888):
        a = problem((3, 17, k), dtype, vector, kind, post=True, gate="batch", modulate="batch", alpha=1.5, seed=5)
        Reference(**a).check(run(a, precision), precision)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("modulate", [False, "vector", "batch", "row"])
def test_parts_left_out(kind, residual, weight, modulate):
    for gate in ("none", "vector", "batch", "row") if residual else ("none",):
        a = problem((2, 9, 520), kind=kind, residual=residual, weight=weight, gate=gate, modulate=modulate, seed=2)
        for precision in (None, "nvfp4"):
            Reference(**a).check(run(a, precision), precision)
    if modulate:
        for name in ("scale", "shift"):  # one of the two
            b = dict(a)
            del b[name]
            Reference(**b).check(run(b))


@pytest.mark.parametrize("rows,k", [(2, 1000), (16, 2048), (40, 4096), (700, 512), (3000, 64), (33, 20000), (2100, 128)])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_nvfp4_in_one_launch_and_two(rows, k, kind):
    a = problem((rows, k), kind=kind, post=rows % 2 == 0, gate="vector", modulate="vector", seed=rows)
    Reference(**a).check(run(a, "nvfp4"), "nvfp4")
    a = problem((rows, k), kind=kind, residual=False, modulate="row", seed=rows)
    Reference(**a).check(run(a, "nvfp4"), "nvfp4")
    gs = torch.tensor(0.003)
    got = run(a, "nvfp4", global_scale=gs.cuda())
    assert got[2].item() == gs.item()
    Reference(**a).check(got, "nvfp4", gs)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layer_norm_of_rows_with_a_large_mean(dtype):
    for mean in (30.0, -1000.0):
        a = problem((6, 3000), dtype, "fp32", "layer", post=True, gate="vector", mean=mean)
        Reference(**a).check(run(a))
        a = problem((6, 3000), dtype, "fp32", "layer", residual=False, mean=mean)
        Reference(**a).check(run(a))
        Reference(**a).check(run(a, "int8"), "int8")


def test_rows_of_one_value():
    x = torch.tensor([3.0, 0.0, -0.375, 1000.0])[:, None].expand(4, 777).contiguous()
    for dt in DTYPES.values():
        y = ops().block_norm(x.to(dt).cuda(), kind="layer", shift=torch.full((777,), 0.5, device="cuda"))
        assert (y == 0.5).all()
        q, sf, gs = ops().block_norm(x.to(dt).cuda(), kind="layer", precision="nvfp4")
        assert gs.item() == 0 and not q.any() and not sf.view(torch.uint8).any()
    y = ops().block_norm(torch.zeros((4, 300), device="cuda"), kind="rms")
    assert (y == 0).all()


@pytest.mark.parametrize("dtype,value,other", [("fp16", 1000.0, 1000.5), ("bf16", 1000.0, 1004.0), ("bf16", -3.0, -3.015625), ("fp16", 0.25, 0.250244140625)])
def test_rows_of_one_value_but_for_one_element(dtype, value, other):
    """The variance is a 2^-37th of the square of the mean at the least: what 64 bits hold of the difference has to do."""
    for k in (3000, 32768):
        x = torch.full((4, k), value)
        x[torch.arange(4), torch.tensor([0, 7, 1000, k - 1])] = other
        a = dict(x=x.to(DTYPES[dtype]), kind="layer", eps=0.0)
        Reference(**a).check(run(a))
        Reference(**a).check(run(a, "int8"), "int8")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_values_near_the_largest_of_the_type(dtype):
    big = 2.0 ** 126
    x = data((5, 1000), torch.float32, 3).clamp(-1.9, 1.9) * big
    a = dict(x=x.to(DTYPES[dtype]), kind="layer", weight=torch.ones(1000, dtype=DTYPES[dtype]))
    Reference(**a).check(run(a))
    a["kind"] = "rms"
    Reference(**a).check(run(a))
    Reference(**a).check(run(a, "fp8e4m3"), "fp8e4m3")


@pytest.mark.parametrize("precision", [None, "fp8e4m3", "int8"])
def test_rows_that_are_not_finite_stay_apart(precision):
    a = problem((40, 600), post=True, gate="vector", modulate="vector")
    clean = run(a, precision)
    a["x"][3, 5], a["x"][17, 599], a["residual"][30, 0] = float("nan"), float("inf"), float("-inf")
    got = run(a, precision)
    others = [i for i in range(40) if i not in (3, 17, 30)]
    for p, q in zip(got, clean):
        p, q = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (p, q))
        assert torch.equal(p[others], q[others])
    assert all(got[-1][i].isnan().any() or got[-1][i].isinf().any() for i in (3, 17, 30))
    if precision is None:
        assert all(got[0][i].isnan().any() for i in (3, 17, 30))


def test_strided_vectors_and_rows():
    a = problem((3, 8, 640), gate="batch", modulate="batch", kind="layer")
    want = run(a)
    wide = torch.randn((3, 6, 640)).to(torch.bfloat16)
    wide[:, 1], wide[:, 3], wide[:, 5] = a["gate"][:, 0], a["scale"][:, 0], a["shift"][:, 0]
    six = wide.cuda().chunk(6, dim=1)
    b = {**on_gpu(a), "gate": six[1], "scale": six[3], "shift": six[5]}
    rows = torch.zeros((3, 8, 700), dtype=torch.bfloat16, device="cuda")
    rows[..., 9:649] = b["x"]
    b["x"] = rows[..., 9:649]
    for p, q in zip(want, ops().block_norm(**b)):
        assert torch.equal(p, q)
    b["x"] = a["x"].cuda().transpose(0, 1).contiguous().transpose(0, 1)     # no single stride: copied
    b["residual"] = a["residual"].cuda().transpose(0, 1).contiguous().transpose(0, 1)
    b["gate"] = a["gate"].cuda().transpose(0, 2).contiguous().transpose(0, 2)
    for p, q in zip(want, ops().block_norm(**b)):
        assert torch.equal(p, q)
    # vectors that several leading dims share: [2, 3, 1, 1, K] of [2, 3, 4, 5, K]
    a = problem((2, 3, 4, 5, 130), gate="row", modulate="row")
    a["gate"], a["scale"], a["shift"] = a["gate"][:, :, :1, :1], a["scale"][:, :1, :1, :1], a["shift"][:1, :1, :1, :1]
    Reference(**a).check(run(a))
    # both types: taken in fp32
    a = problem((4, 256), gate="vector", modulate="vector")
    a["gate"] = a["gate"].float()
    Reference(**a).check(run(a))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_outputs_in_place(kind):
    for shape in ((5, 100), (300, 4096), (9, 20000)):
        a = problem(shape, kind=kind, post=True, gate="vector", modulate="vector")
        y, h = run(a)
        for name in ("x", "residual"):
            g = on_gpu(a)
            got = ops().block_norm(**g, residual_out=g[name])
            assert got[1] is g[name] and torch.equal(got[0], y) and torch.equal(got[1], h)
            g = on_gpu(a)
            got = ops().block_norm(**g, residual_out=g[name], precision="nvfp4")
            assert torch.equal(got[3], h)
        g = on_gpu(a)
        got = ops().block_norm(**g, residual_out=g["residual"], out=g["x"])
        assert got[0] is g["x"] and torch.equal(got[0], y) and torch.equal(got[1], h)
    # columns around an output stay as they are
    a = problem((6, 333), kind=kind)
    y, h = run(a)
    buffer = torch.full((6, 2, 400), 7.0, dtype=torch.bfloat16, device="cuda")
    ops().block_norm(**on_gpu(a), out=buffer[:, 0, 11:344], residual_out=buffer[:, 1, 11:344])
    assert torch.equal(buffer[:, 0, 11:344], y) and torch.equal(buffer[:, 1, 11:344], h)
    assert (buffer[..., :11] == 7).all() and (buffer[..., 344:] == 7).all()


def test_one_tensor_as_both_operands_and_shared_rows():
    a = problem((30, 1000), kind="layer", gate="vector", post=True)
    a["residual"] = a["x"]
    y, h = run(a)
    Reference(**a).check((y, h))
    g = on_gpu(a)
    x = g["x"]
    got = ops().block_norm(**{**g, "residual": x}, residual_out=x)
    assert got[1] is x and torch.equal(got[0], y) and torch.equal(x, h)
    # one row for all of the residual; windows of one buffer as rows
    a = problem((30, 1000))
    a["residual"] = a["residual"][:1].expand(30, 1000)
    Reference(**a).check(run(a))
    buffer = data((5000,), torch.bfloat16).cuda()
    windows = buffer.as_strided((64, 1000), (50, 1))
    assert torch.equal(ops().block_norm(windows, kind="layer"), ops().block_norm(windows.contiguous(), kind="layer"))


def test_no_rows():
    for precision in PRECISIONS:
        x = torch.zeros((2, 0, 96), device="cuda")
        got = ops().block_norm(x, x, gate=torch.zeros((2, 1, 96), device="cuda"), precision=precision)
        assert got[-1].shape == x.shape
        if precision == "nvfp4":
            assert got[2].item() == 0


@pytest.mark.parametrize("precision", PRECISIONS)
@pytest.mark.parametrize("shape", [(2, 3, 256), (4, 300, 1024)])
def test_captured_and_on_another_stream(shape, precision):
    a = on_gpu(problem(shape, kind="layer", post=True, gate="batch", modulate="batch"))
    ops().block_norm(**a, precision=precision)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops().block_norm(**a, precision=precision)
    for seed in range(3):
        for n, t in on_gpu(problem(shape, kind="layer", post=True, gate="batch", modulate="batch", seed=seed + 9)).items():
            if isinstance(t, torch.Tensor):
                a[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            want = ops().block_norm(**a, precision=precision)
        stream.synchronize()
        for p, q in zip(got, want):
            assert torch.equal(p.reshape(-1).view(torch.uint8), q.reshape(-1).view(torch.uint8))


def test_as_rms_norm_without_the_rest():
    x, r, w = data((50, 1000), torch.bfloat16).cuda(), data((50, 1000), torch.bfloat16, 1).cuda(), torch.rand(1000, device="cuda")
    for precision in PRECISIONS:
        for p, q in zip(ops().block_norm(x, r, w, precision=precision), ops().rms_norm(x, w, residual=r, precision=precision)):
            assert torch.equal(p.reshape(-1).view(torch.uint8), q.reshape(-1).view(torch.uint8))


def test_many_rows():
    x = torch.randn((300001, 64), device="cuda", dtype=torch.float32)
    gate, shift = torch.randn((64,), device="cuda"), torch.randn((300001, 64), device="cuda")
    y, h = ops().block_norm(x, x, gate=gate, shift=shift, kind="layer")
    hh = x.double() + x.double() * gate.double()
    yy = (h.double() - h.double().mean(1, keepdim=True)) / (h.double().var(1, unbiased=False, keepdim=True) + EPS).sqrt() + shift.double()
    assert ((h - hh).abs() <= hh.abs() * U + 2 * U * (x.abs() + (x * gate).abs())).all()
    assert ((y - yy).abs() <= 2 * U * yy.abs() + 8 * U * (yy - shift).abs() + 2.0 ** -40).all()


def test_python_refusals():
    x = torch.zeros((4, 6, 64), dtype=torch.bfloat16, device="cuda")
    v, h = torch.zeros(64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, dtype=torch.float16, device="cuda")
    b = ops().block_norm
    for kw in (dict(x=x.cpu()), dict(x=x.double()), dict(x=[1.0]), dict(x=x[..., :0]), dict(residual=x[:2]), dict(residual=x.float()), dict(residual=1.0), dict(residual_out=x),
               dict(gate=v), dict(post_weight=v), dict(weight=h), dict(weight=v[:32]), dict(weight=v.cpu()), dict(weight=v.expand(4, 64)), dict(weight=1.0), dict(scale=v[:63]),
               dict(scale=x[:2]), dict(scale=x[0]), dict(scale=x[:, :3]), dict(scale=x[:1]), dict(shift=x[:, 0]), dict(shift=v.cpu()), dict(shift=2.0), dict(scale=h), dict(residual=x, gate=x[:3, :1]),
               dict(residual=x, gate=v, scale=h), dict(kind="batch"), dict(precision="fp4"), dict(precision="int8", out=x), dict(precision="int8", global_scale=torch.ones((), device="cuda")),
               dict(precision="nvfp4", global_scale=torch.ones(1, device="cuda")), dict(precision="nvfp4", global_scale=0.5), dict(eps=-1.0), dict(out=x.float()), dict(out=x[:2]), dict(out=1.0),
               dict(residual=x.clone(), residual_out=x[:2]), dict(residual=x.clone(), residual_out=x[:, :1].expand(4, 6, 64)), dict(x=x[:, :5], out=x[:, 1:]),
               dict(x=torch.zeros((2, 32769), device="cuda"))):
        with pytest.raises(RuntimeError):
            b(**{**dict(x=x), **kw})
    y = x.clone()
    scale = x[:, :1]
    with pytest.raises(RuntimeError, match="vector"):
        b(y, scale=scale, out=x)
    with pytest.raises(RuntimeError, match="vector"):
        b(y, y.clone(), scale=scale, residual_out=x)
