"""GPU tests of `rms_norm` and `dequantize`: against the formula in 64 bits, bit for bit where the output is quantized (the factor of
a row is the correctly rounded one, and everything behind it is a fixed order of fp32 operations), through views, in place, in
graphs and on other streams.

Unquantized: |y - exact| <= |exact| * (eps/2 of the type + 4 * 2^-24) + half the smallest subnormal number: one rounding to the type
behind the roundings of the factor and of two products."""
import math

import pytest
import torch

from conftest import make_input
from oracle import nvfp4_oracle as T

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def data(shape, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    return torch.where(torch.rand(shape, generator=g) < 0.002, x * 20, x).to(dtype)


def reference(x, weight, residual=None, eps=EPS):
    """(h, exact y in 64 bits, y in 32 bits as the kernel's order of operations gives it), all on the CPU."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h64 = h.double()
    factor = 1.0 / (h64.square().mean(-1, keepdim=True) + eps).sqrt()
    w = torch.ones(x.shape[-1]) if weight is None else weight
    return h, h64 * factor * w.double(), (h.float() * factor.float()) * w.float()


def check_plain(y, exact):
    y = y.cpu()
    info = torch.finfo(y.dtype)
    bound = exact.abs() * (info.eps / 2 + 4 * 2.0 ** -24) + info.tiny * info.eps / 2
    assert torch.isfinite(y.float()).all() and ((y.double() - exact).abs() <= bound).all()


def quantized(y, precision, gs=None):
    """y fp32 [rows, K] on the CPU -> the expected bytes of the output, the scales and the global scale."""
    rows, k = y.shape
    rp = T.align_up(rows, 16)
    if precision == "nvfp4":
        y = torch.nn.functional.pad(y, (0, -k % 64))
        blk = y.reshape(rows, -1, 16)
        m = blk.abs().amax(-1)
        if gs is None:
            amax = m.amax()
            gs = torch.where(amax < 2.0 ** -100, 0.0, amax) * (torch.tensor(1.0) / torch.tensor(2688.0))
        alpha = torch.where(gs.abs() < 2.0 ** -112, 0.0, 1.0 / gs)
        bits = T.f32_to_e4m3_bits(alpha * (m * T.ONE_SIXTH_F32))
        s = T.e4m3_bits_to_f32(bits)
        o = torch.where(s != 0, alpha * (1.0 / s), torch.zeros_like(s))
        q = T.f32_to_e2m1_bits(blk * o.unsqueeze(-1)).reshape(rows, -1, 2)
        sf = torch.zeros((y.shape[1] // 64, rp, 4), dtype=torch.uint8)
        sf[:, :rows] = bits.reshape(rows, -1, 4).permute(1, 0, 2)
        return q[..., 0] | (q[..., 1] << 4), sf, gs
    most = 448.0 if precision == "fp8e4m3" else 127.0
    m = y.abs().amax(-1)
    m = torch.where(m < 2.0 ** -100, 0.0, m)
    factor = torch.where(m == 0, 0.0, (torch.tensor(1.0) / m) * most)
    q = torch.nn.functional.pad(y * factor[:, None], (0, -k % 16))
    q = T.f32_to_e4m3_bits(q) if precision == "fp8e4m3" else T.f32_to_s8_sat(q)
    return q, torch.nn.functional.pad(m * (torch.tensor(1.0) / torch.tensor(most)), (0, rp - rows)), None


def same(a, b):
    return torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def raw(t):
    return t.cpu() if t.dtype not in (torch.float8_e4m3fn,) else t.cpu().view(torch.uint8)


def check_quantized(got, y32, precision, gs=None):
    eo, es, eg = quantized(y32, precision, gs)
    assert torch.equal(raw(got[0]), eo)
    assert torch.equal(raw(got[1]), es)
    if precision == "nvfp4":
        assert got[2].item() == eg.item()


# one row and many, K in one vector, in a piece of one, behind every split of a row over waves
SHAPES = [(1, 1), (1, 8), (3, 5), (16, 64), (7, 63), (17, 100), (1, 8192), (2, 16384), (15, 2048), (16, 2056), (33, 2047), (5, 5003),
          (600, 1040), (513, 4104), (2050, 520), (4101, 515), (2049, 1031), (2, 33000), (1, 65536)]


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("residual", [False, True])
def test_unquantized(rows, k, dtype, residual):
    x, w = data((rows, k), DTYPES[dtype], rows + k), data((k,), DTYPES[dtype], 3, 0.2) + 1
    r = data((rows, k), DTYPES[dtype], 7, 3.0) if residual else None
    h, exact, _ = reference(x, w, r)
    got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, residual=None if r is None else r.cuda())
    y = got[0] if residual else got
    assert y.dtype == x.dtype and y.shape == x.shape
    check_plain(y, exact)
    if residual:
        assert torch.equal(got[1].cpu(), h)


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("precision", ["nvfp4", "fp8e4m3", "int8"])
@pytest.mark.parametrize("dtype,w32,residual", [("bf16", False, True), ("bf16", True, False), ("fp16", False, False), ("fp16", True, True),
                                                ("fp32", True, True)])
def test_quantized(rows, k, precision, dtype, w32, residual):
    x, w = data((rows, k), DTYPES[dtype], rows + k), (data((k,), torch.float32, 3, 0.2) + 1).to(torch.float32 if w32 else DTYPES[dtype])
    r = data((rows, k), DTYPES[dtype], 7, 3.0) if residual else None
    h, exact, y32 = reference(x, w, r)
    got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, residual=None if r is None else r.cuda(), precision=precision)
    assert len(got) == (3 if precision == "nvfp4" else 2) + residual
    check_quantized(got, y32, precision)
    if residual:
        assert torch.equal(got[-1].cpu(), h)


# rows shared by a wave (heads of 128 and less), many turns of a workgroup, more rows than first-launch workgroups
@pytest.mark.parametrize("rows,k", [(9000, 64), (70001, 40), (5000, 128), (300, 250), (20001, 256), (300, 8192), (9001, 1100), (2100, 13000)])
@pytest.mark.parametrize("precision", [None, "nvfp4", "fp8e4m3", "int8"])
def test_many_rows(rows, k, precision):
    x, w, r = data((rows, k), torch.bfloat16, rows), data((k,), torch.bfloat16, 2), data((rows, k), torch.bfloat16, 3)
    h, exact, y32 = reference(x, w, r)
    got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, residual=r.cuda(), precision=precision)
    assert torch.equal(got[-1].cpu(), h)
    if precision is None:
        check_plain(got[0], exact)
    else:
        check_quantized(got, y32, precision)


@pytest.mark.parametrize("rows,k", [(1, 64), (5, 200), (600, 1040), (4101, 515), (9000, 64)])
def test_given_global_scale(rows, k):
    x, w = data((rows, k), torch.bfloat16, 1), data((k,), torch.bfloat16, 2)
    _, _, y32 = reference(x, w)
    for gs in (0.004, 1e-4, 0.0):  # 1e-4: saturates
        g = torch.tensor(gs, dtype=torch.float32)
        got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, precision="nvfp4", global_scale=g.cuda())
        check_quantized(got, y32, "nvfp4", g)
        assert got[2].item() == g.item()


def test_a_scale_that_is_no_scale():
    """Negative: zero codes and scales; NaN: NaN everywhere."""
    x = data((5, 200), torch.bfloat16, 1).cuda()
    q, sf, _ = ops().rms_norm(x, precision="nvfp4", global_scale=torch.tensor(-0.01, device="cuda"))
    assert (sf.float() == 0).all() and ((q & 0x77) == 0).all()
    q = ops().rms_norm(x, precision="nvfp4", global_scale=torch.tensor(math.nan, device="cuda"))
    assert torch.isnan(ops().dequantize(*q)).all()


def test_found_scale_given_back_gives_the_same():
    x, w = data((300, 1000), torch.bfloat16, 1).cuda(), data((1000,), torch.bfloat16, 2).cuda()
    a = ops().rms_norm(x, w, precision="nvfp4")
    b = ops().rms_norm(x, w, precision="nvfp4", global_scale=a[2])
    assert torch.equal(a[0], b[0]) and torch.equal(raw(a[1]), raw(b[1]))


@pytest.mark.parametrize("precision", [None, "nvfp4", "fp8e4m3", "int8"])
def test_views(precision):
    """Rows cut out of wider ones at odd places, several leading dims, every second row, a transposed batch (copied)."""
    wide = data((6, 50, 141), torch.bfloat16, 5)
    w = data((100,), torch.bfloat16, 6)
    for view in (lambda t: t[:, :, 17:117], lambda t: t[2, ::2, 1:101], lambda t: t[0, 3, 9:109], lambda t: t.transpose(0, 1)[..., :100]):
        x = view(wide)
        _, exact, y32 = reference(x, w)
        got = ops().rms_norm(view(wide.cuda()), w.cuda(), eps=EPS, precision=precision)
        if precision is None:
            assert got.shape == x.shape
            check_plain(got, exact)
        else:
            check_quantized(got, y32.reshape(-1, 100), precision)


def test_residual_views_and_in_place():
    for rows, k in ((70, 300), (5, 5003), (3, 2050)):
        x, r, w = data((rows, k), torch.bfloat16, 1), data((rows, k), torch.bfloat16, 2), data((k,), torch.float32, 3)
        h, exact, y32 = reference(x, w, r)
        big = torch.full((rows, k + 9), 5.0, dtype=torch.bfloat16, device="cuda")
        big[:, 3:3 + k] = r.cuda()
        res = big[:, 3:3 + k]
        y, s = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, residual=res, residual_out=res)  # the residual stream, in place
        assert s is res and torch.equal(res.cpu(), h) and (big[:, :3] == 5).all() and (big[:, 3 + k:] == 5).all()
        check_plain(y, exact)
        xc = x.cuda()
        got = ops().rms_norm(xc, w.cuda(), eps=EPS, residual=r.cuda(), residual_out=xc, precision="nvfp4")
        assert torch.equal(xc.cpu(), h)
        check_quantized(got, y32, "nvfp4")
        xc = x.cuda()
        assert ops().rms_norm(xc, w.cuda(), eps=EPS, out=xc) is xc
        check_plain(xc, reference(x, w)[1])


def test_no_weight_and_eps():
    x = data((9, 200), torch.float16, 1, 1e-3)
    for eps in (0.0, 1e-5, 1.0):
        check_plain(ops().rms_norm(x.cuda(), eps=eps), reference(x, None, eps=eps)[1])


@pytest.mark.parametrize("precision", [None, "nvfp4", "fp8e4m3", "int8"])
def test_zero_rows_and_zero_tensors(precision):
    x = data((20, 300), torch.bfloat16, 1)
    x[3] = 0
    x[19] = 0
    w = data((300,), torch.bfloat16, 2)
    for t in (x, torch.zeros_like(x), torch.zeros((5000, 40), dtype=torch.bfloat16)):
        wt = w[:t.shape[1]].contiguous()
        _, exact, y32 = reference(t, wt)
        got = ops().rms_norm(t.cuda(), wt.cuda(), eps=EPS, precision=precision)
        if precision is None:
            check_plain(got, exact)
        else:
            check_quantized(got, y32, precision)
            d = ops().dequantize(*got, dtype=torch.float32)
            assert torch.isfinite(d).all() and (d[(t == 0).all(-1).cuda()] == 0).all()
    tiny = torch.full((4, 64), 1e-30, dtype=torch.bfloat16)  # y under 2^-100 where eps holds the factor down
    wt = torch.full((64,), 1e-9, dtype=torch.bfloat16)
    if precision is not None:
        got = ops().rms_norm(tiny.cuda(), wt.cuda(), eps=1.0, precision=precision)
        assert (ops().dequantize(*got) == 0).all() and (got[1].float() == 0).all()


def test_rows_that_are_not_finite():
    """An infinite or NaN row comes out as 1/sqrt(inf) and inf * 0 say; the other rows are as without it."""
    x = data((40, 300), torch.bfloat16, 1)
    w = data((300,), torch.bfloat16, 2)
    clean = ops().rms_norm(x.cuda(), w.cuda())
    bad = x.clone()
    bad[5, 7] = math.inf
    bad[6, 299] = math.nan
    y = ops().rms_norm(bad.cuda(), w.cuda())
    keep = [i for i in range(40) if i not in (5, 6)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[6]).all() and torch.isnan(y[5, 7]) and (y[5, :7] == 0).all()
    for precision in ("fp8e4m3", "int8"):
        q, sf = ops().rms_norm(bad.cuda(), w.cuda(), precision=precision)
        cq, csf = ops().rms_norm(x.cuda(), w.cuda(), precision=precision)
        assert torch.equal(raw(q[keep]), raw(cq[keep])) and torch.equal(sf[keep], csf[keep]) and torch.isnan(sf[5:7]).all()


def test_large_values_do_not_overflow():
    x = torch.full((3, 4096), 3e38, dtype=torch.float32)
    x[1] = 1e-20
    check_plain(ops().rms_norm(x.cuda(), eps=0.0), reference(x, None, eps=0.0)[1])


@pytest.mark.parametrize("precision", ["nvfp4", "fp8e4m3", "int8"])
@pytest.mark.parametrize("rows,k", [(3, 64), (40, 300), (5000, 64)])
def test_largest_rows_quantized(rows, k, precision):
    """Maxima near the largest number of the type, whose reciprocal is a subnormal one: the codes still reach the end of their range."""
    x, w = data((rows, k), torch.float32, 1), torch.full((k,), 1e37)
    x[1] = 0
    x[1, 5] = -1.0  # all of a row in one place: sqrt(k) times the weight, 1.7e38 at k = 300
    _, _, y32 = reference(x, w)
    assert y32.abs().max() > 2.0 ** 125 and torch.isfinite(y32).all()
    got = ops().rms_norm(x.cuda(), w.cuda(), eps=EPS, precision=precision)
    check_quantized(got, y32, precision)
    top = got[0][1].view(torch.uint8).cpu()
    assert (top != 0).any() and torch.isfinite(got[1].float()).all()


def test_empty():
    x, w = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    assert ops().rms_norm(x, w).shape == (0, 64)
    assert ops().rms_norm(x, w, precision="fp8e4m3")[0].shape == (0, 64)


def test_graph_and_streams():
    """Captured calls replayed with other inputs, two graphs in turn, eager calls in between; a call on a side stream."""
    x, r, w = (data((700, 1040), torch.bfloat16, i).cuda() for i in (1, 2, 3))
    w = w[0].contiguous()
    xs, rs = x.clone(), r.clone()
    call = lambda p: ops().rms_norm(xs, w, residual=rs, precision=p)
    graphs = []
    side = torch.cuda.Stream()
    for p in ("nvfp4", "int8", None):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(p)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(p)
        graphs.append((p, g, out))
    for seed in range(4):
        xs.copy_(data((700, 1040), torch.bfloat16, 10 + seed).cuda())
        rs.copy_(data((700, 1040), torch.bfloat16, 20 + seed).cuda())
        for p, g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, call(p)):
                assert same(a, b)
    with torch.cuda.stream(side):
        on_side = call("nvfp4")
    side.synchronize()
    for a, b in zip(on_side, call("nvfp4")):
        assert same(a, b)


def test_outputs_stay_inside():
    """Margins around every output hold their pattern."""
    from ac4k_kernel_amd import _rocm_ops
    def window(shape, dtype):
        n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
        buf = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
        return buf, buf[4096:4096 + n].view(dtype).reshape(shape)
    for rows, k in ((1, 8), (5, 5003), (17, 100), (4101, 515), (2050, 520)):
        x, r, w = data((rows, k), torch.bfloat16, 1).cuda(), data((rows, k), torch.bfloat16, 2).cuda(), data((k,), torch.bfloat16, 3).cuda()
        for p in (None, "nvfp4", "fp8e4m3", "int8"):
            want = ops().rms_norm(x, w, residual=r, precision=p)
            wins = [window(t.shape, t.dtype) for t in want]
            outs = [t for _, t in wins]
            sf, gs = (outs[1] if p else None), (outs[2] if p == "nvfp4" else None)
            _rocm_ops.rms_norm(outs[0], sf, gs, False, x, w, r, outs[-1], p, 1e-6)
            for (buf, t), e in zip(wins, want):
                assert same(t, e)
                n = t.numel() * t.element_size()
                assert (buf[:4096] == 0xA5).all() and (buf[4096 + n:] == 0xA5).all()


# ------------------------------------------------------------------------------------------------------------ dequantize
@pytest.mark.parametrize("shape", [(1, 64), (17, 100), (70, 1000), (3, 33, 200), (2, 5, 7, 64), (300, 5003)])
@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_dequantize(shape, out):
    """One product in 32 bits (the one with the scale of 16 is exact), one rounding to the type: bit for bit."""
    x = make_input(shape, seed=sum(shape), outliers=True)
    c, r = x.ndim - 2, x.ndim - 1
    dt = DTYPES[out]
    q, sf, gs = ops().quantize(x.cuda(), c, r)
    d = ops().dequantize(q, sf, gs, dtype=dt)
    lead, rows = shape[:-2], shape[-2]
    flat_q, flat_s = q.cpu().reshape(-1, rows, q.shape[-1]), sf.cpu().view(torch.uint8).reshape(-1, *sf.shape[-3:])
    for i, (a, b) in enumerate(zip(flat_q, flat_s)):
        values = T.e2m1_unpack(a).reshape(rows, -1, 16) * T.sf_to_linear(b, rows).unsqueeze(-1)
        want = (values.reshape(rows, -1) * gs.cpu()).to(dt)
        assert torch.equal(d.cpu().reshape(-1, rows, want.shape[1])[i], want)
    cut = ops().dequantize(q, sf, gs, dtype=dt, cols=shape[-1])
    assert cut.shape == x.shape and torch.equal(cut, d[..., :shape[-1]])
    for precision in ("fp8e4m3", "int8"):
        q, sf = ops().quantize(x.cuda(), c, r, precision=precision)
        d = ops().dequantize(q, sf, dtype=dt)
        want = (q.cpu().float() * sf.cpu()[..., :rows].unsqueeze(-1)).to(dt)
        assert torch.equal(d.cpu(), want)


def test_dequantize_one_scale_per_plane():
    w = torch.stack([make_input((40, 128), seed=i, std=0.1 * (i + 1)) for i in range(3)]).cuda()
    parts = [ops().quantize(t, 0, 1) for t in w]
    q, sf, gs = (torch.stack([p[i].view(torch.uint8) if i == 1 else p[i] for p in parts]) for i in range(3))
    d = ops().dequantize(q, sf.view(torch.float8_e4m3fn), gs)
    assert torch.equal(d, torch.stack([ops().dequantize(*p) for p in parts]))


def test_dequantize_stays_inside_its_output():
    x = make_input((33, 100), seed=1).cuda()
    q, sf, gs = ops().quantize(x, 0, 1)
    for cols in (128, 100, 99, 3):
        buf = torch.full((33 * cols * 2 + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
        out = buf[4096:4096 + 33 * cols * 2].view(torch.bfloat16).reshape(33, cols)
        ops().dequantize(q, sf, gs, out=out)
        assert torch.equal(out, ops().dequantize(q, sf, gs)[:, :cols])
        assert (buf[:4096] == 0xA5).all() and (buf[4096 + 33 * cols * 2:] == 0xA5).all()
