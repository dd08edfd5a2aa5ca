"""What `rms_norm`, `dequantize`, `rope` and `grouped_linear` refuse: at the C ABI without a GPU (pointers that nothing dereferences: every call is
rejected during validation), and in Python."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(18)


def lib():
    from ac4k_kernel_amd import _lib
    return _lib.load()


def ops():
    from ac4k_kernel_amd import ops as o
    return o


def refused(rc, word):
    assert rc != 0 and word in lib().ac4k_last_error(), lib().ac4k_last_error()


def norm(**kw):
    a = dict(out=ONE, out_stride=64, sf=ONE, gs=ONE, given=1, x=ONE, x_stride=64, res=None, res_stride=0, sum=None, sum_stride=0, w=ONE, w_dtype=0,
             rows=4, K=64, dtype=0, precision=3, eps=1e-6, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib().ac4k_rms_norm(*a.values())


def test_norm_at_the_c_abi():
    refused(norm(x=None), b"null")
    refused(norm(rows=0), b"positive")
    refused(norm(K=65537), b"at most")
    refused(norm(dtype=3), b"bfloat16, half or float")
    refused(norm(w_dtype=1), b"weight must have the type of x")
    refused(norm(precision=4), b"unknown precision")
    refused(norm(res=ONE), b"place for the sum")
    refused(norm(sum=ONE), b"place for the sum")
    refused(norm(sf=None), b"scales")
    refused(norm(sf=ODD), b"scales")
    refused(norm(gs=None), b"global scale")
    refused(norm(eps=-1.0), b"eps")
    refused(norm(eps=float("nan")), b"eps")
    refused(norm(given=0, rows=100, K=4096), b"workspace")
    need = lib().ac4k_rms_norm_workspace_bytes(100, 4096, 0, 3, 0)
    assert need > 0
    refused(norm(given=0, rows=100, K=4096, ws=ONE, ws_bytes=need - 1), b"workspace")


def test_norm_workspace_sizes():
    size = lib().ac4k_rms_norm_workspace_bytes
    assert size(100, 4096, 0, 3, 1) == 0 and size(100, 4096, 0, 1, 0) == 0 and size(1, 8192, 0, 3, 0) == 0  # one workgroup holds it
    assert size(0, 4096, 0, 3, 0) == 0 and size(100, 70000, 0, 3, 0) == 0
    for rows in (17, 512, 4096, 75600):
        assert size(rows, 5120, 0, 3, 0) >= 4 * rows


def dequant(**kw):
    a = dict(out=ONE, dtype=0, q=ONE, sf=ONE, gs=ONE, gs_stride=0, lead=1, R=4, W=64, cols=64, precision=3, stream=None)
    a.update(kw)
    return lib().ac4k_dequantize(*a.values())


def test_dequantize_at_the_c_abi():
    refused(dequant(q=None), b"null")
    refused(dequant(R=0), b"positive")
    refused(dequant(cols=65), b"at most")
    refused(dequant(dtype=5), b"bfloat16, half or float")
    refused(dequant(precision=0), b"unknown precision")
    refused(dequant(gs=None), b"global scale")
    refused(dequant(W=96), b"chunks of 64")
    refused(dequant(q=ODD), b"4 bytes")
    refused(dequant(precision=1, W=40, cols=40), b"pieces of 16")
    refused(dequant(R=1 << 40), b"too large")


def rope(tensors=1, null=False, heads=2, sections=(32,), grid=(4,), **kw):
    from ac4k_kernel_amd import _lib
    t = (_lib.RopeTensor * 2)(*[_lib.RopeTensor(None if null else 16, 16, 0, 0, 0, 0, 0, 0, heads)] * 2)
    a = dict(count=tensors, dtype=0, B=1, N=4, D=64, table=ONE, length=8, pairs=32, sections=(ctypes.c_int64 * 9)(*sections), axes=len(sections),
             pos=None, pos_bytes=0, p0=0, p1=0, p2=0, grid=None if grid is None else (ctypes.c_int64 * 9)(*grid), inter=1, inv=0, stream=None)
    a.update(kw)
    return lib().ac4k_rope(t, *a.values())


def test_rope_at_the_c_abi():
    refused(rope(table=None), b"null")
    refused(rope(null=True), b"null")
    refused(rope(tensors=3), b"one or two")
    refused(rope(sections=(4,) * 9, grid=(1,) * 9), b"axes")
    refused(rope(grid=None), b"one of them")
    refused(rope(pos=ONE, pos_bytes=4), b"one of them")
    refused(rope(pos=ONE, pos_bytes=2, grid=None), b"4 or 8 bytes")
    refused(rope(N=0), b"positive")
    refused(rope(D=1025), b"head dim")
    refused(rope(D=62), b"do not fit")
    refused(rope(sections=(31,)), b"sections of 31 pairs")
    refused(rope(sections=(40, -8), grid=(1, 1)), b"section")
    refused(rope(grid=(9,)), b"the table has 8 positions")
    refused(rope(grid=(0,)), b"at least one place")
    refused(rope(heads=0), b"heads")
    refused(rope(dtype=7), b"bfloat16, half or float")
    refused(rope(table=ctypes.c_void_p(12)), b"8 bytes")
    refused(rope(B=1 << 23, N=1 << 23), b"too many tokens")


def grouped(**kw):
    a = dict(D=ONE, d_dtype=0, A=ONE, A_sf=ONE, A_gs=ONE, T=8, rows=None, B=ONE, B_sf=ONE, B_gs=ONE, gs_stride=0, bias=None, bias_dtype=0, offsets=ONE,
             M=8, N=32, K=128, E=2, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib().ac4k_linear_grouped_nvfp4(*a.values())


def test_grouped_at_the_c_abi():
    refused(grouped(offsets=None), b"null")
    refused(grouped(E=0), b"positive")
    refused(grouped(K=96), b"multiple of 64")
    refused(grouped(T=7), b"one row for each")
    refused(grouped(A=ctypes.c_void_p(24)), b"16-byte aligned")
    refused(grouped(B_sf=ODD), b"4-byte aligned")
    refused(grouped(E=65536), b"too large")
    refused(grouped(M=1 << 27, T=1 << 27), b"too large")
    refused(grouped(d_dtype=3), b"bfloat16, half or float")
    refused(grouped(bias=ONE, bias_dtype=9), b"bias must be")


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    for p in (None, "nvfp4", "int8"):
        with pytest.raises(RuntimeError, match="CUDA"):
            ops().rms_norm(x, precision=p)
    with pytest.raises(RuntimeError):
        ops().dequantize(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(()))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops().rope(x.reshape(1, 4, 1, 64), torch.zeros((4, 32, 2)))
    with pytest.raises(RuntimeError):
        ops().grouped_linear(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(()),
                             torch.zeros((1, 8, 32), dtype=torch.uint8), torch.zeros((1, 1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(()),
                             torch.zeros(2, dtype=torch.int32))


def test_calls_refused_before_the_operands_are_looked_at():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    for kw in (dict(precision="fp4"), dict(precision="int8", out=x), dict(residual_out=x), dict(global_scale=torch.zeros(())),
               dict(precision="int8", global_scale=torch.zeros(()))):
        with pytest.raises(RuntimeError):
            ops().rms_norm(x, **kw)
    with pytest.raises(RuntimeError, match="layout"):
        ops().rope(x.reshape(1, 4, 1, 64), torch.zeros((4, 32, 2)), layout="NBHD")
    with pytest.raises(RuntimeError, match="several axes"):
        ops().rope(x.reshape(1, 4, 1, 64), torch.zeros((4, 32, 2)), sections=(16, 16))
    for bad in (dict(sections=(), length=4), dict(sections=(0,), length=4), dict(sections=(4,), length=0), dict(sections=(4, -1), length=4)):
        with pytest.raises(RuntimeError):
            ops().rope_table(**bad, device="cpu")


def test_table_on_the_cpu():
    t = ops().rope_table((3, 2), 7, theta=100.0, device="cpu").double()
    ang = torch.arange(7).double()[:, None] * torch.tensor([1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3), 1.0, 0.1], dtype=torch.float64)
    assert t.shape == (7, 5, 2) and (t[..., 0] - ang.cos()).abs().max() <= 2.0 ** -24 and (t[..., 1] - ang.sin()).abs().max() <= 2.0 ** -24


@pytest.mark.gpu
def test_norm_operands():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(1024, dtype=torch.bfloat16, device="cuda")
    shifted, over = flat[:256].view(4, 64), flat[32:288].view(4, 64)
    for args, kw in (((x, w[:63]), {}), ((x, w.half()), {}), ((x.int(), w), {}), ((x, w, 1e-6, x.half()), {}), ((x, w, 1e-6, x[:3]), {}),
                     ((x, w, -1.0), {}), ((x, w), dict(out=x[:3])), ((x, w), dict(residual=x, residual_out=x.float())),
                     ((shifted, w), dict(out=over)), ((shifted, w), dict(residual=x, residual_out=over)),
                     ((x, w), dict(residual=shifted, residual_out=over)), ((x, w), dict(residual=x.clone(), out=(o := torch.empty_like(x)), residual_out=o)),
                     ((x, w), dict(precision="nvfp4", global_scale=torch.zeros(1, device="cuda"))),
                     ((x, w), dict(residual=x, residual_out=x[:1].expand(4, 64))), ((x[0], w), dict(out=w)), ((x[0], w), dict(residual=x[1], residual_out=w)), ((torch.zeros((2, 65537), device="cuda"),), {})):
        with pytest.raises(RuntimeError):
            ops().rms_norm(*args, **kw)


@pytest.mark.gpu
def test_dequantize_operands():
    q, sf, gs = ops().quantize(torch.ones((4, 64), dtype=torch.bfloat16, device="cuda"), 0, 1)
    for args, kw in (((q, sf), {}), ((q, sf[:, :8], gs), {}), ((q[:3], sf.float(), gs), {}), ((q, sf, gs.reshape(1)), {}), ((q, sf, gs), dict(cols=65)),
                     ((q, sf, gs), dict(dtype=torch.int8)), ((q.int(), sf, gs), {}), ((q[:, :31], sf, gs), {}),
                     ((q, sf, gs), dict(out=q.view(torch.bfloat16)))):
        with pytest.raises(RuntimeError):
            ops().dequantize(*args, **kw)


@pytest.mark.gpu
def test_rope_operands():
    x, t = torch.zeros((2, 4, 3, 64), device="cuda"), ops().rope_table(32, 8)
    pos = torch.zeros((1, 2, 4), dtype=torch.int64, device="cuda")
    buf = torch.zeros(4096, device="cuda")
    a, b = buf[:1536].view(2, 4, 3, 64), buf[64:1600].view(2, 4, 3, 64)
    for args, kw in (((x, t), dict(positions=pos.float())), ((x, t), dict(positions=pos[:, :, :3])), ((x, t), dict(positions=pos.expand(2, 2, 4))),
                     ((x, t), dict(positions=pos, grid=(4,))), ((x, t), dict(grid=(9,))), ((x, t), dict(grid=(2, 2))), ((x, t), dict(sections=(31,))),
                     ((x, t.half()), {}), ((x[..., :62], t), {}), (((x, x.half()), t), {}), (((x, x[:, :3]), t), {}), (((x, x, x), t), {}),
                     ((x, t), dict(out=x[:1])), ((a, t), dict(out=b)), (((a, a), t), dict(out=(a, a))), (((a, x), t), dict(out=(x, a))),
                     ((x, t), dict(positions=pos.cpu())), ((x[:, :, :1].expand(2, 4, 3, 64), t), dict(out=x[:, :, :1].expand(2, 4, 3, 64)))):
        with pytest.raises(RuntimeError):
            ops().rope(*args, **kw)


@pytest.mark.gpu
def test_grouped_operands():
    x = ops().quantize(torch.ones((6, 64), dtype=torch.bfloat16, device="cuda"), 0, 1)
    w = ops().quantize(torch.ones((2, 8, 64), dtype=torch.bfloat16, device="cuda"), 1, 2)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    rows = torch.zeros(6, dtype=torch.int32, device="cuda")
    ops().grouped_linear(*x, *w, off)
    for args, kw in (((*x, *w, off.long()), {}), ((*x, *w, off[:2]), {}), ((*x, *w, off), dict(rows=rows.long())),
                     ((*x, *w, off), dict(bias=torch.zeros(8, device="cuda"))), ((*x, *w, off), dict(out=torch.empty((5, 8), device="cuda"))),
                     ((*x, *w, off), dict(out=torch.empty((6, 9), device="cuda"))), ((*x, w[0][0], *w[1:], off), {}),
                     ((*x, w[0], w[1][:, :, :8], w[2], off), {}), ((*x, w[0], w[1], torch.zeros(3, device="cuda"), off), {}), ((*x, *w, off.cpu()), {}),
                     ((x[0][:, :16].contiguous(), x[1], x[2], *w, off), {})):
        with pytest.raises(RuntimeError):
            ops().grouped_linear(*args, **kw)
