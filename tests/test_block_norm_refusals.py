"""What `block_norm` refuses at the C ABI, without a GPU (pointers that nothing dereferences: every call is rejected during validation)."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(18)


def lib():
    from ac4k_kernel_amd import _lib
    return _lib.load()


def refused(rc, word):
    assert rc != 0 and word in lib().ac4k_last_error(), lib().ac4k_last_error()


def norm(**kw):
    a = dict(out=ONE, out_stride=64, sf=ONE, gs=ONE, given=1, x=ONE, x_stride=64, res=ONE, res_stride=64, sum=ONE, sum_stride=64, weight=ONE, post=ONE, gate=ONE, gate_stride=0,
             gate_rows=0, scale=ONE, scale_stride=0, scale_rows=0, shift=ONE, shift_stride=0, shift_rows=0, vector_dtype=0, rows=4, K=64, dtype=0, precision=3, kind=1, alpha=1.0,
             eps=1e-6, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib().ac4k_block_norm(*a.values())


def test_at_the_c_abi():
    for name in ("out", "x"):
        refused(norm(**{name: None}), b"null")
    refused(norm(rows=0), b"positive")
    refused(norm(K=0), b"positive")
    refused(norm(K=32769), b"at most")
    refused(norm(rows=1 << 31), b"too many rows")
    refused(norm(dtype=3), b"bfloat16, half or float")
    refused(norm(vector_dtype=1), b"vectors must have")
    refused(norm(precision=4), b"unknown precision")
    refused(norm(kind=2), b"unknown kind")
    refused(norm(res=None), b"place for the sum")
    refused(norm(sum=None), b"place for the sum")
    refused(norm(res=None, sum=None, post=None), b"comes with a residual")
    refused(norm(res=None, sum=None, gate=None), b"comes with a residual")
    refused(norm(sf=None), b"scales")
    refused(norm(out=ODD), b"scales")
    refused(norm(gs=None), b"global scale")
    refused(norm(eps=-1.0), b"eps")
    refused(norm(eps=float("nan")), b"eps")
    for name in ("gate_rows", "scale_rows", "shift_rows"):
        refused(norm(**{name: -1}), b"rows of a vector")
        refused(norm(**{name: 1 << 31}), b"rows of a vector")
    need = lib().ac4k_block_norm_workspace_bytes(100, 4096, 0, 3, 0)
    refused(norm(given=0, rows=100, K=4096), b"workspace")
    refused(norm(given=0, rows=100, K=4096, ws=ONE, ws_bytes=need - 1), b"workspace")
    refused(norm(given=0, rows=100, K=4096, ws=ODD, ws_bytes=need), b"workspace")


def test_workspace_sizes():
    size = lib().ac4k_block_norm_workspace_bytes
    assert size(100, 4096, 0, 3, 1) == 0 and size(100, 4096, 0, 1, 0) == 0 and size(1, 8192, 0, 3, 0) == 0  # one workgroup holds it
    assert size(0, 4096, 0, 3, 0) == 0 and size(100, 40000, 0, 3, 0) == 0
    for rows in (17, 512, 4096, 75600):
        assert size(rows, 5120, 0, 3, 0) >= 12 * rows


def test_operands_on_the_cpu_are_refused():
    from ac4k_kernel_amd import ops
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.block_norm(torch.zeros((4, 64)))
