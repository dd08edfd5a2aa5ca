"""What the linear with an epilogue refuses at the C ABI, without a GPU (pointers that nothing dereferences: every call is rejected during validation)."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(258)


def lib():
    from ac4k_kernel_amd import _lib
    return _lib.load()


def refused(rc, word):
    assert rc != 0 and word in lib().ac4k_last_error(), lib().ac4k_last_error()


def linear(**kw):
    a = dict(D=ONE, d_dtype=0, A=ONE, A_sf=ONE, A_gs=ONE, B=ONE, B_sf=ONE, B_gs=ONE, bias=None, bias_dtype=0, activation=1, residual=None, residual_stride=0, M=4, N=64, K=64,
             ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib().ac4k_linear_nvfp4_epilogue(*a.values())


def test_at_the_c_abi():
    for name in ("D", "A", "A_sf", "A_gs", "B", "B_sf", "B_gs"):
        refused(linear(**{name: None}), b"null")
    for name in ("M", "N", "K"):
        refused(linear(**{name: 0}), b"positive")
    refused(linear(K=24), b"multiple of 16")
    refused(linear(d_dtype=3), b"bfloat16, half or float")
    refused(linear(bias=ONE, bias_dtype=3), b"bias must be")
    refused(linear(activation=-1), b"unknown activation")
    refused(linear(activation=5), b"unknown activation")
    for name in ("A", "B", "A_sf", "B_sf"):
        refused(linear(**{name: ODD}), b"aligned")
    refused(linear(M=1 << 24, N=1 << 24), b"too large")
    need = lib().ac4k_linear_nvfp4_scratch_bytes(64, 128, 14336)
    assert need > 0
    refused(linear(M=64, N=128, K=14336), b"workspace")
    refused(linear(M=64, N=128, K=14336, ws=ONE, ws_bytes=need - 1), b"workspace")
    refused(linear(M=64, N=128, K=14336, ws=ODD, ws_bytes=need), b"workspace")


def test_operands_on_the_cpu_are_refused():
    from ac4k_kernel_amd import ops
    x, sf, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((1, 16, 4)).to(torch.float8_e4m3fn), torch.zeros(())
    with pytest.raises(RuntimeError):
        ops.linear(x, sf, s, x, sf, s, activation="relu")
