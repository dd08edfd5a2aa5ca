"""What the routing operators refuse at the C ABI, without a GPU (pointers that nothing dereferences: every call is rejected during validation)."""
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


def route(**kw):
    a = dict(weights=ONE, experts=ONE, offsets=ONE, rows=ONE, places=ONE, logits=ONE, dtype=0, stride=64, bias=None, T=4, E=64, k=4, scoring=0, groups=1, top_groups=1,
             best=1, renormalize=1, scale=1.0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib().ac4k_route_experts(*a.values())


def test_route_at_the_c_abi():
    for name in ("weights", "experts", "offsets", "rows", "places", "logits"):
        refused(route(**{name: None}), b"null")
    refused(route(dtype=3), b"bfloat16, half or float")
    refused(route(T=0), b"positive")
    refused(route(E=0), b"experts 1 to")
    refused(route(E=1025), b"experts 1 to")
    refused(route(scoring=2), b"scoring")
    refused(route(groups=3), b"divide")
    refused(route(groups=0), b"divide")
    refused(route(E=130, groups=65), b"divide")
    refused(route(groups=4, top_groups=5), b"top_groups")
    refused(route(groups=4, top_groups=0), b"top_groups")
    refused(route(best=3), b"best one or two")
    refused(route(k=0), b"k must be")
    refused(route(k=65), b"k must be")
    refused(route(groups=16, top_groups=1, k=5), b"k must be")
    refused(route(T=1 << 26, k=2), b"too many tokens")
    refused(route(T=(1 << 26) - 15, k=1), b"too many tokens")  # 2^22 workgroups of 1024 threads
    refused(route(T=1000), b"workspace")
    need = lib().ac4k_route_experts_workspace_bytes(1000, 64, 4, 1, 1)
    assert need > 0
    refused(route(T=1000, ws=ONE, ws_bytes=need - 1), b"workspace")
    refused(route(T=1000, ws=ODD, ws_bytes=need), b"workspace")


def test_workspace_sizes():
    size = lib().ac4k_route_experts_workspace_bytes
    assert size(64, 64, 4, 1, 1) == 0 and size(0, 64, 4, 1, 1) == 0 and size(100, 1025, 4, 1, 1) == 0 and size(100, 64, 0, 1, 1) == 0
    # one workgroup: 128 tokens on 16 lanes each, 64 on a wave
    assert size(128, 64, 4, 1, 1) == size(128, 128, 16, 4, 4) == 0 < size(129, 64, 4, 1, 1)
    assert size(65, 64, 4, 4, 2) > 0 and size(65, 64, 17, 1, 1) > 0 and size(65, 129, 4, 1, 1) > 0 and size(64, 129, 4, 1, 1) == 0
    for t in (300, 1000, 100000):
        blocks = -(-t // 16)
        assert size(t, 64, 4, 1, 1) >= 4 * 64 + 7 * blocks * 64


def combine(**kw):
    a = dict(out=ONE, out_stride=64, y=ONE, y_stride=64, weights=ONE, places=ONE, residual=None, residual_stride=0, T=4, k=2, M=8, N=64, dtype=0, stream=None)
    a.update(kw)
    return lib().ac4k_combine_experts(*a.values())


def test_combine_at_the_c_abi():
    for name in ("out", "y", "weights", "places"):
        refused(combine(**{name: None}), b"null")
    refused(combine(dtype=3), b"bfloat16, half or float")
    for name in ("T", "k", "N"):
        refused(combine(**{name: 0}), b"positive")
    refused(combine(T=1 << 24), b"too large")
    refused(combine(T=1 << 20, N=1 << 20), b"too large")
    refused(combine(k=1 << 16), b"too large")


def test_operands_on_the_cpu_are_refused():
    from ac4k_kernel_amd import ops
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.route_experts(torch.zeros((4, 64)), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.combine_experts(torch.zeros((8, 64)), torch.zeros((4, 2)), torch.zeros((4, 2), dtype=torch.int32))
