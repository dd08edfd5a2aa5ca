"""The test of whether two tensors share memory that the operators with caller's outputs make, on the CPU: it may never miss a shared byte, and it must
know slices of the same rows apart."""
import itertools
import random

import torch


def may_overlap(a, b):
    from ac4k_kernel_amd import _rocm_ops
    return _rocm_ops._may_overlap(a, b)


def places(t):
    """Every byte that t has, from the start of its storage."""
    got = set()
    for index in itertools.product(*map(range, t.shape)):
        first = (t.storage_offset() + sum(i * s for i, s in zip(index, t.stride()))) * t.element_size()
        got.update(range(first, first + t.element_size()))
    return got


def test_no_shared_byte_is_missed():
    rng = random.Random(1)
    base = torch.zeros(4096, dtype=torch.uint8)
    found = apart = 0
    for _ in range(4000):
        pair = []
        for _ in range(2):
            dtype = rng.choice([torch.uint8, torch.bfloat16, torch.float32])
            flat = base.view(dtype)
            shape = [rng.randint(1, 4) for _ in range(rng.randint(0, 3))]
            stride = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48]) for _ in shape]
            pair.append(flat.as_strided(shape, stride, rng.randint(0, 60)))
        shared = bool(places(pair[0]) & places(pair[1]))
        said = may_overlap(*pair)
        assert said == may_overlap(*pair[::-1])
        assert said or not shared
        found += shared
        apart += not said
    assert found > 300 and apart > 300  # (both kinds were among them)


def test_slices_of_the_same_rows():
    wide = torch.zeros((6, 5, 96), dtype=torch.bfloat16)
    assert not may_overlap(wide[:, :, :32], wide[:, :, 32:])
    assert not may_overlap(wide[:, :, 32:], wide[:, :, :32])
    assert may_overlap(wide[:, :, :33], wide[:, :, 32:])
    assert may_overlap(wide[:, :, :32], wide.as_strided((5, 5, 2), wide.stride(), 95))  # into the next row
    assert not may_overlap(wide[::2], wide[1::2]) and may_overlap(wide[::2], wide[::3])
    assert not may_overlap(wide[:, 1], wide[:, 2:4]) and not may_overlap(wide[3, 2, 32:64], wide[:, :, :32])
    qkv = torch.zeros((2, 7, 9, 16))  # heads of a projection, also as [B, H, N, D]
    for t in (qkv, qkv.transpose(1, 2)):
        dim = t.shape.index(9)
        q, k = t.narrow(dim, 0, 4), t.narrow(dim, 4, 3)
        assert not may_overlap(q, k) and may_overlap(q, t.narrow(dim, 3, 3))


def test_tensors_without_elements():
    empty = torch.zeros((2, 0, 8))
    assert not may_overlap(empty, empty) and not may_overlap(empty, torch.zeros(4))
