"""Whether tensors share memory, against the sets of their bytes."""

import random

import pytest
import torch

from myflows_amd import memory


def _bytes(value, base):
    size, first = value.element_size(), value.data_ptr() - base
    offsets = torch.zeros((1,), dtype=torch.int64)
    for count, stride in zip(value.shape, value.stride()):
        offsets = (offsets[:, None] + torch.arange(count) * stride).reshape(-1)
    return {first + int(o) * size + k for o in offsets for k in range(size)}


@pytest.mark.parametrize("seed", range(6))
def test_random_views_of_one_buffer(seed):
    rng = random.Random(seed)
    held = torch.zeros(4000, dtype=torch.int64)
    found = {True: 0, False: 0}

    def view():
        flat = held.view(rng.choice([torch.float16, torch.float32, torch.int64]))
        shape = [rng.randint(0 if rng.random() < 0.03 else 1, 6) for _ in range(rng.randint(0, 3))]
        strides = [rng.choice([0, 1, 2, 3, 6, 7, 12, 18, 40, 41, 60]) for _ in shape]
        return flat.as_strided(shape, strides, rng.randint(0, 400 // flat.element_size()))

    for _ in range(1500):
        one, other = view(), view()
        want = not _bytes(one, held.data_ptr()).isdisjoint(_bytes(other, held.data_ptr()))
        assert memory.share_memory(one, other) is want and memory.share_memory(other, one) is want
        found[want] += 1
    assert min(found.values()) > 100


@pytest.mark.parametrize("seed", range(4))
def test_random_lists_of_written_and_read_views(seed):
    rng = random.Random(seed)
    held = torch.zeros(3000)
    found = {True: 0, False: 0}

    def view():
        shape = [rng.randint(1, 4) for _ in range(2)]
        return held.as_strided(shape, [rng.choice([0, 1, 2, 3, 4, 8, 16, 16]) for _ in shape] if rng.random() < 0.5 else [shape[1], 1],
                               rng.randint(0, 700))

    for _ in range(800):
        written = [view() for _ in range(rng.randint(1, 4))]
        read = [(rng.choice(written) if rng.random() < 0.2 else view(), rng.choice([None, *range(len(written))]))
                for _ in range(rng.randint(0, 3))]
        base = held.data_ptr()
        sets = [_bytes(value, base) for value in written]
        want = any(len(s) < value.numel() * 4 for s, value in zip(sets, written))
        want |= any(not a.isdisjoint(b) for i, a in enumerate(sets) for b in sets[:i])
        want |= any(not _bytes(value, base).isdisjoint(s) for value, own in read for i, s in enumerate(sets) if i != own)
        assert memory.overlap(written, read) is want
        found[want] += 1
    assert min(found.values()) > 50


def test_a_tensor_read_by_many():
    held = torch.zeros(40000)
    written = [held[i:i + 1] for i in range(20000)]
    assert not memory.overlap(written, [(held[20000:], None)] * 20000)
    assert memory.overlap(written, [(held[19999:], None)] * 20000)
    matrix = torch.zeros((50, 200))
    assert not memory.overlap(list(matrix.split(2, dim=1)), [(matrix[:, 2:4], 1)])
    assert memory.overlap([matrix[:, 2:4], matrix[:, 4:6]], [(matrix[:, 2:4], 1)])


def test_slices_of_a_large_matrix():
    matrix = torch.empty_strided((100000, 64), (64, 1), dtype=torch.bfloat16)
    left, right = matrix[:, :20], matrix[:, 20:]
    assert not memory.share_memory(left, right) and memory.share_memory(left, matrix[:, 19:])
    assert not memory.share_memory(matrix[0::2], matrix[1::2]) and memory.share_memory(matrix[0::2], matrix[2::3])
    assert not memory.share_memory(left.t(), right) and memory.share_memory(left.t(), left)
    assert not memory.share_memory(left, torch.zeros(5)) and not memory.share_memory(left, left[:0])
