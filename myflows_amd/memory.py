"""Whether tensors share memory, told from their addresses, sizes and strides alone.

The entry points whose kernels read some tensors while they write others refuse calls in which one of the first
lies on one of the second. Tensors of unlike strides may lie between one another's rows (two slices of one
matrix's columns): they share nothing, and are told apart exactly.
"""

from __future__ import annotations

from functools import lru_cache
from heapq import heappop, heappush
from itertools import chain

import torch


def span(value):
    """The addresses from a tensor's first byte to behind its last one."""
    first = value.data_ptr()
    if value.is_contiguous():
        return first, first + value.numel() * value.element_size()
    last = sum((size - 1) * stride for size, stride in zip(value.shape, value.stride()))
    return first, first + (last + 1) * value.element_size()


@lru_cache(maxsize=1024)
def _runs(shape, strides, size):
    """A tensor's bytes as runs: (the length of one, ((step in bytes, number), ...) of the rest, falling steps)."""
    run, rest = size, []
    for stride, count in sorted((stride * size, count) for stride, count in zip(strides, shape) if count > 1 and stride):
        if not rest and stride <= run:
            run += stride * (count - 1)
        else:
            rest.append((stride, count))
    return run, tuple(reversed(rest))


def _reaches(steps, low, high):
    """Whether a sum of one multiple of each step, taken from first to last times, lies between low and high (exclusive);
    steps are (step, first, last), the largest step first."""
    if not steps:
        return low < 0 < high
    (step, first, last), *rest = steps
    least, most = sum(s * f for s, f, _ in rest), sum(s * l for s, _, l in rest)
    begin = max(first, (low - most) // step + 1)
    end = min(last, -((least - high) // step) - 1)
    return any(_reaches(rest, low - k * step, high - k * step) for k in range(begin, end + 1))


@lru_cache(maxsize=4096)
def _runs_meet(one, other, distance):
    """Whether runs that begin `distance` bytes apart share a byte: two of them, the first ones' i-th and the second ones'
    j-th, do where the difference of their steps lies within their lengths of the distance."""
    ranges = {}
    for (_, rest), sign in ((one, 1), (other, -1)):
        for step, count in rest:
            first, last = ranges.get(step, (0, 0))
            ranges[step] = (first, last + count - 1) if sign > 0 else (first - count + 1, last)
    steps = [(step, *ranges[step]) for step in sorted(ranges, reverse=True)]
    return _reaches(steps, distance - one[0], distance + other[0])


def share_memory(one, other):
    """Whether two tensors of one device share a byte."""
    first, end = span(one)
    other_first, other_end = span(other)
    if end <= other_first or other_end <= first or first == end or other_first == other_end:
        return False
    if one.is_contiguous() and other.is_contiguous():
        return True
    return _runs_meet(_runs(tuple(one.shape), one.stride(), one.element_size()),
                      _runs(tuple(other.shape), other.stride(), other.element_size()), other_first - first)


@lru_cache(maxsize=1024)
def _folded(shape, strides):
    """Whether two of the elements of these sizes and strides are one."""
    reach = 1
    for stride, count in sorted((stride, count) for stride, count in zip(strides, shape) if count > 1):
        if stride < reach:
            break
        reach += stride * (count - 1)
    else:
        return False
    offsets = torch.zeros((1,), dtype=torch.int64)
    for stride, count in zip(strides, shape):
        if count > 1 and not stride:
            return True
        offsets = (offsets[:, None] + torch.arange(count) * stride).reshape(-1)
    return offsets.unique().numel() < offsets.numel()


def overlap(written, read=()):
    """Whether one of the tensors written shares memory with itself, with another of them, or with a tensor read that is
    not its own: ``read`` holds (tensor, the index in ``written`` of the tensor that may lie on it, or None)."""
    entries = [(*span(value), index, False, value) for index, value in enumerate(written) if value.numel()]
    if any(not value.is_contiguous() and _folded(tuple(value.shape), value.stride()) for *_, value in entries):
        return True
    entries += [(*span(value), own, True, value) for value, own in read if value.numel()]
    entries.sort(key=lambda entry: entry[:2])
    writes, reads = [], []  # those whose spans have not ended, the one that ends first at the front
    for order, (first, end, own, is_read, value) in enumerate(entries):
        for held in (writes, reads):
            while held and held[0][0] <= first:
                heappop(held)
        for _, _, other_own, other_is_read, other in writes if is_read else chain(writes, reads):
            if (is_read or other_is_read) and own == other_own:
                continue
            if share_memory(value, other):
                return True
        heappush(reads if is_read else writes, (end, order, own, is_read, value))
    return False
