"""Orthogonalised matrices of sizes whose products take each of the tile kernels' ways, against the definition in 64 bits.

Tiles are of 64 x 64, or of 128 x 128 where a launch has enough of them (half as many as CUs of a symmetric product, five
quarters of them of another one, of matrices of at least 256 rows and columns); the steps of few tiles, or of those of a last short round,
are split over workgroups. What each list takes below is worked out for 256 CUs.

The bound is that of the other sizes: 4 times the error of the same steps in float32, 2^-20 of the result, and half a step
of its type. Both sets of steps are formed on the GPU here, which takes seconds instead of minutes.
"""

import pytest
import torch

from myflows_amd import native
from myflows_amd import orthogonal as ops

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
RESNET18 = ([(64, 147)] + [(64, 576)] * 4 + [(128, 576)] + [(128, 1152)] * 3 + [(128, 64), (256, 1152)] + [(256, 2304)] * 3 +
            [(256, 128), (512, 2304)] + [(512, 4608)] * 3 + [(512, 256), (512, 2)])
LISTS = {
    # G and B of 276 small tiles, split; B X of 529 small ones
    "square": [(1425, 1425)],
    # G and B of 171 small tiles, split; B X of 324 large ones, less than a round
    "part_round": [(1152, 4608)],
    # G and B of 210 small tiles, split; B X of 530 large ones, a whole round and 18 that are split
    "wide": [(1217, 6700)],
    "tall": [(6700, 1217)],
    # B X of 1040 small tiles, a whole round and 16 that are split
    "small_rounds": [(1000, 4100)],
    # G and B of 153 large tiles, split; B X of 1089 small ones, a whole round and 65 that are split
    "two_sizes": [(2100, 2100)],
    # all products of large tiles in two or three rounds, the last one split
    "large_rounds": [(4100, 4100)],
    # B X of 821 tiles of both sizes in two rounds, none split
    "network": RESNET18,
    # G and B of 178 tiles of both sizes, some split
    "both_sizes": [(2100, 2100), (200, 3000), (70, 90), (90, 70), (300, 290)],
    # B X of exactly one round of large tiles
    "one_round": [(1024, 4096), (4096, 1024)],
}


def _steps(matrix, dtype):
    a, b, c = ops.COEFFICIENTS
    x = matrix.to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.double().square().sum().sqrt() + 1e-7).to(dtype)
    for _ in range(ops.STEPS):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


def _check(got, matrix):
    want = _steps(matrix, torch.float64)
    size = float(want.norm())
    rounding = torch.finfo(matrix.dtype).eps / 2 * size
    if matrix.dtype is torch.float16:
        rounding += 2.0 ** -25 * want.numel() ** 0.5
    bound = 4 * float((_steps(matrix, torch.float32).double() - want).norm()) + 2.0 ** -20 * size + rounding
    off = float((got.double() - want).norm())
    print(f"{tuple(matrix.shape)} off {off / size:.2e}, bound {bound / size:.2e}", flush=True)
    assert got.dtype is matrix.dtype and got.shape == matrix.shape and off <= bound


def _matrices(shapes, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(shape, generator=g, device="cuda") * 0.01).to(TYPES[dtype]) for shape in shapes]


def _spoil_workspace():
    """The bytes that the calls before left in the stream's workspace become NaN of every type."""
    native.stream_workspace(1, torch.float64).view(torch.int64).fill_(-1)


@pytest.mark.parametrize("name,dtype", [(name, "float32") for name in LISTS] +
                         [(name, dtype) for name in ("wide", "tall", "small_rounds", "both_sizes") for dtype in ("bfloat16", "float16")])
def test_every_kind_of_launch_matches_the_definition(name, dtype):
    print("orthogonalize", name, dtype, flush=True)
    matrices = _matrices(LISTS[name], dtype, len(name))
    got = ops.orthogonalize_many(matrices)
    for value, to in zip(matrices, got):
        _check(to, value)
    for _ in range(3):
        _spoil_workspace()
        for to, again in zip(got, ops.orthogonalize_many(matrices)):
            assert torch.equal(to, again)
    assert ops.orthogonalize_many(matrices, out=matrices)[0] is matrices[0]
    assert all(torch.equal(to, value) for to, value in zip(got, matrices))


@pytest.mark.parametrize("name", ["wide", "large_rounds", "both_sizes"])
def test_strided_matrices_and_their_neighbours(name):
    g = torch.Generator(device="cuda").manual_seed(1)
    shapes = LISTS[name]
    wide = [torch.randn((rows, cols + 13), generator=g, device="cuda") for rows, cols in shapes]
    parts = [value[:, 5:5 + cols] for value, (_, cols) in zip(wide, shapes)]
    want = ops.orthogonalize_many([part.contiguous() for part in parts])
    assert all(torch.equal(a, b) for a, b in zip(ops.orthogonalize_many(parts), want))
    # A result's neighbours in memory stay as they are.
    held = [torch.full((rows * cols + 128,), 7.0, device="cuda") for rows, cols in shapes]
    out = [value[64:-64].view(shape) for value, shape in zip(held, shapes)]
    ops.orthogonalize_many(parts, out=out)
    for value, to, same in zip(held, out, want):
        assert torch.equal(to, same) and bool((value[:64] == 7).all()) and bool((value[-64:] == 7).all())


def test_captured_graphs_side_by_side():
    lists = [_matrices(LISTS[name], "float32", 3) for name in ("wide", "two_sizes")]
    alone = [ops.orthogonalize_many(matrices) for matrices in lists]
    torch.cuda.synchronize()
    graphs, held = [], []
    for matrices in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(ops.orthogonalize_many(matrices))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in lists]
    for _ in range(4):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        again = ops.orthogonalize_many(lists[0])
        torch.cuda.synchronize()
        for got, want in zip([*held, again], [*alone, alone[0]]):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
