"""Matrices orthogonalised by Newton-Schulz products, against the definition in 64 bits.

Tolerance. The steps raise an error in a small singular direction by up to a = 3.4 each, whatever the arithmetic, so
the error is measured against that of the same steps in float32 on the CPU. A value held as two float16 has an error
of 2^-23 of it, twice float32's half step; a product leaves out lo lo, 2^-24 of it at most; its sums are float32. So
each product has at most three times the error of a float32 one, and the order of the sums may differ: in the
Frobenius norm the result is within 4 times float32's error, plus 2^-20 of the result for matrices so small that
float32's own error happens to be near 0, plus half a step of the type (of a float16 result below 2^-14, half of 2^-24).
With one row or column there is one singular value, 1, and float32 may well have no error at all: there the bound is
the worst case. A step holds G, B and X with relative errors of 2^-23, so with g = x^2 up to 1.24 its X is off by at most
(2 |b| g + 3 |c| g^2 + |a| + 1) 2^-23 < 26 2^-23 of 1. The default steps take 1 to .701, 1.114, .721, 1.090, where the
derivative a + 3 b g + 5 c g^2 is -1.14, 1.30, -1.26, .76, so an error after the steps 1 to 5 comes out 1.42, 1.25, .96, .76
and 1 times as large: 5.4 times 26 2^-23 in all, below 2^-15.
"""

import pytest
import torch

import myflows_amd as mf
from myflows_amd import native
from myflows_amd import orthogonal as ops

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
gpu = pytest.mark.gpu


def _steps(matrix, dtype, steps=5, coefficients=ops.COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = matrix.detach().cpu().to(dtype).reshape(matrix.shape[0], -1)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.double().square().sum().sqrt() + eps).to(dtype)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.T if tall else x).reshape(matrix.shape)


def _check(got, matrix, **options):
    want = _steps(matrix, torch.float64, **options)
    size = float(want.norm())
    rounding = torch.finfo(matrix.dtype).eps / 2 * size
    if matrix.dtype is torch.float16:
        rounding += 2.0 ** -25 * want.numel() ** 0.5
    bound = 4 * float((_steps(matrix, torch.float32, **options).double() - want).norm()) + 2.0 ** (-15 if min(want.shape[0], want[0].numel()) == 1 else -20) * size + rounding
    off = float((got.detach().cpu().double() - want).norm())
    print(f"off {off / size if size else off:.2e}, bound {bound / size if size else bound:.2e}", flush=True)
    assert got.dtype is matrix.dtype and got.shape == matrix.shape and off <= bound


def _matrix(rows, cols, dtype, seed, spectrum="noise"):
    g = torch.Generator().manual_seed(seed)
    if spectrum == "noise":
        x = torch.randn((rows, cols), generator=g)
    else:  # singular values that fall over four orders of magnitude
        short = min(rows, cols)
        u, _ = torch.linalg.qr(torch.randn((rows, short), generator=g, dtype=torch.float64))
        v, _ = torch.linalg.qr(torch.randn((cols, short), generator=g, dtype=torch.float64))
        x = (u * 10.0 ** (-4.0 * torch.arange(short) / short) @ v.T).float()
    return (x * 0.01).to(TYPES[dtype]).cuda()


SIZES = [(1, 1), (1, 7), (9, 1), (4, 5), (24, 25), (64, 64), (65, 63), (64, 576), (500, 2), (128, 600), (130, 500), (255, 256),
         (256, 256), (257, 300), (256, 2304), (1000, 333), (777, 1500), (64, 5000)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_orthogonalised_matrices_match_the_definition(rows, cols, dtype):
    print("orthogonalize", rows, cols, dtype, flush=True)
    for spectrum in ("noise", "falling"):
        matrix = _matrix(rows, cols, dtype, rows + cols, spectrum)
        got = ops.orthogonalize(matrix)
        _check(got, matrix)
        assert torch.equal(ops.orthogonalize(matrix), got)


@gpu
def test_lists_of_unlike_matrices():
    shapes = [(64, 147), (64, 576), (128, 64), (300, 700), (700, 300), (2, 512), (1, 1), (0, 4), (257, 257)] * 5
    matrices = [_matrix(r, c, list(TYPES)[i % 3], i) if r else torch.zeros((r, c), device="cuda") for i, (r, c) in enumerate(shapes)]
    got = ops.orthogonalize_many(matrices)
    assert len(got) == len(matrices) and ops.orthogonalize_many([]) == []
    for value, to, again in zip(matrices, got, ops.orthogonalize_many(matrices)):
        assert to.dtype is value.dtype and to.shape == value.shape and torch.equal(to, again)
        if value.numel():
            _check(to, value)
    narrow = [matrices[i] for i in (0, 1, 2, 5, 6)]  # no side of 64 or less is one of the others
    for value, to in zip(narrow, ops.orthogonalize_many(narrow)):
        _check(to, value)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_kernels_strides_and_results_in_place(dtype):
    kernel = _matrix(40, 27, dtype, 1).reshape(40, 3, 3, 3)
    got = ops.orthogonalize(kernel)
    _check(got, kernel)
    assert torch.equal(ops.orthogonalize(kernel.reshape(40, 27)), got.reshape(40, 27))
    wide = _matrix(70, 300, dtype, 2)
    part = wide[:, 11:211]
    _check(ops.orthogonalize(part), part)
    assert torch.equal(ops.orthogonalize(part.contiguous()), ops.orthogonalize(part))
    assert torch.equal(ops.orthogonalize(part.t()), ops.orthogonalize(part.t().contiguous()))
    _check(ops.orthogonalize(part.t()), part.t())
    want = ops.orthogonalize(wide)
    assert ops.orthogonalize(wide, out=wide) is wide and torch.equal(wide, want)


@gpu
def test_other_polynomials_and_steps():
    matrix = _matrix(90, 200, "float32", 3)
    for steps, coefficients in ((1, ops.COEFFICIENTS), (2, ops.COEFFICIENTS), (12, (1.5, -0.5, 0.0)), (6, (15 / 8, -10 / 8, 3 / 8))):
        options = dict(steps=steps, coefficients=coefficients)
        _check(ops.orthogonalize(matrix, **options), matrix, **options)
    orthogonal = ops.orthogonalize(matrix, steps=30, coefficients=(1.5, -0.5, 0.0)).double()
    assert float((orthogonal @ orthogonal.T - torch.eye(90, device="cuda")).abs().max()) < 1e-5


@gpu
def test_sizes_of_the_values_do_not_matter():
    base = _matrix(100, 170, "float32", 4)
    want = ops.orthogonalize(base, eps=0.0)
    for factor in (2.0 ** 100, 2.0 ** -100, 2.0 ** -126):  # the last leaves values below the normal range: not compared
        got = ops.orthogonalize(base * factor, eps=0.0)
        assert bool(got.isfinite().all())
        if factor > 2.0 ** -110:
            assert torch.equal(got, want)
    spike = torch.zeros((100, 170), device="cuda")
    spike[3, 5] = 1e30
    _check(ops.orthogonalize(spike), spike)
    tiny = _matrix(64, 100, "float32", 5) * 1e-9  # eps counts here
    _check(ops.orthogonalize(tiny), tiny)


@gpu
def test_zeros_infinities_and_nan():
    zeros = torch.zeros((70, 90), device="cuda")
    assert torch.equal(ops.orthogonalize(zeros), zeros)
    for bad in (float("nan"), float("inf"), float("-inf")):
        matrix = torch.randn((70, 90), device="cuda")
        matrix[69, 89] = bad
        other = torch.randn((80, 30), device="cuda")
        got = ops.orthogonalize_many([matrix, other])
        assert bool(got[0].isnan().all())
        _check(got[1], other)


@gpu
def test_streams_and_captured_graphs_have_workspaces_of_their_own():
    first, second = _matrix(300, 500, "float32", 6), _matrix(256, 800, "float32", 7)
    alone = [ops.orthogonalize(first), ops.orthogonalize(second)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        got = []
        for stream, matrix in zip(streams, (first, second)):
            with torch.cuda.stream(stream):
                got.append(ops.orthogonalize(matrix))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    graphs, held = [], []
    for matrix in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(ops.orthogonalize(matrix))
        graphs.append(graph)
    for _ in range(3):
        for stream, graph in zip(streams, graphs):  # side by side
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, alone))
        assert torch.equal(ops.orthogonalize(first), alone[0])


def test_refusals_without_a_gpu():
    with pytest.raises(TypeError, match="on the GPU"):
        ops.orthogonalize(torch.zeros((3, 4)))
    for options in (dict(steps=0), dict(steps=65), dict(coefficients=(1.0, 2.0)), dict(coefficients=(1.0, float("nan"), 0.0)),
                    dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(2.0, 0.0, 0.0), steps=4), dict(eps=-1.0),
                    dict(eps=float("inf"))):
        with pytest.raises(ValueError):
            ops.orthogonalize_many([], **options)


@pytest.mark.parametrize("steps,coefficients", [(1, (14.9, -44.5, 27.0)), (1, (12.0, -55.0, 46.0)), (1, (13.0, -30.0, 13.6)),
                                                (2, (13.0, -30.0, 13.6))])
def test_polynomials_whose_products_leave_the_range_are_refused(steps, coefficients):
    # Each keeps the values below 3.5 and a + b x^2 + c x^4 below 15, but b x^2 + c x^4 passes 16 on 0 .. 1.
    with pytest.raises(ValueError, match="out of range"):
        ops.orthogonalize_many([], steps=steps, coefficients=coefficients)


def test_polynomials_within_the_range_are_taken():
    for steps, coefficients in ((64, ops.COEFFICIENTS), (1, (12.507, -49.235, 38.123)), (1, (13.424, -50.472, 40.054)),
                                (5, (1.5, -0.5, 0.0)), (1, (2.0, 0.0, 0.0))):
        assert ops._polynomial(coefficients, steps) == (coefficients, steps)


@gpu
@pytest.mark.parametrize("coefficients", [(12.507, -49.235, 38.123), (13.424, -50.472, 40.054), (5.0, -17.0, 12.0)])
@pytest.mark.parametrize("side", [2, 130])
def test_products_near_the_end_of_the_range(side, coefficients):
    """Two singular values, one where |b x^2 + c x^4| is largest on 0 .. 1. With u = 2^-23, X is held to u and a product is
    formed to 2.5 u: lo is up to 2^-11 of its value, so lo lo up to 2 u, and a float32 rounding. So G = x^2 is held to 5.5 u
    (2 from X), b G + c G G to (8 |b| x^2 + 16 |c| x^4) u (5.5 and 11 from G, 2.5 for G G, half a u for a coefficient, its
    product and the sum, 1 for holding it), and with X's error, the product's and two roundings more the step's result to
    x (3 |a| + 13 |b| x^2 + 21 |c| x^4) u."""
    a, b, c = coefficients
    grid = torch.arange(1, 4097, dtype=torch.float64) / 4096
    x = float(grid[(b * grid ** 2 + c * grid ** 4).abs().argmax()])
    values = torch.tensor([x, (1.0 - x * x) ** 0.5], dtype=torch.float64)
    matrix = torch.zeros((side, side), device="cuda")
    matrix[0, 0], matrix[1, 1] = values.float()
    got = ops.orthogonalize(matrix, steps=1, coefficients=coefficients).cpu().double()
    want = _steps(matrix, torch.float64, steps=1, coefficients=coefficients)
    bound = values * (3 * abs(a) + 13 * abs(b) * values ** 2 + 21 * abs(c) * values ** 4) * 2.0 ** -23
    off = (got - want).abs()
    assert bool((off.diagonal()[:2] <= bound).all())
    got[0, 0] = got[1, 1] = 0.0
    assert not bool(got.any())


@gpu
def test_refusals():
    matrix = torch.zeros((3, 4), device="cuda")
    for bad in (matrix.double(), matrix.int(), [[1.0]]):
        with pytest.raises(TypeError):
            ops.orthogonalize(bad)
    for bad in (matrix[0], matrix[0, 0], torch.zeros((1, 1), device="cuda").expand(1, (1 << 20) + 1)):
        with pytest.raises(ValueError):
            ops.orthogonalize(bad)
    for out in (matrix.half(), matrix.t(), matrix.cpu(), torch.zeros((3, 8), device="cuda")[:, :4]):
        with pytest.raises(ValueError, match="out"):
            ops.orthogonalize(matrix, out=out)
    with pytest.raises(ValueError, match="out"):
        ops.orthogonalize_many([matrix], out=[])
    held = torch.randn(40, device="cuda")
    first, second = held[:12].view(3, 4), held[20:32].view(3, 4)
    for out in ([first, first], [second, first], [held[16:28].view(3, 4), first], [held[10:22].view(3, 4), second]):
        with pytest.raises(ValueError, match="share no memory"):
            ops.orthogonalize_many([first, second], out=out)
    want = [ops.orthogonalize(first.clone()), ops.orthogonalize(second.clone())]
    moved = held.clone()  # a result that lies across its own matrix: all are read before any result is written
    assert torch.equal(ops.orthogonalize(moved[:12].view(3, 4), out=moved[5:17].view(3, 4)), want[0])
    got = ops.orthogonalize_many([first, second], out=[first, second])
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=0.0, atol=1e-5)


@pytest.mark.parametrize("eps", [1e-50, 1e39, -1e-50, -1.0, float("inf"), float("nan")])
def test_an_eps_that_float32_does_not_hold_is_refused(eps):
    for call in (lambda: ops.orthogonalize_many([], eps=eps), lambda: ops.muon_update_many([], eps=eps)):
        with pytest.raises(ValueError, match="eps"):
            call()


@gpu
def test_zeros_stay_zeros_for_the_smallest_eps():
    zeros = torch.zeros((3, 70), device="cuda")
    assert torch.equal(ops.orthogonalize(zeros, eps=2.0 ** -149), zeros)
    matrix = _matrix(40, 70, "float32", 8)
    assert torch.equal(ops.orthogonalize(matrix, eps=2.0 ** -149), ops.orthogonalize(matrix, eps=0.0))


@gpu
@pytest.mark.parametrize("rows,cols,count", [(500, 500, 4), (512, 4608, 2), (1024, 4096, 2)])
def test_errors_of_long_sums_are_those_of_float32_steps(rows, cols, count):
    """Root mean square over matrices. Of the errors of float32 steps, those of the sums are no larger here, which round a
    sum once for 16 products; those of a value's rounding as hi + lo are as a rule the same (2^-24 of a power of two, and
    2^-23 at most), and what is left out, lo lo, is as a rule 2^-25 of a product. Two independent errors for one: 2^.5."""
    ours = theirs = 0.0
    for seed in range(count):
        matrix = _matrix(rows, cols, "float32", seed)
        want = _steps(matrix, torch.float64)
        ours += float((ops.orthogonalize(matrix).cpu().double() - want).square().sum())
        theirs += float((_steps(matrix, torch.float32).double() - want).square().sum())
    print(f"{rows} x {cols}: {(ours / theirs) ** 0.5:.2f} times float32's error", flush=True)
    assert ours <= 2 * theirs


EXACT = dict(coefficients=(3.4375, -4.75, 2.03125))  # float32 holds them
THIN = [(1, 1), (1, 7), (2, 2), (512, 2), (2, 513), (8, 8), (3, 1025), (8, 3000), (5000, 7), (6, 70001), (200003, 4), (1, 1 << 20)]


def _check_thin(got, matrix, **options):
    """A matrix of at most 8 rows or columns is formed in 64 bits: an element is off by its rounding to float32 and to its
    type, and by 2^-40 of the largest for 64-bit steps on both sides, whose errors are raised 500 times at most."""
    want = _steps(matrix, torch.float64, **{**EXACT, **options})
    info = torch.finfo(matrix.dtype)
    half_step = info.eps / 2 + (0.0 if matrix.dtype is torch.float32 else 2.0 ** -24)
    bound = half_step * want.abs().clamp(min=info.smallest_normal) + 2.0 ** -40 * want.abs().max()
    assert got.dtype is matrix.dtype and got.shape == matrix.shape
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", THIN)
def test_matrices_of_a_few_rows_are_rounded_once(rows, cols, dtype):
    print("orthogonalize", rows, cols, dtype, flush=True)
    for spectrum in ("noise", "falling"):
        matrix = _matrix(rows, cols, dtype, rows + cols, spectrum)
        got = ops.orthogonalize(matrix, **EXACT)
        _check_thin(got, matrix)
        _check_thin(ops.orthogonalize(matrix, steps=1, **EXACT), matrix, steps=1)
        assert torch.equal(ops.orthogonalize(matrix, **EXACT), got)
        wide = torch.full((rows, cols + 5), 7.0, dtype=TYPES[dtype], device="cuda")
        wide[:, 3:3 + cols] = matrix
        assert torch.equal(ops.orthogonalize(wide[:, 3:3 + cols], **EXACT), got)
        assert ops.orthogonalize(matrix, out=matrix, **EXACT) is matrix and torch.equal(matrix, got)


@gpu
def test_matrices_of_a_few_rows_among_others():
    shapes = [(512, 2), (64, 100), (3, 70), (130, 140), (8, 9), (9, 8), (9, 9), (1, 5)] * 12
    matrices = [_matrix(r, c, list(TYPES)[i % 3], i) for i, (r, c) in enumerate(shapes)]
    native.stream_workspace(1, torch.float64).view(torch.int64).fill_(-1)
    for value, to in zip(matrices, ops.orthogonalize_many(matrices, **EXACT)):
        if min(value.shape) <= 8:
            _check_thin(to, value)
            assert torch.equal(ops.orthogonalize(value, **EXACT), to)
        else:
            _check(to, value, **EXACT)
    held = torch.randn(5000, device="cuda")  # a result that lies across its own matrix
    want = ops.orthogonalize(held[:4000].clone().view(4, 1000))
    assert torch.equal(ops.orthogonalize(held[:4000].view(4, 1000), out=held[777:4777].view(4, 1000)), want)


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 9), (2, 512), (700, 8)])
def test_zeros_infinities_nan_and_sizes_of_a_few_rows(rows, cols):
    zeros = torch.zeros((rows, cols), device="cuda")
    assert torch.equal(ops.orthogonalize(zeros), zeros)
    for bad in (float("nan"), float("inf"), float("-inf")):
        matrix = torch.randn((rows, cols), device="cuda")
        matrix[-1, -1] = bad
        assert bool(ops.orthogonalize(matrix).isnan().all())
    base = _matrix(rows, cols, "float32", 4)
    want = ops.orthogonalize(base, eps=0.0)
    for factor in (2.0 ** 100, 2.0 ** -100):
        assert torch.equal(ops.orthogonalize(base * factor, eps=0.0), want)
    assert bool(ops.orthogonalize(base * 2.0 ** -126, eps=0.0).isfinite().all())


@gpu
@pytest.mark.parametrize("rows,cols,count", [(40, 70, 16), (64, 147, 8), (64, 576, 8)])
def test_errors_of_few_rows_are_those_of_float32_steps(rows, cols, count):
    """Root mean square over matrices. In float32 steps a value held is rounded by .58 of 2^-24 of its power of two (the
    standard deviation of a rounding), and the sums and the polynomial's three operations add at least as much again. Here a
    value is held as hi + lo, rounded by .87 of that (lo has 11 bits of what hi leaves), and nothing else is lost:
    ((.87^2 + .58^2) / (2 .58^2))^.5 < 1.3."""
    ours = theirs = 0.0
    for seed in range(count):
        matrix = _matrix(rows, cols, "float32", seed)
        want = _steps(matrix, torch.float64)
        ours += float((ops.orthogonalize(matrix).cpu().double() - want).square().sum())
        theirs += float((_steps(matrix, torch.float32).double() - want).square().sum())
    print(f"{rows} x {cols}: {(ours / theirs) ** 0.5:.2f} times float32's error", flush=True)
    assert ours <= 1.3 ** 2 * theirs


@gpu
def test_small_matrices_ask_for_little_workspace():
    assert ops._workspace(((4, 4),)) < 1 << 16 and ops._muon_workspace(((4, 4), (2, 9))) < 1 << 17
    assert ops._workspace(((64, 576),)) < 1 << 21 and ops._workspace(((64, 576),) * 40) < 30 << 21
    assert ops._workspace(((1, 1 << 20),)) < 5 << 20


@gpu
def test_few_rows_on_two_streams_and_in_graphs():
    lists = [[_matrix(2, 3000, "float32", 1), _matrix(90, 80, "float32", 2)], [_matrix(70001, 5, "float32", 3)]]
    alone = [ops.orthogonalize_many(matrices) for matrices in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lists]
    graphs, held = [], []
    for matrices in lists:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(ops.orthogonalize_many(matrices))
        graphs.append(graph)
    for _ in range(4):
        eager = []
        for stream, graph, matrices in zip(streams, graphs, lists):
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(ops.orthogonalize_many(matrices))
        torch.cuda.synchronize()
        for got, want in zip([*held, *eager], [*alone, *alone]):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
