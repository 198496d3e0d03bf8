"""Group norm with an activation, channels last, on libmfhip against the definition in 64 bits.

Bounds (u = 2^-24). A sum over `count` values has at most count / 64 + 40 additions in a chain; a = (count / 64 +
40) u bounds its relative error against the sum of magnitudes. The mean is off by at most a mean|x|, the
variance by the square of that and a relative 2 a, inv_std by a relative a + 4 u. These carry into xhat, u, y and
the gradients by the derivatives of the formulas; SiLU's slope is at most 1.1 and its slope's slope 1/2, its
sigmoid within (2 |u| + 6) u. Where a ReLU's input may lie on either side of 0 its gradient may be dy or 0.
"""

import pytest
import torch

import myflows_amd as mf
from myflows_amd import group_norm as ops

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# Half a unit in the last place of a correctly rounded result, relative and (below the normal range) absolute.
ROUNDING = {t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) for t in TYPES.values()}

gpu = pytest.mark.gpu

SHAPES = [
    # n, positions, channels, groups: single positions and channels, odd sizes, every vector width, one group,
    # a group a channel, groups across vectors, samples in one workgroup and over many, few and many samples
    (1, 1, 8, 1), (2, 1, 64, 8), (3, 7, 3, 1), (2, 5, 6, 6), (1, 20, 512, 32), (5, 33, 15, 5), (2, 100, 90, 6),
    (4, 1131, 64, 32), (1, 3000, 96, 3), (2, 257, 1000, 8), (1, 16384, 32, 4), (3, 5000, 130, 13), (70, 50, 48, 16),
    (1, 1, 1024, 1024), (2, 9, 2050, 2), (1, 40000, 8, 8), (1, 2000, 640, 1), (300, 16, 32, 2), (1, 70000, 33, 11),
]


def _data(n, positions, channels, dtype, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, positions, channels), generator=g) * (0.5 + torch.rand(channels, generator=g))
    x = (x + torch.randn(channels, generator=g) + offset).to(TYPES[dtype])
    dy = torch.randn((n, positions, channels), generator=g).to(TYPES[dtype])
    gamma, beta = 1.0 + 0.3 * torch.randn(channels, generator=g), 0.2 * torch.randn(channels, generator=g)
    return x.cuda(), dy.cuda(), gamma.cuda(), beta.cuda()


def _near(got, want, bound, name):
    off = (got.detach().cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"{name}: off by up to {float((off - bound).max()):.3e} beyond its bound"


def _rounded(bound, want, dtype):
    unit, least = ROUNDING[dtype]
    return bound + unit * (want.abs() + bound) + least


def _reference(x, gamma, beta, groups, eps, act):
    n, c = x.shape[0], x.shape[-1]
    flat = x.detach().cpu().double().reshape(n, -1, groups, c // groups)
    gamma, beta = (v.cpu().double().reshape(groups, -1) for v in (gamma, beta))
    count = flat.shape[1] * flat.shape[3]
    a = (count / 64 + 40) * U
    mean = flat.mean(dim=(1, 3), keepdim=True)
    var = (flat - mean).square().mean(dim=(1, 3), keepdim=True)
    inv = (var + eps).rsqrt()
    mean_err = a * flat.abs().mean(dim=(1, 3), keepdim=True)
    inv_rel = a + 4 * U + mean_err.square() * inv.square()
    hat = (flat - mean) * inv
    hat_err = inv * (U * (flat.abs() + mean.abs()) + mean_err) + hat.abs() * (inv_rel + 2 * U)
    u = hat * gamma + beta
    u_err = gamma.abs() * hat_err + 2 * U * (u.abs() + beta.abs())
    sig = torch.sigmoid(u)
    if act == "silu":
        y, y_err = u * sig, 1.1 * u_err + (u * sig).abs() * (2 * u.abs() + 6) * U
    elif act == "relu":
        y, y_err = u.relu(), u_err
    else:
        y, y_err = u, u_err
    return dict(flat=flat, mean=mean, inv=inv, mean_err=mean_err, inv_rel=inv_rel, hat=hat, hat_err=hat_err, u=u, u_err=u_err,
                sig=sig, y=y, y_err=y_err, a=a, gamma=gamma, count=count)


def _check(x, dy, gamma, beta, groups, act, eps=1e-5, old=None):
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, groups, eps=eps, activation=act)
    f = _reference(x, gamma, beta, groups, eps, act)
    n, c = x.shape[0], x.shape[-1]
    assert y.dtype == x.dtype and y.shape == x.shape
    _near(mean, f["mean"].reshape(n, groups), (f["mean_err"] + U * f["mean"].abs()).reshape(n, groups), "mean")
    _near(inv, f["inv"].reshape(n, groups), (f["inv"] * f["inv_rel"]).reshape(n, groups), "inv_std")
    want = f["y"].reshape(x.shape)
    _near(y, want, _rounded(f["y_err"].reshape(x.shape), want, x.dtype), "y")

    add = old is not None
    targets = old if add else (torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta))
    before = [t.detach().cpu().double() if add else torch.zeros_like(t.cpu(), dtype=torch.float64) for t in targets]
    ops.group_norm_backward(x, dy, gamma, beta, mean, inv, activation=act, x_grad=targets[0], gamma_grad=targets[1],
                            beta_grad=targets[2], accumulate=(add, add, add))
    d, u, hat = dy.cpu().double().reshape(f["flat"].shape), f["u"], f["hat"]
    if act == "silu":
        slope = f["sig"] * (1 + u * (1 - f["sig"]))
        du, du_err = d * slope, d.abs() * (0.5 * f["u_err"] + (2 * u.abs() + 8) * U * f["sig"] * (1 + u.abs()))
    elif act == "relu":
        du = torch.where(u > 0, d, torch.zeros_like(d))
        du_err = torch.where(u.abs() <= f["u_err"], d.abs(), torch.zeros_like(d))
    else:
        du, du_err = d, torch.zeros_like(d)
    gd, gd_err = f["gamma"] * du, f["gamma"].abs() * (du_err + U * du.abs())
    over = dict(dim=(1, 3), keepdim=True)
    first, second = gd.mean(**over), (gd * hat).mean(**over)
    first_err = gd_err.mean(**over) + f["a"] * gd.abs().mean(**over)
    second_err = (gd_err * hat.abs() + gd.abs() * f["hat_err"]).mean(**over) + f["a"] * (gd * hat).abs().mean(**over)
    dx = f["inv"] * (gd - first - hat * second)
    dx_err = f["inv"] * (gd_err + first_err + hat.abs() * second_err + second.abs() * f["hat_err"]) + (f["inv_rel"] + 6 * U) * f[
        "inv"] * (gd.abs() + first.abs() + (hat * second).abs())
    want = dx.reshape(x.shape) + before[0]
    extra = U * want.abs() if add else 0.0
    _near(targets[0], want, _rounded(dx_err.reshape(x.shape) + extra, want, x.dtype), "dx")
    rows = (n * f["flat"].shape[1] / 64 + 40) * U
    for name, target, old_value, terms, err in (
            ("dgamma", targets[1], before[1], du * hat, du_err * hat.abs() + du.abs() * f["hat_err"]),
            ("dbeta", targets[2], before[2], du, du_err)):
        want = terms.sum(dim=(0, 1)).reshape(c) + old_value
        bound = (err.sum(dim=(0, 1)) + rows * terms.abs().sum(dim=(0, 1))).reshape(c) + 2 * U * want.abs()
        _near(target, want, bound, name)
    return y, mean, inv


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,positions,channels,groups", SHAPES)
def test_group_norm_matches_the_definition(n, positions, channels, groups, dtype):
    for act in (None, "relu", "silu"):
        print("group_norm", n, positions, channels, groups, dtype, act, flush=True)
        x, dy, gamma, beta = _data(n, positions, channels, dtype, channels + positions)
        _check(x, dy, gamma, beta, groups, act)


@gpu
@pytest.mark.parametrize("n,positions,channels,groups", [(2, 33, 24, 3), (3, 6000, 64, 8)])
def test_gradients_are_added_to_what_is_there(n, positions, channels, groups):
    x, dy, gamma, beta = _data(n, positions, channels, "float32", 1)
    g = torch.Generator().manual_seed(2)
    old = tuple(torch.randn(t.shape, generator=g).cuda() for t in (x, gamma, beta))
    _check(x, dy, gamma, beta, groups, "silu", old=old)


@gpu
@pytest.mark.parametrize("n,positions,channels,groups", [(2, 40, 32, 4), (2, 9000, 32, 4)])
def test_a_large_mean_does_not_swallow_the_variance(n, positions, channels, groups):
    """Values near 1000 with a spread of 1: the bound follows from mean|x| and stays at 1e-3 of the spread."""
    x, dy, gamma, beta = _data(n, positions, channels, "float32", 7, offset=1000.0)
    _check(x, dy, gamma, beta, groups, None)


@gpu
@pytest.mark.parametrize("positions", (50, 20000))
def test_one_far_value_does_not_swallow_the_variance(positions):
    x, dy, gamma, beta = _data(2, positions, 16, "float32", 8)
    x[0, 0, 0] = 3.0e4
    _check(x, dy, gamma, beta, 2, None)


@gpu
def test_a_constant_group_and_shapes_with_more_dimensions():
    x = torch.full((2, 4, 5, 8), 3.0, device="cuda")
    gamma, beta = torch.ones(8, device="cuda"), torch.full((8,), 0.5, device="cuda")
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 2)
    assert torch.equal(y, torch.full_like(x, 0.5)) and torch.equal(mean, torch.full_like(mean, 3.0))
    x, dy, gamma, beta = _data(2, 20, 8, "float32", 3)
    a = ops.group_norm_forward(x, gamma, beta, 2)[0]
    b = ops.group_norm_forward(x.reshape(2, 4, 5, 8), gamma, beta, 2)[0]
    assert torch.equal(a, b.reshape(a.shape))


@gpu
@pytest.mark.parametrize("positions", (40, 9000))
def test_nan_and_infinity_stay_in_their_group(positions):
    x, dy, gamma, beta = _data(3, positions, 12, "float32", 4)
    x[1, positions // 2, 5] = float("nan")
    x[2, 0, 0] = float("inf")
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 3)
    bad = torch.isnan(y).any(dim=1).reshape(3, 3, 4).any(dim=2).cpu()
    assert bad.tolist() == [[False] * 3, [False, True, False], [True, False, False]]
    dx = torch.empty_like(x)
    ops.group_norm_backward(x, dy, gamma, beta, mean, inv, x_grad=dx, accumulate=(False,) * 3)
    assert torch.equal(torch.isnan(dx).any(dim=1).reshape(3, 3, 4).any(dim=2).cpu(), bad)


@gpu
@pytest.mark.parametrize("positions", (60, 9000))
def test_a_sample_does_not_depend_on_its_batch(positions):
    x, dy, gamma, beta = _data(5, positions, 32, "bfloat16", 5)
    whole = ops.group_norm_forward(x, gamma, beta, 4, activation="silu")
    for i in (0, 4):
        alone = ops.group_norm_forward(x[i:i + 1], gamma, beta, 4, activation="silu")
        for a, b in zip(whole, alone):
            assert bool(((a[i:i + 1].float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -10).all())


@gpu
def test_samples_beyond_32_bit_offsets():
    """Three samples of 2^30 elements: the last one's results are its own, alone, on the same plan."""
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.empty((3, 2 ** 20, 1024), dtype=torch.bfloat16, device="cuda")
    x[2] = torch.randn((2 ** 20, 1024), generator=g, device="cuda", dtype=torch.bfloat16)
    x[:2] = 1.0
    gamma, beta = torch.rand(1024, generator=g, device="cuda"), torch.rand(1024, generator=g, device="cuda")
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 8, activation="silu")
    alone = ops.group_norm_forward(x[2:], gamma, beta, 8, activation="silu")
    assert bool(((mean[2] - alone[1][0]).abs() <= 2.0 ** -20).all()) and bool(((inv[2] / alone[2][0] - 1).abs() <= 2.0 ** -18).all())
    assert bool(((y[2].float() - alone[0][0].float()).abs() <= 2.0 ** -6 * alone[0][0].float().abs() + 2.0 ** -8).all())
    del alone
    dx = torch.empty_like(x)
    ops.group_norm_backward(x, x, gamma, beta, mean, inv, activation="silu", x_grad=dx, accumulate=(False,) * 3)
    want = torch.empty_like(x[2:])
    ops.group_norm_backward(x[2:], x[2:], gamma, beta, mean[2:], inv[2:], activation="silu", x_grad=want, accumulate=(False,) * 3)
    assert bool(((dx[2].float() - want[0].float()).abs() <= 2.0 ** -6 * want[0].float().abs() + 2.0 ** -8).all())


def _same_as_alone(x, dy, gamma, beta, groups, parts):
    """A call's results for these samples against calls on them alone (the same plan, so the same bits); dbeta of a
    gradient of ones against the number of values, dgamma against the sum of xhat in 64 bits."""
    n, positions, channels = x.shape
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, groups)
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    ops.group_norm_backward(x, dy, gamma, beta, mean, inv, x_grad=dx, gamma_grad=dgamma, beta_grad=dbeta, accumulate=(False,) * 3)
    for part in parts:
        alone = ops.group_norm_forward(x[part], gamma, beta, groups)
        for a, b in zip((y, mean, inv), alone):
            assert torch.equal(a[part], b)
        want = torch.empty_like(x[part])
        ops.group_norm_backward(x[part], dy[part], gamma, beta, *alone[1:], x_grad=want, accumulate=(False,) * 3)
        assert torch.equal(dx[part], want)
    ops.group_norm_backward(x, torch.ones_like(x), gamma, beta, mean, inv, gamma_grad=dgamma, beta_grad=dbeta, accumulate=(False,) * 3)
    assert bool((dbeta == n * positions).all())  # whole numbers that float32 holds
    spread = lambda v: v.repeat_interleave(channels // groups, dim=1).double()  # noqa: E731
    total, size = 0.0, 0.0
    for first in range(0, n, 2 ** 24 // channels):
        rows = slice(first, first + 2 ** 24 // channels)
        hat = (x[rows].double() - spread(mean[rows])[:, None]) * spread(inv[rows])[:, None]
        total, size = total + hat.sum(dim=(0, 1)), size + hat.abs().sum(dim=(0, 1))
    # A column's 16 runs of samples are added in order, then the runs: n / 16 + 20 additions; xhat takes two roundings.
    assert bool(((dgamma - total).abs() <= (n / 16 + 40) * U * size).all())


@gpu
def test_wide_groups_of_more_samples_than_a_launch_takes():
    """n C = 2100 x 65536: the join of the column sums takes 2^21 threads a sample, so the samples go in two slices."""
    print("wide groups, sliced", flush=True)
    g = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn((2100, 1, 65536), generator=g, device="cuda").half()
    dy = torch.randn((2100, 1, 65536), generator=g, device="cuda").half()
    gamma, beta = torch.rand(65536, generator=g, device="cuda"), torch.rand(65536, generator=g, device="cuda")
    _same_as_alone(x, dy, gamma, beta, 1, (slice(0, 3), slice(2045, 2050), slice(2090, 2100)))


@gpu
def test_more_samples_than_a_launch_takes():
    """2^24 + 8 samples of one position and two channels: a workgroup each would be 2^32 threads and more."""
    print("many samples, sliced", flush=True)
    n = 2 ** 24 + 8
    g = torch.Generator(device="cuda").manual_seed(22)
    x = torch.randn((n, 1, 2), generator=g, device="cuda").half()
    dy = torch.randn((n, 1, 2), generator=g, device="cuda").half()
    gamma, beta = torch.rand(2, generator=g, device="cuda"), torch.rand(2, generator=g, device="cuda")
    _same_as_alone(x, dy, gamma, beta, 1, (slice(0, 1000), slice(n - 1009, n)))


@gpu
def test_single_gradients_and_unaligned_views():
    x, dy, gamma, beta = _data(4, 300, 64, "float16", 6)
    shifted = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 8, activation="silu")
    y2, mean2, inv2 = ops.group_norm_forward(shifted, gamma, beta, 8, activation="silu")
    assert bool(((y.float() - y2.float()).abs() <= 2.0 ** -9 * y.float().abs() + 2.0 ** -16).all())
    every = (torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta))
    names = ("x_grad", "gamma_grad", "beta_grad")
    ops.group_norm_backward(x, dy, gamma, beta, mean, inv, activation="silu", accumulate=(False,) * 3,
                            **dict(zip(names, every)))
    for name, target in zip(names, every):
        alone = torch.empty_like(target)
        ops.group_norm_backward(x, dy, gamma, beta, mean, inv, activation="silu", accumulate=(False,) * 3, **{name: alone})
        assert torch.equal(alone, target), name
    out = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
    ops.group_norm_backward(shifted, dy, gamma, beta, mean, inv, activation="silu", x_grad=out, accumulate=(False,) * 3)
    assert bool(((out.float() - every[0].float()).abs() <= 2.0 ** -9 * every[0].float().abs() + 2.0 ** -14).all())


@gpu
def test_gradient_matches_differences():
    """Central differences of sum(dy y) in a direction of length 1: values below 64 within 2^-18, third derivatives of
    the normalised, activated sum below 64 in these groups of 96; a step of 1/64."""
    x, dy, gamma, beta = _data(2, 12, 24, "float32", 9)
    g = torch.Generator().manual_seed(10)
    v = torch.randn(x.shape, generator=g).cuda()
    v /= v.norm()
    step = 1 / 64
    value = lambda t: float((ops.group_norm_forward(t, gamma, beta, 3, activation="silu")[0].double() * dy.double()).sum())  # noqa: E731
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 3, activation="silu")
    dx = torch.empty_like(x)
    ops.group_norm_backward(x, dy, gamma, beta, mean, inv, activation="silu", x_grad=dx, accumulate=(False,) * 3)
    slope = (value(x + step * v) - value(x - step * v)) / (2 * step)
    assert abs(slope - float((dx * v).double().sum())) <= 64 * step * step / 6 + 2.0 ** -18 * 64


@gpu
def test_group_norm_layer_in_a_graph():
    x, dy, _, _ = _data(6, 10, 16, "float32", 11)
    rows = mf.Variable(x.reshape(60, 16), requires_grad=True)
    layer = mf.GroupNorm(4, 16, activation="silu", positions=10)
    layer.gamma.value = 1.0 + 0.1 * torch.arange(16, device="cuda")
    weight = mf.Variable(dy.reshape(60, 16), requires_grad=False)
    out = layer(rows)
    loss = mf.MSELoss(out, weight)
    graph = mf.Graph(loss)
    graph.forward()
    graph.backward()
    y, mean, inv = ops.group_norm_forward(x, layer.gamma.value, layer.beta.value, 4, activation="silu")
    assert torch.equal(out.value, y.reshape(60, 16))
    seed = (2.0 * (y - dy) / y.numel())
    grads = (torch.empty_like(x), torch.empty(16, device="cuda"), torch.empty(16, device="cuda"))
    ops.group_norm_backward(x, seed, layer.gamma.value, layer.beta.value, mean, inv, activation="silu", x_grad=grads[0],
                            gamma_grad=grads[1], beta_grad=grads[2], accumulate=(False,) * 3)
    for node, want in zip((rows, layer.gamma, layer.beta), grads):
        got = node.grad.reshape(want.shape)
        assert bool(((got - want).abs() <= 2.0 ** -18 * want.abs().max()).all())


@gpu
@pytest.mark.parametrize("n,positions,channels,groups", [
    (4096, 1, 64, 4), (300, 16, 32, 2), (16, 405, 90, 6), (2, 9000, 64, 8), (3, 20000, 33, 3), (2, 5, 40000, 2)])
def test_the_relu_gate_of_the_gradient_is_that_of_the_output(n, positions, channels, groups):
    """The gradient passes exactly where y > 0. beta cancels gamma xhat of one position a channel up to its
    rounding, so that many u lie within a rounding of 0; dy = 1 and dbeta count what passes."""
    x, _, gamma, _ = _data(n, positions, channels, "float32", 13)
    x = x.round(decimals=1)  # many equal values
    _, mean, inv = ops.group_norm_forward(x, gamma, torch.zeros_like(gamma), groups)
    per = channels // groups
    spread = lambda v: v[0].repeat_interleave(per)  # noqa: E731
    beta = -gamma * ((x[0, 0] - spread(mean)) * spread(inv))
    x[:] = x[:1, :1]  # of every sample and position; the statistics are those that the forward takes
    x += torch.arange(positions, device="cuda").reshape(1, -1, 1) % 3 * 0.25
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, groups, activation="relu")
    beta = -gamma * ((x[0, 0] - spread(mean)) * spread(inv))
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, groups, activation="relu")
    grads = torch.empty_like(gamma), torch.empty_like(gamma)
    ops.group_norm_backward(x, torch.ones_like(x), gamma, beta, mean, inv, activation="relu", gamma_grad=grads[0],
                            beta_grad=grads[1], accumulate=(False,) * 3)
    assert torch.equal(grads[1], (y > 0).sum(dim=(0, 1)).float())  # whole numbers below 2^24: exact


@gpu
def test_no_samples_and_refusals():
    gamma, beta = torch.ones(6, device="cuda"), torch.zeros(6, device="cuda")
    empty = torch.empty((0, 4, 6), device="cuda")
    y, mean, inv = ops.group_norm_forward(empty, gamma, beta, 2)
    assert y.shape == (0, 4, 6) and mean.shape == (0, 2)
    dg = torch.ones(6, device="cuda")
    ops.group_norm_backward(empty, empty, gamma, beta, mean, inv, gamma_grad=dg, accumulate=(False,) * 3)
    assert not dg.any()
    x = torch.zeros((2, 4, 6), device="cuda")
    for bad in (4, 0, -1):
        with pytest.raises(ValueError):
            ops.group_norm_forward(x, gamma, beta, bad)
    with pytest.raises(ValueError):
        ops.group_norm_forward(x, gamma[:3], beta, 2)
    with pytest.raises(ValueError):
        ops.group_norm_forward(x, gamma, beta, 2, activation="tanh")
    with pytest.raises(ValueError):
        ops.group_norm_forward(x, gamma, beta, 2, eps=-1.0)
    with pytest.raises(ValueError):
        ops.group_norm_forward(x[:, :0], gamma, beta, 2)
    with pytest.raises(TypeError):
        ops.group_norm_forward(x.double(), gamma, beta, 2)
    with pytest.raises(TypeError):
        ops.group_norm_forward(x, gamma.half(), beta, 2)
    y, mean, inv = ops.group_norm_forward(x, gamma, beta, 2)
    with pytest.raises(ValueError):
        ops.group_norm_backward(x, x[:1], gamma, beta, mean, inv, x_grad=torch.empty_like(x))
    with pytest.raises(ValueError):
        ops.group_norm_backward(x, x, gamma, beta, mean, inv, x_grad=torch.empty_like(x).half())
    with pytest.raises(ValueError):
        ops.group_norm_backward(x, x, gamma, beta, mean[:1], inv, x_grad=torch.empty_like(x))
    with pytest.raises(ValueError):
        mf.Graph(mf.GroupNorm(2, 6, positions=5)(mf.Variable(torch.zeros((7, 6), device="cuda")))).forward()
    lib = mf.native._library()
    assert lib.mfh_group_norm_workspace(1, 1, 6, 4, 0, 0) == -1 and lib.mfh_group_norm_workspace(1, 0, 6, 2, 0, 0) == -1


def test_host_tensors_are_refused():
    with pytest.raises(TypeError):
        ops.group_norm_forward(torch.zeros((1, 2, 4)), torch.ones(4), torch.zeros(4), 2)
    with pytest.raises(ValueError):
        mf.Graph(mf.GroupNorm(2, 4)(mf.Variable(torch.zeros((1, 2, 4))))).forward()
    with pytest.raises(ValueError):
        mf.GroupNorm(3, 4)
