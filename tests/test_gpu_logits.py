"""Rows of logits on libmfhip against the definitions in 64 bits: log probabilities with entropy and top
alternatives, the distillation loss, their gradients and their Graph losses.

Bounds (u = 2^-24). A term e^(z - m) takes one rounding of the difference, one of its product with log2 e and
the exp's own two ulp: a relative error of (2 |z - m| + 4) u, where terms below e^-40 of the largest do not
count. A thread's chain of additions has at most vocab / 64 + 20 links. So s is within S = (104 + vocab / 64) u
of itself, ln s within S + u |ln s|, and the values formed from them as written at each check. A half-precision
gradient adds its own rounding (2^-8 of a bfloat16, 2^-11 of a float16, 2^-25 below float16's normal range).
"""

import numpy as np
import pytest
import torch

import myflows_amd as mf
from myflows_amd import logits as ops

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# Half a unit in the last place of a correctly rounded result, relative and (below the normal range) absolute.
ROUNDING = {name: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) for name, t in TYPES.items()}
NEG = float("-inf")

gpu = pytest.mark.gpu


def _z(rows, vocab, dtype, seed, pad=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((rows, vocab + pad), generator=g) * scale
    z[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 6.0
    return z.to(TYPES[dtype]).cuda()[:, :vocab], g


def _exact(z):
    """(d = z - m, s, p, H) in 64 bits with the conventions of an empty row."""
    z = z.detach().cpu().double()
    m = z.amax(dim=1, keepdim=True)
    d = torch.where(z == NEG, torch.full_like(z, NEG), z - torch.where(m == NEG, torch.zeros_like(m), m))
    e = d.exp()
    s = e.sum(dim=1, keepdim=True)
    p = torch.where(s > 0, e / s, torch.zeros_like(e))
    log_p = torch.where(s > 0, d - s.log(), torch.full_like(d, NEG))
    h = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(dim=1)
    return d, s[:, 0], p, log_p, h, m[:, 0]


def _top(z, k):
    z = z.detach().cpu().double().numpy()
    ids = np.stack([np.lexsort((np.arange(z.shape[1]), -row))[:k] for row in z]) if len(z) else np.zeros((0, k), int)
    return torch.as_tensor(ids)


def _sum_error(vocab):
    return (104 + vocab / 64) * U


def _near(got, want, bound, name):
    got = got.detach().cpu().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    worst = (off - bound).max() if off.numel() else torch.tensor(0.0)
    assert bool((off <= bound).all()), f"{name}: off by up to {float(worst):.3e} beyond its bound"


def _check_forward(r, z, tokens, top):
    d, s, p, log_p, h, m = _exact(z)
    vocab = z.shape[1]
    err = _sum_error(vocab)
    ln_s = torch.where(s > 0, s.log(), torch.zeros_like(s))
    log_sum = torch.where(s > 0, m + ln_s, torch.full_like(s, NEG))
    base = err + 4 * U * ln_s.abs()
    _near(r.log_sum, log_sum, base + 2 * U * torch.nan_to_num(log_sum, neginf=0.0).abs(), "log_sum")
    _near(r.entropy, h, err * (1 + 2 * (h + ln_s.abs())) + 4 * U * (h + ln_s.abs()), "entropy")
    if tokens is not None:
        t = tokens.cpu().long()
        lp = torch.where(t >= 0, log_p[torch.arange(len(t)), t.clamp(min=0)], torch.zeros_like(h))
        lp = lp.float().double()  # a difference of the largest and the lowest float32 lies beyond float32: -inf
        _near(r.log_prob, lp, base + 4 * U * torch.nan_to_num(lp, neginf=0.0).abs(), "log_prob")
    else:
        assert r.log_prob is None
    if top:
        ids = _top(z, top)
        assert torch.equal(r.top_ids.cpu().long(), ids)
        want = log_p.gather(1, ids).float().double()
        _near(r.top_log_probs, want, base[:, None] + 4 * U * torch.nan_to_num(want, neginf=0.0).abs(), "top_log_probs")
    else:
        assert r.top_ids is None and r.top_log_probs is None


FORWARD = [
    # rows, vocab, top, pad: one logit, odd and unaligned sizes, each size class of the kernels, splits of a row
    (1, 1, 1, 0), (3, 2, 2, 0), (5, 17, 17, 3), (4, 64, 64, 0), (7, 65, 20, 1), (64, 1000, 5, 0), (33, 1001, 64, 7),
    (300, 2, 0, 0), (2, 2049, 20, 5), (9, 4097, 33, 0), (3, 8193, 64, 1), (1, 50021, 20, 0), (2, 131072, 64, 0),
    (2, 131071, 7, 1), (700, 9000, 20, 0), (2100, 600, 3, 0), (3000, 4500, 1, 3), (2500, 8195, 64, 0),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top,pad", FORWARD)
def test_log_probs_match_the_definition(rows, vocab, top, pad, dtype):
    print("log_probs", rows, vocab, top, pad, dtype, flush=True)
    z, g = _z(rows, vocab, dtype, 100 + vocab + rows, pad)
    tokens = torch.randint(-1, vocab, (rows,), generator=g).cuda()
    _check_forward(ops.log_probs_forward(z, tokens, top=top), z, tokens, top)
    again = ops.log_probs_forward(z, tokens.int(), top=top)  # int32 tokens, the same bits
    first = ops.log_probs_forward(z, tokens, top=top)
    for a, b in zip(first, again):
        assert (a is None and b is None) or torch.equal(a, b)


def _special_rows(vocab, dtype):
    lowest = float(torch.finfo(TYPES[dtype]).min)
    rows = []

    def row(fill):
        rows.append(torch.full((vocab,), fill))
        return rows[-1]

    row(NEG)                                    # nothing left
    row(NEG)[vocab - 1] = 1.5                   # one token left, the last
    row(NEG)[vocab // 2:vocab // 2 + 3] = 0.25  # three equal ones
    row(lowest)                                 # masked by the lowest value, all of it
    row(lowest)[vocab // 3] = 2.0               # and all but one
    row(0.0)                                    # all equal
    row(-0.0)[::2] = 0.0                        # both zeros are equal
    rows.append(torch.linspace(-4, 4, vocab))   # rising
    rows.append(torch.linspace(4, -4, vocab))   # falling
    row(NEG)[:vocab // 2] = torch.linspace(-9, 9, vocab // 2)
    big = float(torch.finfo(TYPES[dtype]).max)
    row(big)[vocab // 4:] = -big
    row(-1e4)[1] = -1.0001e4
    return torch.stack(rows).to(TYPES[dtype]).cuda()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", (6, 100, 1000, 3001, 20000, 70001))
def test_log_probs_of_masked_equal_and_ordered_rows(vocab, dtype):
    print("special rows", vocab, dtype, flush=True)
    z = _special_rows(vocab, dtype)
    tokens = torch.full((z.shape[0],), vocab - 1, device="cuda")
    for top in (0, min(vocab, 5), min(vocab, 64)):
        _check_forward(ops.log_probs_forward(z, tokens, top=top), z, tokens, top)
        for i in (0, 3, 5):  # and alone, where a row is split over the GPU
            _check_forward(ops.log_probs_forward(z[i:i + 1], tokens[:1], top=top), z[i:i + 1], tokens[:1], top)
    r = ops.log_probs_forward(z, tokens, top=3)
    grad = ops.log_probs_backward(z, tokens, r, log_prob_grad=torch.ones(z.shape[0], device="cuda"),
                                  entropy_grad=torch.ones(z.shape[0], device="cuda"))
    assert bool(torch.isfinite(grad).all())
    assert not grad[0].any()  # nothing to learn where nothing is left


@gpu
@pytest.mark.parametrize("vocab", (50, 5000, 40000))
def test_nan_and_infinite_logits_stay_in_their_row(vocab):
    z = torch.randn((6, vocab), generator=torch.Generator().manual_seed(1)).cuda()
    z[1, 7] = float("nan")
    z[3, vocab - 2] = float("inf")
    z[4] = float("nan")
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    tokens[5] = vocab  # beyond the vocabulary
    r = ops.log_probs_forward(z, tokens, top=4)
    bad = torch.tensor([False, True, False, True, True, False])
    for value in (r.log_sum, r.entropy, r.top_log_probs[:, 0]):
        assert torch.equal(torch.isnan(value).cpu() | torch.isinf(value).cpu(), bad)
    assert torch.equal(torch.isnan(r.log_prob).cpu(), torch.tensor([False, True, False, True, True, True]))
    clean = torch.tensor([0, 2, 5])
    assert torch.equal(r.top_ids[clean].cpu().long(), _top(z[clean.cuda()], 4))
    assert 7 not in r.top_ids[1].tolist() and r.top_ids[3, 0] == vocab - 2 and r.top_ids[4].tolist() == [-1] * 4
    ones = torch.ones(6, device="cuda")
    grad = ops.log_probs_backward(z, tokens, r, log_prob_grad=ones)
    assert torch.equal(torch.isnan(grad).any(dim=1).cpu(), torch.tensor([False, True, False, True, True, True]))
    masked = ops.log_probs_backward(z, torch.full_like(tokens, -1), r, log_prob_grad=ones)
    assert not masked.any()  # rows without a token: zeros whatever they hold


def _check_log_probs_gradient(got, z, tokens, g, h, old=None):
    d, s, p, log_p, entropy, _ = _exact(z)
    t = tokens.cpu().long()
    g = torch.where((t >= 0) & (s > 0), g.cpu().double(), torch.zeros_like(s))[:, None]
    h = torch.where(s > 0, h.cpu().double(), torch.zeros_like(s))[:, None]
    inner = torch.where(p > 0, log_p, torch.zeros_like(p)) + entropy[:, None]
    want = -g * p - h * p * inner
    want[torch.arange(len(t)), t.clamp(min=0)] += g[:, 0]
    err = _sum_error(z.shape[1])
    ln_s = torch.where(s > 0, s.log(), torch.zeros_like(s))[:, None]
    size = p * (g.abs() + h.abs() * (torch.where(p > 0, d.abs(), torch.zeros_like(d)) + entropy[:, None] + 2 * ln_s.abs()))
    rel = err + (2 * torch.where(p > 0, d.abs(), torch.zeros_like(d)) + 12) * U
    bound = rel * size + 2 * err * p * h.abs() * (1 + 2 * (entropy[:, None] + ln_s.abs())) + 4 * U * g.abs() * (want.abs() > 0)
    if old is not None:
        want = want + old.cpu().double()
        bound = bound + U * want.abs()
    name = str(got.dtype).split(".")[1]
    unit, least = ROUNDING[name]
    _near(got, want, bound + unit * (want.abs() + bound) + least, "gradient")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 2, 1), (5, 17, 0), (64, 1000, 0), (33, 1001, 7), (9, 4097, 3),
                                            (2, 50021, 0), (1, 131072, 0), (600, 2051, 0)])
def test_log_probs_gradient_matches_the_formula(rows, vocab, pad, dtype):
    print("log_probs gradient", rows, vocab, pad, dtype, flush=True)
    z, gen = _z(rows, vocab, dtype, vocab, pad)
    tokens = torch.randint(-1, vocab, (rows,), generator=gen).cuda()
    g, h = torch.randn(rows, generator=gen).cuda(), torch.randn(rows, generator=gen).cuda()
    r = ops.log_probs_forward(z, tokens)
    zero = torch.zeros_like(g)
    _check_log_probs_gradient(ops.log_probs_backward(z, tokens, r, log_prob_grad=g, entropy_grad=h), z, tokens, g, h)
    _check_log_probs_gradient(ops.log_probs_backward(z, tokens, r, log_prob_grad=g), z, tokens, g, zero)
    _check_log_probs_gradient(ops.log_probs_backward(z, None, r, entropy_grad=h), z, tokens, zero, h)
    # a broadcast gradient, into rows of a wider buffer, added to what is there
    wide = torch.randn((rows, vocab + 5), generator=gen).to(z.dtype).cuda()
    out, kept = wide[:, :vocab], wide.clone()
    one = torch.full((), 0.5, device="cuda").expand(rows)
    ops.log_probs_backward(z, tokens, r, log_prob_grad=one, out=out, add=True)
    _check_log_probs_gradient(out, z, tokens, one, zero, kept[:, :vocab])
    assert torch.equal(wide[:, vocab:], kept[:, vocab:])


@gpu
def test_log_probs_gradient_matches_differences():
    """Central differences in a random direction: the third derivatives of these rows are below 1 and their values
    below 40, so a step of 1/64 leaves 2^-12 / 6 of truncation and 40 * 2^-21 * 64 of rounding a row."""
    z, gen = _z(8, 300, "float32", 5, scale=1.0)
    tokens = torch.randint(0, 300, (8,), generator=gen).cuda()
    v = torch.randn((8, 300), generator=gen).cuda()
    v /= v.norm(dim=1, keepdim=True)
    step = 1 / 64

    def value(x):
        r = ops.log_probs_forward(x, tokens)
        return (r.log_prob + 0.5 * r.entropy).double()

    r = ops.log_probs_forward(z, tokens)
    ones = torch.ones(8, device="cuda")
    grad = ops.log_probs_backward(z, tokens, r, log_prob_grad=ones, entropy_grad=0.5 * ones)
    slope = (value(z + step * v) - value(z - step * v)) / (2 * step)
    assert float((slope - (grad * v).double().sum(dim=1)).abs().max()) <= 2.0 ** -12 / 6 + 40 * 2.0 ** -21 * 64


@gpu
@pytest.mark.parametrize("vocab", (9, 5000))
def test_a_row_without_gradient_gets_zeros_whatever_its_token(vocab):
    """A padding row whose token lies beyond the vocabulary: its log probability is NaN, its gradient only where the
    row's gradient is not 0."""
    z, gen = _z(7, vocab, "float32", 31)
    z[4:6] = NEG
    tokens = torch.tensor([vocab, vocab + 2 ** 32, vocab, 1, vocab, vocab, -1], device="cuda")
    g = torch.tensor([0.0, -0.0, 1.0, 2.0, 0.0, 1.0, 3.0], device="cuda")
    r = ops.log_probs_forward(z, tokens)
    assert torch.isnan(r.log_prob).tolist() == [True, True, True, False, True, True, False]
    grad = ops.log_probs_backward(z, tokens, r, log_prob_grad=g)
    assert torch.isnan(grad).all(dim=1).tolist() == [False, False, True, False, False, True, False]
    assert not grad[[0, 1, 4, 6]].any() and bool(grad[3].any())
    # with a gradient of the entropy, the row has that one alone
    h = torch.tensor([0.5, 0.0, 0.0, 0.0, 0.5, 0.0, 0.0], device="cuda")
    both = ops.log_probs_backward(z, tokens, r, log_prob_grad=g, entropy_grad=h)
    alone = ops.log_probs_backward(z, None, r, entropy_grad=h)
    assert torch.equal(both[:2], alone[:2]) and bool(both[0].any()) and not both[[1, 4, 6]].any()
    # added to what is there: nothing
    out = torch.ones_like(z)
    ops.log_probs_backward(z, tokens, r, log_prob_grad=g, out=out, add=True)
    assert bool((out[[0, 1, 4, 6]] == 1.0).all())


# ---- distillation -----------------------------------------------------------------------------
def _record(rows, vocab, held, gen, ragged=True, duplicates=False):
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:held] if vocab >= held else
                       torch.randint(0, vocab, (held,), generator=gen) for _ in range(rows)])
    teacher = torch.randn((rows, held), generator=gen) * 3.0
    if duplicates and held > 2:
        ids[:, 2] = ids[:, 0]
    if ragged:
        counts = torch.randint(0, held + 1, (rows,), generator=gen)
        ids = torch.where(torch.arange(held) < counts[:, None], ids, torch.full_like(ids, -1))
    return ids.cuda(), teacher.cuda()


def _check_distill(r, grad, z, ids, teacher, weights, t, seed=1.0, old=None):
    d, s, q, log_q, _, _ = _exact(z.double().cpu() / t)
    vocab = z.shape[1]
    ids, u = ids.cpu().long(), teacher.cpu().double() / t
    held = ids >= 0
    u = torch.where(held, u, torch.full_like(u, NEG))
    most = u.amax(dim=1, keepdim=True)
    du = torch.where(held & (most > NEG), u - torch.where(most > NEG, most, torch.zeros_like(most)), torch.full_like(u, NEG))
    e = du.exp()
    total = e.sum(dim=1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    log_p = torch.where(p > 0, du - total.log(), torch.zeros_like(u))
    at = ids.clamp(min=0)
    terms = torch.where(p > 0, p * (log_p - log_q.gather(1, at)), torch.zeros_like(p))
    w = torch.ones(len(ids), dtype=torch.float64) if weights is None else weights.cpu().double()
    w = torch.where(total[:, 0] > 0, w, torch.zeros_like(w))
    row = torch.where(w != 0, t * t * terms.sum(dim=1), torch.zeros_like(w))
    whole = w.sum()
    # p and q by the same reckoning as s, the record's sums having held / 64 + 8 links; one rounding of z / t more
    err = _sum_error(vocab) + (2 * torch.where(s > 0, s.log(), torch.zeros_like(s)).abs() + 8) * U
    target_err = (104 + ids.shape[1] / 64) * U
    sizes = torch.where(p > 0, p * (log_p.abs() + torch.nan_to_num(log_q.gather(1, at), neginf=0.0).abs()), torch.zeros_like(p))
    row_bound = t * t * (err + (target_err + 12 * U) * (sizes.sum(dim=1) + 1))
    _near(r.row_loss, row, row_bound, "row_loss")
    loss = (torch.where(w != 0, w * row, torch.zeros_like(w))).sum() / whole if whole != 0 else torch.zeros((), dtype=torch.float64)
    worst = (w.abs() * row_bound).sum() / whole.abs() if whole != 0 else 0.0
    _near(r.loss, loss, worst + 2 * U * torch.nan_to_num(loss, posinf=0.0).abs(), "loss")
    if grad is None:
        return
    coef = (seed * t * w / whole if whole != 0 else torch.zeros_like(w))[:, None]
    want = torch.where(w[:, None] != 0, coef * q, torch.zeros_like(q))
    target = torch.zeros_like(q).scatter_add_(1, at, p)
    want = torch.where(w[:, None] != 0, want - coef * target, want)
    size = coef.abs() * (q + target)
    bound = size * (err[:, None] + target_err + (2 * torch.where(q > 0, d.abs(), torch.zeros_like(d)) + 12) * U)
    if old is not None:
        want = want + old.cpu().double()
        bound = bound + U * want.abs()
    unit, least = ROUNDING[str(grad.dtype).split(".")[1]]
    _near(grad, want, bound + unit * (want.abs() + bound) + least, "distillation gradient")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,held,pad,t", [
    (1, 1, 1, 0, 1.0), (3, 2, 2, 1, 2.0), (5, 17, 17, 0, 1.5), (64, 1000, 5, 0, 2.0), (33, 1001, 64, 7, 4.0),
    (9, 4097, 65, 3, 1.0), (2, 50021, 256, 0, 2.0), (1, 131072, 64, 0, 1.0), (600, 2051, 20, 0, 0.5),
    (2100, 700, 3, 0, 2.0)])
def test_distillation_matches_the_definition(rows, vocab, held, pad, t, dtype):
    print("distill", rows, vocab, held, pad, t, dtype, flush=True)
    z, gen = _z(rows, vocab, dtype, vocab + held, pad)
    seed = torch.full((), 0.75, device="cuda")
    for ragged, duplicates, weighted in ((False, False, False), (True, True, True)):
        ids, teacher = _record(rows, vocab, held, gen, ragged, duplicates)
        weights = (torch.rand(rows, generator=gen) * (torch.rand(rows, generator=gen) < 0.7)).cuda() if weighted else None
        r = ops.distill_loss_forward(z, ids, teacher, temperature=t, row_weights=weights)
        grad = ops.distill_loss_backward(z, ids, r, seed, temperature=t)
        _check_distill(r, grad, z, ids, teacher, weights, t, 0.75)
    wide = torch.randn((rows, vocab + 3), generator=gen).to(z.dtype).cuda()
    kept = wide.clone()
    ops.distill_loss_backward(z, ids.int(), r, seed, temperature=t, out=wide[:, :vocab], add=True)
    _check_distill(r, wide[:, :vocab], z, ids, teacher, weights, t, 0.75, kept[:, :vocab])
    assert torch.equal(wide[:, vocab:], kept[:, vocab:])


@gpu
@pytest.mark.parametrize("vocab", (40, 3000, 50000))
def test_distillation_rows_that_do_not_count(vocab):
    z = torch.randn((8, vocab), generator=torch.Generator().manual_seed(3)).cuda()
    ids, teacher = _record(8, vocab, 6, torch.Generator().manual_seed(4), ragged=False)
    weights = torch.ones(8, device="cuda")
    z[0] = float("nan")
    weights[0] = 0.0               # weight 0: the row's NaN is not read into anything
    ids[1] = -1                    # no target
    teacher[2] = NEG               # targets without probability
    teacher[3, 2:] = NEG           # some of them
    ids[4, 0], weights[4] = vocab, 0.0
    z[5, vocab // 2] = NEG         # a ruled-out token that the teacher does not hold
    ids[5] = torch.arange(6)
    z[6] = float(torch.finfo(torch.float32).min)  # a whole row of the lowest value is uniform
    z[7, 3:] = NEG
    ids[7] = torch.tensor([0, 1, 2, -1, -1, -1])
    r = ops.distill_loss_forward(z, ids, teacher, row_weights=weights)
    grad = ops.distill_loss_backward(z, ids, r, torch.ones((), device="cuda"))
    zc, tc, ic = z.clone(), teacher.clone(), ids.clone()
    zc[0], ic[4, 0] = 0.0, 0
    _check_distill(r, grad, zc, ic, tc, weights, 1.0)
    assert not grad[[0, 1, 2, 4]].any() and r.weights.tolist() == [0, 0, 0, 1, 0, 1, 1, 1]
    none = ops.distill_loss_forward(z, torch.full_like(ids, -1), teacher)
    assert none.loss == 0 and not none.row_loss.any()
    assert not ops.distill_loss_backward(z, torch.full_like(ids, -1), none, torch.ones((), device="cuda")).any()
    # a target that the student rules out costs infinitely, and is still learnt
    z[5, 0] = NEG
    r = ops.distill_loss_forward(z[5:6], ids[5:6], teacher[5:6])
    assert r.row_loss[0] == float("inf") and r.loss == float("inf")
    grad = ops.distill_loss_backward(z[5:6], ids[5:6], r, torch.ones((), device="cuda"))
    assert bool(torch.isfinite(grad).all()) and grad[0, 0] < 0
    # an id beyond the vocabulary: its row, and so the mean, are NaN
    ids[5, 0] = vocab
    r = ops.distill_loss_forward(z[5:7], ids[5:7], teacher[5:7])
    assert torch.isnan(r.row_loss).tolist() == [True, False] and torch.isnan(r.loss)
    grad = ops.distill_loss_backward(z[5:7], ids[5:7], r, torch.ones((), device="cuda"))
    assert bool(torch.isnan(grad[0]).all())


@gpu
def test_distillation_gradient_matches_differences():
    """As for the log probabilities: losses below 40, third derivatives below T^2 / T^3 = 1 / T."""
    z, gen = _z(6, 200, "float32", 9, scale=1.0)
    ids, teacher = _record(6, 200, 12, gen, ragged=False, duplicates=True)
    v = torch.randn((6, 200), generator=gen).cuda()
    v /= v.norm()
    step = 1 / 64
    loss = lambda x: ops.distill_loss_forward(x, ids, teacher, temperature=2.0).loss.double()  # noqa: E731
    r = ops.distill_loss_forward(z, ids, teacher, temperature=2.0)
    grad = ops.distill_loss_backward(z, ids, r, torch.ones((), device="cuda"), temperature=2.0)
    slope = (loss(z + step * v) - loss(z - step * v)) / (2 * step)
    assert abs(float(slope - (grad * v).double().sum())) <= 2.0 ** -12 / 6 + 40 * 2.0 ** -21 * 64


@gpu
def test_a_teachers_answers_are_a_record():
    """log_probs_forward's alternatives distil as they are: a student equal to the teacher has the loss of what the
    record leaves out, -T^2 ln(sum of the kept probabilities) at T = 1."""
    z, _ = _z(40, 3000, "float32", 11)
    r = ops.log_probs_forward(z, top=32)
    loss = ops.distill_loss_forward(z, r.top_ids, r.top_log_probs).row_loss
    want = -r.top_log_probs.double().exp().sum(dim=1).log()
    # both sides take a few dozen roundings of values below 16
    assert float((loss.double() - want).abs().max()) <= 2 * _sum_error(3000) + 64 * 16 * U


# ---- the Graph's losses -----------------------------------------------------------------------
@gpu
def test_cross_entropy_loss_of_a_graph():
    z, gen = _z(37, 1000, "float32", 21)
    labels = torch.randint(-1, 1000, (37,), generator=gen).cuda()
    x = mf.Variable(z.clone(), requires_grad=True)
    loss = mf.CrossEntropyLoss(x, mf.Variable(labels, requires_grad=False))
    graph = mf.Graph(loss)
    graph.forward()
    graph.backward(loss_scale=3.0)
    _, s, _, log_p, _, _ = _exact(z)
    t = labels.cpu()
    lp = log_p[torch.arange(37), t.clamp(min=0)][t >= 0]
    assert abs(float(loss.value) + float(lp.mean())) <= _sum_error(1000) + 12 * U * float(lp.abs().max() + s.log().max())
    g = torch.full((37,), -3.0 / int((t >= 0).sum()), dtype=torch.float64)
    _check_log_probs_gradient(x.grad, z, labels, g, torch.zeros(37))
    nothing = mf.CrossEntropyLoss(x, mf.Variable(torch.full_like(labels, -1), requires_grad=False))
    graph = mf.Graph(nothing)
    graph.forward()
    graph.backward()
    assert nothing.value == 0 and not x.grad.any()


@gpu
def test_losses_on_one_node_add_their_gradients():
    z, gen = _z(20, 500, "float32", 22)
    labels = torch.randint(0, 500, (20,), generator=gen).cuda()
    ids, teacher = _record(20, 500, 8, gen)
    weights = torch.rand(20, generator=gen).cuda()
    constant = lambda v: mf.Variable(v, requires_grad=False)  # noqa: E731
    x = mf.Variable(z.clone(), requires_grad=True)
    ce = mf.CrossEntropyLoss(x, constant(labels))
    kd = mf.DistillationLoss(x, constant(ids), constant(teacher), constant(weights), temperature=2.0)
    graph = mf.Graph(mf.Add(ce, kd))
    graph.forward()
    graph.backward()
    r = ops.distill_loss_forward(z, ids, teacher, temperature=2.0, row_weights=weights)
    first = ops.distill_loss_backward(z, ids, r, torch.ones((), device="cuda"), temperature=2.0)
    g = torch.full((20,), -1.0 / 20, dtype=torch.float64)
    _check_log_probs_gradient(x.grad, z, labels, g, torch.zeros(20), old=first)
    assert float(kd.value) == float(r.loss)


@gpu
def test_results_do_not_depend_on_the_stream_or_the_run():
    z, gen = _z(3, 70000, "bfloat16", 23)
    tokens = torch.randint(0, 70000, (3,), generator=gen).cuda()
    first = ops.log_probs_forward(z, tokens, top=64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = ops.log_probs_forward(z, tokens, top=64)
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@gpu
def test_rows_beyond_32_bit_offsets():
    """A row that starts past 2^31 elements: a view with a large row stride into one allocation."""
    stride = 2 ** 30 + 8
    held = torch.zeros(2 * stride + 300, dtype=torch.bfloat16, device="cuda")
    z = held.as_strided((3, 300), (stride, 1))
    fresh, gen = _z(3, 300, "bfloat16", 24)
    z.copy_(fresh)
    tokens = torch.randint(0, 300, (3,), generator=gen).cuda()
    r = ops.log_probs_forward(z, tokens, top=5)
    _check_forward(r, fresh, tokens, 5)
    g = torch.ones(3, device="cuda")
    want = ops.log_probs_backward(fresh, tokens, r, log_prob_grad=g)
    ops.log_probs_backward(z, tokens, r, log_prob_grad=g, out=z)  # in place: each logit is read before it is written
    assert torch.equal(z, want)


@gpu
def test_gradients_in_the_logits_place_and_strided_inputs():
    z, gen = _z(5, 3000, "float32", 25)
    ids, teacher = _record(5, 3000, 40, gen, duplicates=True)
    d = ops.distill_loss_forward(z, ids, teacher)
    one = torch.ones((), device="cuda")
    want = ops.distill_loss_backward(z, ids, d, one)
    taken = z.clone()
    ops.distill_loss_backward(taken, ids, d, one, out=taken)  # logits at the ids are read before any write
    assert torch.equal(taken, want)
    # logits whose rows are not contiguous, and whole numbers and gradients that are columns of wider tensors
    turned = z.t().contiguous().t()
    tokens = torch.randint(0, 3000, (5, 3), generator=gen).cuda()[:, 1]
    g = torch.randn((5, 2), generator=gen).cuda()[:, 0]
    first, second = ops.log_probs_forward(z, tokens.contiguous(), top=9), ops.log_probs_forward(turned, tokens, top=9)
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    a = ops.log_probs_backward(z, tokens.contiguous(), first, log_prob_grad=g.contiguous())
    assert torch.equal(ops.log_probs_backward(turned, tokens, first, log_prob_grad=g), a)


@gpu
def test_no_rows():
    z = torch.empty((0, 10), device="cuda")
    tokens = torch.empty((0,), dtype=torch.int64, device="cuda")
    r = ops.log_probs_forward(z, tokens, top=3)
    assert r.log_prob.shape == (0,) and r.top_ids.shape == (0, 3)
    assert ops.log_probs_backward(z, tokens, r, log_prob_grad=r.log_prob).shape == (0, 10)
    d = ops.distill_loss_forward(z, torch.empty((0, 2), dtype=torch.int32, device="cuda"), torch.empty((0, 2), device="cuda"))
    assert d.loss == 0


@gpu
def test_refusals():
    z = torch.randn((4, 10), device="cuda")
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        ops.log_probs_forward(z.double(), tokens)
    with pytest.raises(ValueError):
        ops.log_probs_forward(z[0], tokens)
    with pytest.raises(ValueError):
        ops.log_probs_forward(z, tokens[:3])
    with pytest.raises(TypeError):
        ops.log_probs_forward(z, tokens.float())
    for top in (-1, 11, 65):
        with pytest.raises(ValueError):
            ops.log_probs_forward(z, tokens, top=top)
    with pytest.raises(ValueError):
        ops.log_probs_forward(torch.empty((3, 0), device="cuda"))
    r = ops.log_probs_forward(z, tokens)
    g = torch.ones(4, device="cuda")
    with pytest.raises(ValueError):
        ops.log_probs_backward(z, None, r, log_prob_grad=g)
    with pytest.raises(ValueError):
        ops.log_probs_backward(z[:2], tokens[:2], r, log_prob_grad=g[:2])
    with pytest.raises(ValueError):
        ops.log_probs_backward(z, tokens, r, log_prob_grad=g, add=True)
    with pytest.raises(ValueError):
        ops.log_probs_backward(z, tokens, r, log_prob_grad=g, out=torch.empty((10, 4), device="cuda").t())
    with pytest.raises(TypeError):
        ops.log_probs_backward(z, tokens, r, log_prob_grad=g.double())
    ids, teacher = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    for t in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            ops.distill_loss_forward(z, ids, teacher, temperature=t)
    with pytest.raises(ValueError):
        ops.distill_loss_forward(z, ids[:, :0], teacher[:, :0])
    with pytest.raises(ValueError):
        ops.distill_loss_forward(z, ids, teacher[:, :1])
    with pytest.raises(ValueError):
        ops.distill_loss_forward(z, ids.repeat(1, 200), teacher.repeat(1, 200))
    with pytest.raises(ValueError):
        ops.distill_loss_forward(z, ids, teacher, row_weights=torch.ones(3, device="cuda"))
    d = ops.distill_loss_forward(z, ids, teacher)
    with pytest.raises(ValueError):
        ops.distill_loss_backward(z, ids, d, torch.ones(2, device="cuda"))
    lib = mf.native._library()
    assert lib.mfh_log_probs_workspace(1, 0, 0, 0) == -1 and lib.mfh_log_probs_workspace(1, 10, 3, 0) == -1
    assert lib.mfh_log_probs_workspace(1, 10, 0, 11) == -1 and lib.mfh_distill_workspace(2 ** 23, 10, 0) == -1
    assert b"out of range" in lib.mfh_last_error()


@gpu
def test_temperatures_whose_square_is_no_normal_float_are_refused():
    """T^2 scales the loss and 1 / T the logits: beyond these the results were NaN."""
    z, ids, teacher = torch.randn((2, 9), device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda"), torch.ones((2, 1), device="cuda")
    for t in (1e-39, 1e-30, 2.0 ** -64, 2.0 ** 64, 1e30, 1e300):
        with pytest.raises(ValueError, match="temperature"):
            ops.distill_loss_forward(z, ids, teacher, temperature=t)
        with pytest.raises(ValueError, match="temperature"):
            mf.DistillationLoss(mf.Variable(z), mf.Variable(ids), mf.Variable(teacher), temperature=t)
    for t in (2.0 ** -63, 2.0 ** 63):
        r = ops.distill_loss_forward(z, ids, teacher, temperature=t)
        assert not torch.isnan(r.row_loss).any()
        assert bool(torch.isfinite(ops.distill_loss_backward(z, ids, r, torch.ones((), device="cuda"), temperature=t)).all())


def test_host_tensors_are_refused():
    z = torch.zeros((2, 3))
    with pytest.raises(TypeError):
        ops.log_probs_forward(z)
    with pytest.raises(TypeError):
        ops.distill_loss_forward(z, torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)))
    for loss in (mf.CrossEntropyLoss(mf.Variable(z), mf.Variable(torch.zeros(2, dtype=torch.int64))),
                 mf.DistillationLoss(mf.Variable(z), mf.Variable(torch.zeros((2, 1), dtype=torch.int32)),
                                     mf.Variable(torch.zeros((2, 1))))):
        with pytest.raises(ValueError):
            mf.Graph(loss).forward()
