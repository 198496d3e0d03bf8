"""Logits adjusted by a history's penalties, biases and a grammar's mask, against the definition in 64 bits.

Bounds (u = 2^-24): the quotient or product q, frequency * n, the two differences and the sum with the bias take
one float32 rounding each, the bias's own sum of k values at most k - 1, so the result is within u (|q| + |f n| +
|q - f n| + |q - f n - p| + k sum |b| + |result|), times 1.01 for the products of roundings, plus half a step of
the logits' type. A logit that nothing names keeps its bits, and a ruled-out one is -inf exactly.
"""

import pytest
import torch

import myflows_amd as mf
from myflows_amd import logits as ops

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
NEG = float("-inf")
gpu = pytest.mark.gpu


def _column(value, rows):
    value = torch.as_tensor(value, dtype=torch.float32).cpu().double()
    return (value.expand(rows) if value.ndim == 0 else value)[:, None]


def _check(got, z, tokens=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None,
           bias_values=None, allowed=None):
    rows, vocab = z.shape
    x = z.detach().cpu().double()
    n, seen = torch.zeros_like(x), torch.zeros_like(x)
    if tokens is not None:
        t = tokens.cpu().long()
        given = (t >= 0) & (t < vocab)
        at = torch.where(given, t, 0)
        prompt = torch.zeros(rows) if prompt_lengths is None else prompt_lengths.cpu()
        answer = given & (torch.arange(t.shape[1]) >= prompt[:, None])
        seen.scatter_add_(1, at, given.double())
        n.scatter_add_(1, at, answer.double())
    b, b_size, b_count = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    if bias_ids is not None:
        ids, values = bias_ids.cpu().long().expand(rows, -1), bias_values.cpu().double().expand(rows, -1)
        given = (ids >= 0) & (ids < vocab)
        at, values = torch.where(given, ids, 0), torch.where(given, values, 0.0)
        b.scatter_add_(1, at, values)
        b_size.scatter_add_(1, at, values.abs())
        b_count.scatter_add_(1, at, given.double())
    r, p, f = (_column(v, rows) for v in (repetition, presence, frequency))
    q = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    first = q - f * n
    second = torch.where(n > 0, first - p, first)
    want = second + b
    bound = 1.01 * U * (q.abs() + (f * n).abs() + first.abs() + second.abs() + b_count * b_size + want.abs())
    info = torch.finfo(z.dtype)
    bound = bound + info.eps / 2 * want.abs().clamp(min=info.smallest_normal)
    named = (seen > 0) | (b_count > 0)
    want = torch.where(named, want, x)
    bound = torch.where(named, bound, 0.0)
    if allowed is not None:
        words = allowed.cpu().long().expand(rows, -1) & 0xFFFFFFFF
        place = torch.arange(vocab)
        ruled = (words[:, place // 32] >> (place % 32)) & 1 == 0
        want, bound = torch.where(ruled, NEG, want), torch.where(ruled, 0.0, bound)
    have = got.detach().cpu().double()
    same = (have == want) | (have.isnan() & want.isnan())
    off = torch.where(same, 0.0, (have - want).abs())
    assert bool((off <= bound).all()), f"off by up to {float((off - bound).nan_to_num(nan=1e30).max()):.3e} beyond its bound"


def _bits(g, rows, vocab, share):
    packed = (torch.rand((rows, (vocab + 31) // 32, 32), generator=g) < share).long() << torch.arange(32)
    packed = packed.sum(dim=2)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int().cuda()


SIZES = [
    # rows, vocab, held, biases, pad: one logit, no history, odd sizes, chunk ends, both chunk lengths, many biases
    (1, 1, 1, 1, 0), (2, 3, 0, 2, 0), (3, 33, 40, 5, 1), (5, 100, 300, 100, 3), (4, 2048, 7, 0, 0), (1, 2049, 64, 3, 5),
    (7, 1000, 1, 1024, 0), (1, 131072, 2048, 8, 0), (70, 32771, 257, 40, 61), (600, 16385, 100, 12, 0),
    (530, 8193, 9000, 0, 7), (2100, 300, 20, 2, 0),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,held,biases,pad", SIZES)
def test_adjusted_logits_match_the_definition(rows, vocab, held, biases, pad, dtype):
    print("adjust", rows, vocab, held, biases, pad, dtype, flush=True)
    g = torch.Generator().manual_seed(rows + vocab + held)
    z = (torch.randn((rows, vocab + pad), generator=g) * 3).to(TYPES[dtype]).cuda()[:, :vocab]
    tokens = ((vocab + 1.0) ** torch.rand((rows, held), generator=g, dtype=torch.float64)).long() - 1  # often the same
    tokens[torch.rand((rows, held), generator=g) < 0.2] = -1
    options = dict(tokens=tokens.cuda(), prompt_lengths=torch.randint(0, held + 2, (rows,), generator=g).cuda(),
                   repetition=(0.7 + torch.rand(rows, generator=g)).cuda(), presence=torch.randn(rows, generator=g).cuda(),
                   frequency=torch.randn(rows, generator=g).cuda())
    if biases:
        options.update(bias_ids=torch.randint(-1, vocab, (rows, biases), generator=g).cuda(),
                       bias_values=torch.randn((rows, biases), generator=g).cuda())
    before = z.clone()
    got = ops.adjust_logits(z, **options)
    assert got.dtype is z.dtype and torch.equal(z, before)
    _check(got, z, **options)
    narrow = {k: v.int() if v.dtype is torch.int64 else v for k, v in options.items()}
    assert torch.equal(ops.adjust_logits(z, **narrow), got)
    for share in (0.9, 0.03):
        allowed = _bits(g, rows, vocab, share)
        masked = ops.adjust_logits(z, **options, allowed=allowed)
        _check(masked, z, **options, allowed=allowed)
        held_in = torch.empty((rows, vocab + pad), dtype=z.dtype, device="cuda").fill_(7)
        held_in[:, :vocab] = z
        assert ops.adjust_logits(held_in[:, :vocab], **options, allowed=allowed, out=held_in[:, :vocab]).data_ptr() == held_in.data_ptr()
        assert torch.equal(held_in[:, :vocab], masked) and bool((held_in[:, vocab:] == 7).all())
    in_place = z.clone()
    ops.adjust_logits(in_place, **options, out=in_place)
    assert torch.equal(in_place, got)
    only = ops.adjust_logits(z, allowed=allowed)
    _check(only, z, allowed=allowed)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_numbers_for_all_rows_shared_biases_and_strides(dtype):
    g = torch.Generator().manual_seed(9)
    z = torch.randn((6, 500), generator=g).to(TYPES[dtype]).cuda()
    history = torch.randint(-1, 600, (6, 90), generator=g).cuda()  # some beyond the vocabulary
    tokens = history[:, 10:80]
    lengths = torch.randint(0, 70, (6, 3), generator=g).cuda()[:, 1]
    ids, values = torch.tensor([3, 3, 499, -1, 500, 3], device="cuda"), torch.tensor([0.5, 1.0, 2.0, 9.0, 9.0, -4.0], device="cuda")
    allowed = _bits(g, 1, 500, 0.7)[0]
    options = dict(tokens=tokens, prompt_lengths=lengths, repetition=1.3, presence=0.25, frequency=torch.full(
        (1,), 0.5, device="cuda").expand(6), bias_ids=ids, bias_values=values, allowed=allowed)
    got = ops.adjust_logits(z, **options)
    _check(got, z, **options)
    rowed = {**options, "bias_ids": ids.expand(6, -1), "bias_values": values.expand(6, -1).contiguous(),
             "allowed": allowed.expand(6, -1).contiguous(), "tokens": tokens.contiguous(),
             "repetition": torch.full((6,), 1.3, device="cuda"), "presence": torch.full((6,), 0.25, device="cuda")}
    assert torch.equal(ops.adjust_logits(z, **rowed), got)
    across = torch.empty((500, 6), dtype=z.dtype, device="cuda").t()
    across.copy_(z)
    assert torch.equal(ops.adjust_logits(across, **options), got)
    assert torch.equal(ops.adjust_logits(z, **{**options, "tokens": tokens.t().contiguous().t()}), got)
    assert torch.equal(ops.adjust_logits(z), z)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_nan_and_rows_without_a_token_left(dtype):
    t = TYPES[dtype]
    z = torch.tensor([NEG, float("inf"), float("nan"), float(torch.finfo(t).min), 0.0, -0.0, 1.0, -1.0]).repeat(4, 5).to(t).cuda()
    tokens = torch.arange(8, device="cuda").repeat(4, 1)
    allowed = torch.tensor([[-1, -1], [0, 0], [1 << 6, 0], [-1 << 31, 255]], dtype=torch.int32, device="cuda")
    options = dict(tokens=tokens, repetition=2.0, presence=0.5, frequency=0.25, bias_ids=torch.tensor([6, 7], device="cuda"),
                   bias_values=torch.tensor([NEG, 1.0], device="cuda"), allowed=allowed)
    got = ops.adjust_logits(z, **options)
    row = got[0].float().tolist()
    assert row[0] == NEG and row[1] == float("inf") and row[2] != row[2] and row[6] == NEG
    assert row[4:6] == [-0.75, -0.75] and row[7] == -1.75
    assert torch.equal(got[0, 8:].nan_to_num(nan=5.0), z[0, 8:].nan_to_num(nan=5.0))
    assert bool((got[1] == NEG).all()) and bool((got[2] == NEG).all())
    assert got[3, 31].item() == -1.0 and bool((got[3, :31] == NEG).all())
    answer = mf.logits.log_probs_forward(got[1:2], top=2)  # what is made of a row with nothing left
    assert float(answer.entropy) == 0.0 and answer.top_log_probs.tolist() == [[NEG, NEG]]


@gpu
def test_counts_are_of_the_answer_alone_and_a_token_of_both_is_divided_once():
    z = torch.full((1, 8), 4.0, device="cuda")
    tokens = torch.tensor([[2, 3, 2, 3, 3, 5, -1, -1]], device="cuda")
    got = ops.adjust_logits(z, tokens=tokens, prompt_lengths=torch.tensor([3], device="cuda"), repetition=2.0, presence=0.5,
                            frequency=0.125)
    assert got.tolist() == [[4.0, 4.0, 2.0, 2.0 - 0.25 - 0.5, 4.0, 2.0 - 0.125 - 0.5, 4.0, 4.0]]


@gpu
def test_very_long_history_of_one_token():
    held = ops.HELD_LIMIT
    z = torch.zeros((1, 40), device="cuda")
    got = ops.adjust_logits(z, tokens=torch.full((1, held), 7, dtype=torch.int32, device="cuda"), frequency=1.0)
    assert got[0, 7].item() == -float(held) and bool((got[0, :7] == 0).all()) and bool((got[0, 8:] == 0).all())


@gpu
def test_rows_beyond_32_bit_offsets():
    rows, vocab = 40000, 65537  # 2.6e9 logits
    z = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda")
    tokens = torch.full((rows, 1), vocab - 1, device="cuda")
    ops.adjust_logits(z, tokens=tokens, presence=1.0, out=z)
    assert bool((z[:, -1] == -1).all()) and bool((z[-1, :-1] == 0).all()) and bool((z[0, :-1] == 0).all())
    other = ops.adjust_logits(z, tokens=tokens, presence=1.0)
    assert bool((other[:, -1] == -2).all()) and bool((other[-1, :-1] == 0).all())


@gpu
def test_a_captured_answering_step_repeats_the_eager_bits():
    g = torch.Generator().manual_seed(4)
    z = torch.randn((3, 50000), generator=g).to(torch.bfloat16).cuda()
    tokens = torch.randint(-1, 50000, (3, 64), generator=g).cuda()
    allowed = _bits(g, 3, 50000, 0.5)

    def answer():
        adjusted = ops.adjust_logits(z, tokens=tokens, repetition=1.2, presence=0.3, allowed=allowed)
        return adjusted, mf.logits.log_probs_forward(adjusted, top=5).top_ids

    answer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = answer()
    for seed in range(3):
        z.copy_(torch.randn(z.shape, generator=torch.Generator().manual_seed(seed)))
        tokens.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(answer(), captured):
            assert torch.equal(a, b)


def test_refusals_without_a_gpu():
    z = torch.zeros((2, 5))
    with pytest.raises(TypeError, match="on the GPU"):
        ops.adjust_logits(z)


@gpu
def test_refusals():
    z = torch.zeros((4, 50), device="cuda")
    tokens = torch.zeros((4, 3), dtype=torch.int64, device="cuda")
    floats = torch.ones(4, device="cuda")
    words = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    ids, values = tokens, torch.zeros((4, 3), device="cuda")
    type_errors = [dict(tokens=tokens.float()), dict(tokens=tokens.cpu()), dict(tokens=tokens, prompt_lengths=floats),
                   dict(repetition=floats.double()), dict(presence=floats.cpu()), dict(bias_ids=ids, bias_values=values.half()),
                   dict(bias_ids=values, bias_values=values), dict(allowed=words.long()), dict(allowed=words.cpu())]
    value_errors = [dict(tokens=tokens[:3]), dict(tokens=tokens[0]), dict(tokens=[1]), dict(prompt_lengths=tokens[:, 0]),
                    dict(tokens=tokens, prompt_lengths=tokens), dict(repetition=0.0), dict(repetition=-1.0),
                    dict(repetition=float("nan")), dict(presence=float("inf")), dict(frequency=floats[:2]),
                    dict(bias_ids=ids), dict(bias_values=values), dict(bias_ids=ids, bias_values=values[:, :2]),
                    dict(bias_ids=ids[:2], bias_values=values[:2]), dict(allowed=words[:, :1]), dict(allowed=words[:2]),
                    dict(bias_ids=torch.zeros(1025, dtype=torch.int32, device="cuda"), bias_values=torch.zeros(1025, device="cuda")),
                    dict(tokens=torch.zeros((4, 1), dtype=torch.int32, device="cuda").expand(4, 1 << 20)),
                    dict(out=z[:, :40]), dict(out=z.half()), dict(out=z[:2].repeat(2, 1).t().contiguous().t())]
    for error, cases in ((TypeError, type_errors), (ValueError, value_errors)):
        for options in cases:
            with pytest.raises(error):
                ops.adjust_logits(z, **options)
    held = torch.zeros(400, device="cuda")
    with pytest.raises(ValueError, match="share no memory"):
        ops.adjust_logits(held[:200].view(4, 50), out=held[50:250].view(4, 50))
    with pytest.raises(ValueError, match="share no memory"):
        ops.adjust_logits(held[:400].view(4, 100)[:, :50], out=held[:200].view(4, 50))
    side = torch.randn((4, 110), device="cuda")
    got = ops.adjust_logits(side[:, 3:53], presence=1.0, tokens=tokens, out=side[:, 53:103])  # rows side by side
    _check(got, side[:, 3:53], tokens, presence=1.0)
    with pytest.raises(ValueError, match="share no memory"):
        ops.adjust_logits(side[:, 3:53], out=side[:, 52:102])


@gpu
def test_results_written_over_what_logits_are_adjusted_by_are_refused():
    held = torch.zeros(1000, device="cuda")
    z, out, words = torch.zeros((4, 50), device="cuda"), held[100:300].view(4, 50), held.view(torch.int32)
    tokens = words[:200].view(4, 50)
    for options in (dict(tokens=tokens), dict(tokens=tokens[:, :3], prompt_lengths=words[297:301]), dict(repetition=held[150:154]),
                    dict(presence=held[299:303]), dict(frequency=held[97:101]), dict(bias_ids=tokens[:, :2], bias_values=z[:, :2]),
                    dict(bias_ids=torch.zeros((4, 2), dtype=torch.int32, device="cuda"), bias_values=held[290:298].view(4, 2)),
                    dict(allowed=words[292:300].view(4, 2)), dict(allowed=words[299:301])):
        for logits in (z, out):
            with pytest.raises(ValueError, match="share no memory"):
                ops.adjust_logits(logits, out=out, **options)
    # Rows of logits and what they are adjusted by side by side, adjusted in place.
    rows = torch.randn((4, 54), device="cuda")
    rows[:, 50:] = torch.tensor([1.5, 0.5, 0.25, 0.0], device="cuda")
    rows[:, 53] = torch.arange(4, dtype=torch.int32, device="cuda").view(torch.float32)
    at = rows.view(torch.int32)[:, 53:]
    want = ops.adjust_logits(rows[:, :50].clone(), tokens=at.clone(), repetition=1.5, presence=0.5, frequency=0.25)
    got = ops.adjust_logits(rows[:, :50], tokens=at, repetition=rows[:, 50], presence=rows[:, 51], frequency=rows[:, 52],
                            out=rows[:, :50])
    assert torch.equal(got, want)


def test_penalties_that_float32_does_not_hold_are_refused():
    for bad in (1e39, 3.4028236e38, 1e-46, 0.0, -1e-46):
        with pytest.raises(ValueError, match="finite and positive"):
            ops._penalty(bad, 4, "repetition", positive=True)
    for bad in (1e39, -1e39, -3.4028236e38):
        with pytest.raises(ValueError, match="finite"):
            ops._penalty(bad, 4, "presence")
    assert ops._penalty(1e-40, 4, "repetition", positive=True)[2] > 0.0 and ops._penalty(-1e-46, 4, "presence")[2] == 0.0


@gpu
def test_the_smallest_and_largest_penalties():
    z = torch.tensor([[2.0 ** -30, -2.0 ** -30, 0.0, 1.0]], device="cuda")
    tokens = torch.tensor([[0, 1, 2]], device="cuda")
    tiny, huge = 2.0 ** -149, torch.finfo(torch.float32).max
    lengths = torch.tensor([3], device="cuda")
    got = ops.adjust_logits(z, tokens=tokens, prompt_lengths=lengths, repetition=tiny)
    assert got.tolist() == [[2.0 ** 119, 0.0, 0.0, 1.0]]  # 2^-179 lies below float32
    got = ops.adjust_logits(z, tokens=tokens, prompt_lengths=lengths, repetition=2.0 ** 127)
    assert got.tolist() == [[0.0, -2.0 ** 97, 0.0, 1.0]]  # and so does 2^-157
    assert ops.adjust_logits(z, tokens=tokens, presence=huge).tolist() == [[-huge, -huge, -huge, 1.0]]
    for name in ("repetition", "presence", "frequency"):
        with pytest.raises(ValueError, match="finite"):
            ops.adjust_logits(z, tokens=tokens, **{name: 1e39})
