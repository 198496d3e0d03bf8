"""Embeddings on libmfhip: the lookup, the table's gradient by sorted tokens, the graph operator and the layer.

Bounds (u = 2^-24): a looked-up element is one float32 product rounded once to its type, so it equals torch's. A
gradient is a chain of at most L + 1 additions of the L rows of its token (in pieces or not, each row passes
through at most L roundings) and one product, so it is within (L + 2) u scale sum |g| of the sum in 64 bits, plus
half a step of its type: eps / 2 of it, or of the smallest normal number below that.
"""

import pytest
import torch

import myflows_amd as mf
from myflows_amd import embedding as ops

U = 2.0 ** -24
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
gpu = pytest.mark.gpu


def _step(dtype, value):
    info = torch.finfo(dtype)
    return info.eps / 2 * torch.clamp(value.abs(), min=info.smallest_normal)


def _check_gradient(got, grad, ids, vocab, scale, before=None):
    flat = ids.reshape(-1).cpu().long()
    rows = grad.reshape(-1, grad.shape[-1]).cpu().double()
    there = (flat >= 0) & (flat < vocab)
    want = torch.zeros((vocab, rows.shape[1]), dtype=torch.float64).index_add_(0, flat[there], rows[there])
    size = torch.zeros_like(want).index_add_(0, flat[there], rows[there].abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, flat[there], torch.ones(int(there.sum()), dtype=torch.float64))
    want, bound = want * scale, (count + 2)[:, None] * U * abs(scale) * size
    if before is not None:
        want = want + before.cpu().double()
        bound = bound + U * want.abs()
        untouched = count == 0
        assert torch.equal(got.cpu()[untouched], before.cpu()[untouched])
    bound = bound + _step(got.dtype, want)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off - bound).max()):.3e} beyond its bound"


def _zipf(g, vocab, count):
    u = torch.rand(count, generator=g, dtype=torch.float64)
    return ((vocab + 1.0) ** u).long().sub_(1).clamp_(0, vocab - 1)


SIZES = [
    # count, vocab, dim: one token, one row, packs that end inside a row, several columns of packs, pieces of
    # tokens (more than 64 rows), one token only, more positions than a chunk, slices of every size
    (1, 1, 1), (0, 5, 3), (3, 2, 2), (7, 1000, 8), (64, 100, 31), (65, 3, 64), (200, 1, 33), (129, 2, 513),
    (1000, 70000, 5), (1000, 50, 771), (5000, 1000, 512), (4096, 300000, 16), (33000, 130, 24), (40000, 8, 9),
    (140000, 3000, 4), (777, 65537, 1030), (300, 262144, 3), (66000, 5, 20),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,vocab,dim", SIZES)
def test_lookup_and_gradient_match_the_definition(count, vocab, dim, dtype):
    print("embedding", count, vocab, dim, dtype, flush=True)
    g = torch.Generator().manual_seed(count + vocab + dim)
    t = TYPES[dtype]
    table = torch.randn((vocab, dim), generator=g).to(t).cuda()
    ids = _zipf(g, vocab, count)
    ids[torch.rand(count, generator=g) < 0.1] = -1
    ids = ids.cuda()
    y = ops.embedding_forward(table, ids, scale=1.7)
    want = torch.where((ids >= 0)[:, None], table[ids.clamp(min=0)].float() * torch.tensor(1.7), 0.0).to(t)
    assert y.dtype is t and torch.equal(y, want)
    assert torch.equal(ops.embedding_forward(table, ids.int(), scale=1.7), y)
    grad = torch.randn((count, dim), generator=g).to(t).cuda()
    first = ops.embedding_backward(grad, ids, vocab, scale=0.3)
    assert first.dtype is t
    _check_gradient(first, grad, ids, vocab, 0.3)
    assert torch.equal(ops.embedding_backward(grad, ids.int(), vocab, scale=0.3), first)
    wide = ops.embedding_backward(grad, ids, vocab, scale=0.3, out=torch.full((vocab, dim), float("nan"), device="cuda"))
    _check_gradient(wide, grad, ids, vocab, 0.3)
    for held in {t, torch.float32}:
        before = torch.randn((vocab, dim), generator=g).to(held).cuda()
        added = ops.embedding_backward(grad, ids, vocab, scale=0.3, out=before.clone(), add=True)
        _check_gradient(added, grad, ids, vocab, 0.3, before)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_tables_gradients_and_tokens_are_read_in_place(dtype):
    g, t = torch.Generator().manual_seed(3), TYPES[dtype]
    table = torch.randn((300, 77), generator=g).to(t).cuda()[:, 3:70]
    ids = torch.randint(-1, 300, (40, 6), generator=g).cuda()
    y = ops.embedding_forward(table, ids)
    assert y.shape == (40, 6, 67)
    assert torch.equal(y, torch.where((ids >= 0)[..., None], table[ids.clamp(min=0)], 0.0))
    column = ids[:, 2]                          # stride 6
    assert torch.equal(ops.embedding_forward(table, column), y[:, 2])
    assert torch.equal(ops.embedding_forward(table, ids.t()), y.transpose(0, 1))
    grad = torch.randn((40, 90), generator=g).to(t).cuda()[:, 5:72]
    out = torch.full((300, 80), 7.0, device="cuda").to(t)
    ops.embedding_backward(grad, column, 300, out=out[:, 1:68])
    _check_gradient(out[:, 1:68], grad, column, 300, 1.0)
    assert bool((out[:, :1] == 7).all()) and bool((out[:, 68:] == 7).all())
    one = torch.full((1,), 5, device="cuda").expand(90)  # stride 0
    dy = torch.randn((90, 8), generator=g).to(t).cuda()
    _check_gradient(ops.embedding_backward(dy, one, 9), dy, one, 9, 1.0)
    _check_gradient(ops.embedding_backward(dy[:, :1].expand(90, 8), one, 9), dy[:, :1].expand(90, 8), one, 9, 1.0)


@gpu
def test_tokens_outside_of_the_table():
    table = torch.randn((10, 40), device="cuda")
    ids = torch.tensor([3, 10, -1, -(2 ** 40), 2 ** 33 + 3, 9, 2 ** 40], device="cuda")
    y = ops.embedding_forward(table, ids)
    assert torch.equal(y[[0, 5]], table[[3, 9]]) and bool((y[[2, 3]] == 0).all()) and bool(y[[1, 4, 6]].isnan().all())
    grad = torch.randn((7, 40), device="cuda")
    got = ops.embedding_backward(grad, ids, 10)
    want = torch.zeros((10, 40), device="cuda")
    want[3], want[9] = grad[0], grad[5]
    assert torch.equal(got, want)


@gpu
def test_rows_of_nan_and_infinity_stay_in_their_rows():
    table = torch.zeros((5, 70), device="cuda")
    table[1], table[3] = float("nan"), float("inf")
    y = ops.embedding_forward(table, torch.tensor([0, 1, 2, 3, -1], device="cuda"))
    assert bool((y[[0, 2, 4]] == 0).all()) and bool(y[1].isnan().all()) and bool((y[3] == float("inf")).all())
    grad = torch.ones((200, 70), device="cuda")
    ids = torch.arange(200, device="cuda") % 3
    grad[ids == 1] = float("nan")
    got = ops.embedding_backward(grad, ids, 5)
    assert bool(got[1].isnan().all()) and bool((got[0] == 67).all()) and bool((got[2] == 66).all())
    assert bool((got[3:] == 0).all())
    ids[ids == 1] = -1  # a padded row's gradient is not read into any sum
    assert bool((ops.embedding_backward(grad, ids, 5)[1] == 0).all())


@gpu
def test_a_table_beyond_32_bit_offsets():
    vocab, dim = (1 << 21) + 3, 1100  # 2.3e9 elements
    table = torch.zeros((vocab, dim), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device="cuda")
    table[vocab - 1], table[vocab - 2] = 3.0, 2.0
    y = ops.embedding_forward(table, ids)
    assert y[:, 0].tolist() == [3.0, 0.0, 2.0, 3.0] and y[:, -1].tolist() == [3.0, 0.0, 2.0, 3.0]
    ops.embedding_backward(y, ids, vocab, out=table, add=True)
    assert bool((table[vocab - 1] == 9).all()) and bool((table[vocab - 2] == 4).all()) and bool((table[:-2] == 0).all())


@gpu
def test_gradient_equals_differences():
    g = torch.Generator().manual_seed(0)
    table = torch.randint(-8, 9, (6, 3), generator=g).float().cuda()
    ids = torch.tensor([1, 4, 1, -1, 0], device="cuda")
    weight = torch.randint(-4, 5, (5, 3), generator=g).float().cuda()
    grad = ops.embedding_backward(weight, ids, 6, scale=2.0)
    for v in range(6):
        for c in range(3):
            ahead = table.clone()
            ahead[v, c] += 1.0  # whole numbers: the difference is exact
            rise = (ops.embedding_forward(ahead, ids, scale=2.0) * weight).sum() - (
                ops.embedding_forward(table, ids, scale=2.0) * weight).sum()
            assert float(rise) == float(grad[v, c])


@gpu
def test_embedding_layer_in_a_graph_shares_its_table():
    mf.set_device("cuda")
    layer = mf.Embedding(11, 6, scale=0.5, name="tokens")
    assert [p.name for p in layer.params] == ["tokens_W"]
    a = mf.Variable(torch.tensor([1, 2, 1], device="cuda"), requires_grad=False)
    b = mf.Variable(torch.tensor([2, -1, 10], device="cuda"), requires_grad=False)
    target = mf.Variable(torch.zeros((3, 6), device="cuda"), requires_grad=False)
    loss = mf.MSELoss(mf.Add(layer(a), layer(b)), target)
    graph = mf.Graph(loss)
    graph.forward()
    graph.backward()
    w = layer.W.value.double().detach().requires_grad_(True)
    first = 0.5 * w[a.value]
    second = 0.5 * torch.where((b.value >= 0)[:, None], w[b.value.clamp(min=0)], 0.0)
    want = (first + second).square().mean()
    want.backward()
    assert abs(float(loss.value) - float(want.detach())) <= 1e-6 * float(want.detach())
    assert torch.allclose(layer.W.grad.double(), w.grad, rtol=1e-5, atol=1e-7)


@gpu
def test_recorded_and_captured_steps_repeat_the_eager_bits():
    mf.set_device("cuda")

    def network():
        layer = mf.Embedding(500, 32, initializer=mf.make_initializer("normal", seed=1, std=0.5))
        head = mf.Dense(32, 40, initializer=mf.make_initializer(seed=2))
        ids = mf.Variable(torch.arange(300, device="cuda") * 7 % 500, requires_grad=False)
        labels = mf.Variable(torch.arange(300, device="cuda") % 40, requires_grad=False)
        return layer, ids, mf.Adam(mf.Graph(mf.CrossEntropyLoss(head(layer(ids)), labels)), learning_rate=0.01)

    batches = [torch.randint(-1, 500, (300,), generator=torch.Generator().manual_seed(s)).cuda() for s in range(4)]
    results = []
    for kind in (None, mf.RecordedStep, mf.CapturedStep):
        layer, ids, optimizer = network()
        step = optimizer if kind is None else kind(optimizer)
        for batch in batches:
            ids.value.copy_(batch)
            step.one_step()
            step.update()
            torch.cuda.synchronize()
        results.append(layer.W.value.clone())
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@gpu
def test_an_optimized_graph_gives_the_plain_graphs_gradients():
    mf.set_device("cuda")
    ids = mf.Variable(torch.arange(50, device="cuda") % 7, requires_grad=False)
    labels = mf.Variable(torch.arange(50, device="cuda") % 9, requires_grad=False)
    grads = []
    for optimize in (False, True):
        layer = mf.Embedding(7, 12, initializer=mf.make_initializer("normal", seed=1, std=0.5))
        hidden = mf.Dense(12, 16, activation=mf.ReLU, initializer=mf.make_initializer(seed=2))
        head = mf.Dense(16, 9, initializer=mf.make_initializer(seed=3))
        graph = mf.Graph(mf.CrossEntropyLoss(head(hidden(layer(ids))), labels), optimize=optimize)
        graph.forward()
        graph.backward()
        grads.append(layer.W.grad)
    assert torch.equal(grads[0], grads[1])


@gpu
def test_calls_on_two_streams_do_not_share_their_workspace():
    g = torch.Generator().manual_seed(5)
    grads = [torch.randn((20000, 64), generator=g).cuda() for _ in range(2)]
    ids = [torch.randint(0, 37, (20000,), generator=g).cuda() for _ in range(2)]
    alone = [ops.embedding_backward(d, i, 37) for d, i in zip(grads, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, d, i in zip(streams, grads, ids):
            with torch.cuda.stream(s):
                got.append(ops.embedding_backward(d, i, 37))
        torch.cuda.synchronize()
        assert torch.equal(got[0], alone[0]) and torch.equal(got[1], alone[1])


def test_refusals_without_a_gpu():
    table, ids = torch.zeros((4, 3)), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="on the GPU"):
        ops.embedding_forward(table, ids)
    with pytest.raises(TypeError, match="on the GPU"):
        ops.embedding_backward(torch.zeros((2, 3)), ids, 4)
    with pytest.raises(ValueError, match="must be positive"):
        mf.Embedding(0, 3)
    with pytest.raises(ValueError, match="finite"):
        mf.Embedding(3, 3, scale=float("nan"))


@gpu
def test_refusals():
    table, ids = torch.zeros((4, 3), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    grad = torch.zeros((2, 3), device="cuda")
    for bad in (table.double(), table.int(), "table", table.cpu()):
        with pytest.raises(TypeError):
            ops.embedding_forward(bad, ids)
    for bad in (ids.short(), ids.float(), ids.cpu(), [0, 1]):
        with pytest.raises(TypeError):
            ops.embedding_forward(table, bad)
    for bad in (table[0], table.reshape(1, 4, 3), table[:0], table[:, :0]):
        with pytest.raises(ValueError):
            ops.embedding_forward(bad, ids)
    with pytest.raises(ValueError):
        ops.embedding_forward(table, ids, scale=float("inf"))
    for bad in (grad[:1], grad.reshape(2, 3, 1), grad[0], grad[:, :0]):
        with pytest.raises(ValueError):
            ops.embedding_backward(bad, ids, 4)
    for vocab in (0, -1, (1 << 24) + 1):
        with pytest.raises(ValueError):
            ops.embedding_backward(grad, ids, vocab)
    with pytest.raises(ValueError, match="add"):
        ops.embedding_backward(grad, ids, 4, add=True)
    for out in (torch.zeros((4, 4), device="cuda"), torch.zeros((3, 4), device="cuda").t(), table.half(), table.cpu(),
                torch.zeros((1, 3), device="cuda").expand(4, 3)):
        with pytest.raises(ValueError, match="out"):
            ops.embedding_backward(grad, ids, 4, out=out)


@gpu
def test_a_gradient_written_over_what_it_is_made_of_is_refused():
    held = torch.zeros((30, 8), device="cuda")
    ids = torch.zeros(10, dtype=torch.int64, device="cuda")
    for grad, out in ((held[:10], held[:4]), (held[:10], held[9:13]), (held[5:15, :4], held[:6, 3:7]),
                      (held[:10], held[10:14].view(-1).as_strided((4, 8), (8, 1), 79))):
        for add in (False, True):
            with pytest.raises(ValueError, match="share no memory"):
                ops.embedding_backward(grad, ids, out.shape[0], out=out, add=add)
    words = torch.zeros(40, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="share no memory"):
        ops.embedding_backward(torch.zeros((10, 8), device="cuda"), words[20:30], 4, out=words[10:].view(torch.float32)[:32].view(4, 8))
    grad = torch.randn((10, 8), device="cuda")
    want = ops.embedding_backward(grad[:, :3].contiguous(), ids, 10)
    assert torch.equal(ops.embedding_backward(grad[:, :3], ids, 10, out=grad[:, 4:7]), want)  # rows side by side


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.4028236e38, float("inf"), float("nan")])
def test_scales_beyond_float32_are_refused(scale):
    with pytest.raises(ValueError, match="finite"):
        mf.Embedding(3, 3, scale=scale)


@gpu
def test_the_largest_scale_leaves_zeros_and_unnamed_rows():
    scale = torch.finfo(torch.float32).max
    ids = torch.tensor([1, -1], device="cuda")
    y = ops.embedding_forward(torch.ones((3, 5), device="cuda"), ids, scale=scale)
    assert bool((y[0] == scale).all()) and bool((y[1] == 0).all())
    grad = ops.embedding_backward(torch.ones((2, 5), device="cuda"), ids, 3, scale=scale)
    assert bool((grad[1] == scale).all()) and bool((grad[[0, 2]] == 0).all())
    for call in (lambda: ops.embedding_forward(y, ids, scale=1e39), lambda: ops.embedding_backward(y, ids, 3, scale=1e39)):
        with pytest.raises(ValueError, match="finite"):
            call()
