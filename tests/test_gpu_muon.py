"""The Muon optimiser against its formulas in 64 bits, step by step from the state it holds.

Bounds (u = 2^-24). A momentum takes two float32 roundings, or one where the compiler fuses them: within
2 u (|momentum b| + |g|). The direction then carries a relative error of 4 u, which the orthogonalisation treats as
one of its own: as in its tests, the result is within 4 times the error that the same steps have in float32, and
2^-20 of it for the direction's and for matrices whose float32 error happens to be near 0. A parameter adds two roundings.
"""

import pytest
import torch

import myflows_amd as mf
from myflows_amd import orthogonal
from tests.test_gpu_orthogonal import _steps

U = 2.0 ** -24
gpu = pytest.mark.gpu


def _network(seed=0):
    mf.set_device("cuda")
    layer = mf.Embedding(60, 24, name="tokens", initializer=mf.make_initializer("normal", seed=seed, std=0.5))
    hidden = mf.Dense(24, 96, activation=mf.ReLU, name="hidden", initializer=mf.make_initializer(seed=seed + 1))
    back = mf.Dense(96, 24, name="back", initializer=mf.make_initializer(seed=seed + 2))
    head = mf.Dense(24, 60, name="head", initializer=mf.make_initializer(seed=seed + 3))
    ids = mf.Variable(torch.arange(40, device="cuda") % 60, requires_grad=False)
    labels = mf.Variable((torch.arange(40, device="cuda") * 7) % 60, requires_grad=False)
    graph = mf.Graph(mf.CrossEntropyLoss(head(back(hidden(layer(ids)))), labels))
    return graph, layer, hidden, back, head, ids


def _check_step(optimizer, matrices, factors, momentum, nesterov, decay, lr, grads):
    """grads: {node: the averaged gradient}; compares with the state before, which this function is given in factors."""
    for node in matrices:
        p, b, factor = factors[node]
        g = grads[node].double().cpu()
        want_b = momentum * b + g
        off = (optimizer.buffers[node].double().cpu() - want_b).abs()
        assert bool((off <= 2.01 * U * (momentum * b.abs() + g.abs()) + 2.0 ** -149).all())
        direction = (g + momentum * want_b if nesterov else want_b).float()
        o = _steps(direction, torch.float64)
        error = 4 * float((_steps(direction, torch.float32).double() - o).norm()) + 2.0 ** -19 * float(o.norm())
        want = (1 - lr * decay) * p - lr * factor * o
        off = float((node.value.double().cpu() - want).norm())
        assert off <= lr * factor * error + 3 * U * (float(p.norm()) + lr * factor * float(o.norm()))


@gpu
@pytest.mark.parametrize("nesterov,decay,accumulated", [(True, 0.0, 1), (False, 0.1, 1), (True, 0.1, 3)])
def test_steps_match_the_formulas(nesterov, decay, accumulated):
    graph, layer, hidden, back, head, ids = _network()
    matrices = [hidden.W, back.W]
    groups = [{"name": "matrices", "params": matrices, "weight_decay": decay}]
    optimizer = mf.Muon(graph, 0.05, 0.9, nesterov=nesterov, adam_params=[layer.W, head.W], adam_learning_rate=0.01, param_groups=groups)
    factors = {hidden.W: 2.0, back.W: 1.0}  # 24 -> 96, 96 -> 24
    # The others are Adam's, with the bits of an Adam of their own.
    twin, layer2, hidden2, back2, head2, ids2 = _network()
    adam = mf.Adam(twin, 0.01)
    for step in range(3):
        before = {n: (n.value.double().cpu(), optimizer.buffers[n].double().cpu() if n in optimizer.buffers else
                      torch.zeros(n.value.shape, dtype=torch.float64), factors[n]) for n in matrices}
        for k in range(accumulated):
            batch = torch.randint(-1, 60, (40,), generator=torch.Generator().manual_seed(10 * step + k)).cuda()
            for tokens, one in ((ids, optimizer), (ids2, adam)):
                tokens.value = batch
                one.one_step()
        grads = {n: optimizer.get_gradient(n).clone() for n in matrices}
        optimizer.update()
        _check_step(optimizer, matrices, before, 0.9, nesterov, decay, 0.05, grads)
        for mine, other in ((hidden, hidden2), (back, back2)):
            other.W.value.copy_(mine.W.value)
        adam.acc_gradient.pop(hidden2.W), adam.acc_gradient.pop(back2.W)
        adam.update()
        for mine, other in zip((layer.W, head.W, head.b, hidden.b, back.b), (layer2.W, head2.W, head2.b, hidden2.b, back2.b)):
            assert torch.equal(mine.value, other.value)
    assert set(optimizer.buffers) == set(matrices) and optimizer.t == 3


@gpu
def test_convolution_kernels_are_outputs_by_the_rest():
    mf.set_device("cuda")
    conv = mf.Conv2D(3, 70, 3, padding=1, initializer=mf.make_initializer(seed=5))
    x = mf.Variable(torch.randn((4, 3, 9, 9), generator=torch.Generator().manual_seed(1)).cuda(), requires_grad=False)
    loss = mf.MSELoss(conv(x), mf.Variable(torch.ones((4, 70, 9, 9), device="cuda"), requires_grad=False))
    optimizer = mf.Muon(mf.Graph(loss), 0.02)
    before = {conv.kernel: (conv.kernel.value.double().cpu(), torch.zeros(conv.kernel.value.shape, dtype=torch.float64), (70 / 27) ** 0.5)}
    optimizer.one_step()
    grads = {conv.kernel: optimizer.get_gradient(conv.kernel).clone()}
    optimizer.update()
    _check_step(optimizer, [conv.kernel], before, 0.95, True, 0.0, 0.02, grads)
    assert conv.b in optimizer.parameter_steps and conv.kernel not in optimizer.parameter_steps


@gpu
def test_recorded_and_captured_steps_repeat_the_eager_bits():
    results = []
    for kind in (None, mf.RecordedStep, mf.CapturedStep):
        graph, layer, hidden, back, head, ids = _network(3)
        optimizer = mf.Muon(graph, 0.02, adam_params=[layer.W, head.W])
        step = optimizer if kind is None else kind(optimizer)
        for seed in range(4):
            ids.value.copy_(torch.randint(0, 60, (40,), generator=torch.Generator().manual_seed(seed)))
            step.one_step()
            step.update()
            torch.cuda.synchronize()
        results.append([n.value.clone() for n in graph.nodes if getattr(n, "trainable", False)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@gpu
def test_many_parameters_strides_and_empty_ones():
    g = torch.Generator().manual_seed(2)
    make = lambda *shape: torch.randn(shape, generator=g).cuda()  # noqa: E731
    updates = [(make(5 + i, 40), make(5 + i, 40), make(5 + i, 40), 0.1, 0.01) for i in range(70)]
    strided = make(30, 20).t()
    updates += [(strided, make(20, 30), make(30, 20).t(), 0.1, 0.0), (make(0, 4), make(0, 4), make(0, 4), 0.1, 0.0)]
    alone = [[t.clone() for t in update[:3]] for update in updates]
    orthogonal.muon_update_many(updates)
    for (param, grad, buffer, rate, decay), (p, g1, b) in zip(updates, alone):
        orthogonal.muon_update_many([(p, g1, b, rate, decay)])
        assert torch.equal(param, p) and torch.equal(buffer, b) and torch.equal(grad, g1)


@gpu
def test_refusals():
    graph, layer, hidden, back, head, ids = _network()
    for options in (dict(momentum=1.0), dict(momentum=-0.1), dict(steps=0), dict(adam_learning_rate=-1.0),
                    dict(adam_params=[mf.Variable(torch.zeros(3))])):
        with pytest.raises(ValueError):
            mf.Muon(graph, **options)
    p, g, b = (torch.zeros((4, 5), device="cuda") for _ in range(3))
    for bad in ((p, g[:3], b), (p, g, b.t()), (p, p, b), (p, g, p), (p[0], g[0], b[0])):
        with pytest.raises(ValueError):
            orthogonal.muon_update_many([(*bad, 0.1, 0.0)])
    for bad in ((p.half(), g, b), (p, g.cpu(), b), (p, g, b.double())):
        with pytest.raises(TypeError):
            orthogonal.muon_update_many([(*bad, 0.1, 0.0)])
    same = torch.ones((4, 5), device="cuda")  # one gradient of two parameters is no overlap
    orthogonal.muon_update_many([(p.clone(), same, b.clone(), 0.1, 0.0), (p.clone(), same, b.clone(), 0.1, 0.0)])
    with pytest.raises(ValueError, match="overlap"):
        orthogonal.muon_update_many([(p, g, b, 0.1, 0.0), (g, torch.ones_like(p), torch.ones_like(p), 0.1, 0.0)])


@gpu
def test_overlap_is_that_of_the_tensors_given_not_of_their_copies():
    make = lambda *shape: torch.randn(shape, device="cuda")  # noqa: E731
    w, one = make(6, 6), torch.ones((6, 6), device="cuda")
    alike = make(6, 12)
    for updates in ([(w.t(), one, make(6, 6), 0.1, 0.0), (w, one, make(6, 6), 0.1, 0.0)],
                    [(w.t(), one, w, 0.1, 0.0)], [(w.t(), one, w.t(), 0.1, 0.0)], [(w.t(), w, make(6, 6), 0.1, 0.0)],
                    [(alike[:, :6], one, alike[:, 5:11], 0.1, 0.0)], [(make(1, 6).expand(6, 6), one, make(6, 6), 0.1, 0.0)],
                    [(make(6, 6), one, make(6, 1).expand(6, 6), 0.1, 0.0)]):
        before = [[t.clone() for t in update[:3]] for update in updates]
        with pytest.raises(ValueError, match="overlap"):
            orthogonal.muon_update_many(updates)
        assert all(torch.equal(a, b) for update, held in zip(updates, before) for a, b in zip(update, held))
    # Columns side by side are no overlap.
    left, right, momentum = alike[:, :6], alike[:, 6:], torch.zeros((6, 12), device="cuda")
    twins = [(t.clone(), torch.zeros((6, 6), device="cuda")) for t in (left, right)]
    orthogonal.muon_update_many([(left, one, momentum[:, :6], 0.1, 0.0), (right, one, momentum[:, 6:], 0.1, 0.0)])
    orthogonal.muon_update_many([(p, one, b, 0.1, 0.0) for p, b in twins])
    assert torch.equal(alike, torch.cat([p for p, _ in twins], 1)) and torch.equal(momentum, torch.cat([b for _, b in twins], 1))


@gpu
def test_a_head_of_two_outputs_in_recorded_and_captured_steps():
    mf.set_device("cuda")
    results = []
    for kind in (None, mf.RecordedStep, mf.CapturedStep):
        hidden = mf.Dense(40, 70, activation=mf.ReLU, initializer=mf.make_initializer(seed=1))
        head = mf.Dense(70, 2, initializer=mf.make_initializer(seed=2))  # a matrix of two columns beside one of 40 rows
        x = mf.Variable(torch.zeros((30, 40), device="cuda"), requires_grad=False)
        target = mf.Variable(torch.ones((30, 2), device="cuda"), requires_grad=False)
        optimizer = mf.Muon(mf.Graph(mf.MSELoss(head(hidden(x)), target)), 0.02)
        step = optimizer if kind is None else kind(optimizer)
        for seed in range(5):
            x.value.copy_(torch.randn((30, 40), generator=torch.Generator().manual_seed(seed)))
            step.one_step()
            step.update()
            torch.cuda.synchronize()
        assert set(optimizer.buffers) == {hidden.W, head.W}
        results.append([p.value.clone() for p in (hidden.W, head.W, hidden.b, head.b)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
