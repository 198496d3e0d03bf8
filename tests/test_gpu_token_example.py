"""Embedding, Muon and adjusted logits as one program runs them: the example of a small network over tokens."""

import importlib.util
from pathlib import Path

import pytest
import torch

import myflows_amd as mf
from myflows_amd import logits

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def _example():
    spec = importlib.util.spec_from_file_location("token_network", ROOT / "examples" / "token_network.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_runs_and_its_answers_keep_to_the_grammar():
    history, tokens, allowed = _example().main(steps=5, vocab=100, dim=16, width=48, batch=64)
    assert len(history) == 5 and all(torch.isfinite(torch.tensor(history)))
    answers = tokens[:, 3:]
    assert tokens.shape == (4, 15) and bool(((answers >= 0) & (answers < 100)).all()) and bool(allowed[answers].all())


def _network(vocab=40, seed=5):
    mf.set_device("cuda")
    model = _example().TokenNetwork(vocab, 16, 24, groups=4, seed=seed)
    ids = mf.Variable(torch.randint(-1, vocab, (33,), generator=torch.Generator().manual_seed(1)).cuda(), requires_grad=False)
    labels = mf.Variable(torch.randint(0, vocab, (33,), generator=torch.Generator().manual_seed(2)).cuda(), requires_grad=False)
    loss = mf.CrossEntropyLoss(model(ids), labels)
    return model, ids, labels, loss


def test_gradients_of_the_network_against_64_bits():
    model, ids, labels, loss = _network()
    graph = mf.Graph(loss)
    graph.forward()
    graph.backward()
    leaves = {p: p.value.detach().cpu().double().requires_grad_(True) for p in model.params}
    t, w = ids.value.cpu(), lambda p: leaves[p]
    x = torch.where((t >= 0)[:, None], w(model.tokens.W)[t.clamp(min=0)], 0.0)
    x = x @ w(model.inner.W) + w(model.inner.b)
    g = x.reshape(33, 4, 6)
    hat = ((g - g.mean(2, keepdim=True)) / (g.var(2, unbiased=False, keepdim=True) + model.norm.eps).sqrt()).reshape(33, 24)
    u = hat * w(model.norm.gamma) + w(model.norm.beta)
    x = (u * torch.sigmoid(u)) @ w(model.back.W) + w(model.back.b)
    z = x @ w(model.head.W) + w(model.head.b)
    want = torch.nn.functional.cross_entropy(z, labels.value.cpu())
    want.backward()
    assert abs(float(loss.value) - float(want.detach())) <= 1e-5 * float(want.detach())
    for p, leaf in leaves.items():
        # A padded row is the same in every one of its places, so group norm divides by sqrt(eps) there: float32's relative
        # errors of some 2^-20 in the few products of each gradient stand against the largest of its elements.
        off = (p.grad.cpu().double().reshape(leaf.shape) - leaf.grad).abs().max()
        assert float(off) <= 2.0 ** -14 * float(leaf.grad.abs().max()), p.name


def test_a_training_step_and_an_answer_replayed_side_by_side():
    model, ids, labels, loss = _network()
    optimizer = mf.Muon(mf.Graph(loss), 0.02, adam_params=[model.tokens.W, model.head.W])
    step = mf.RecordedStep(optimizer)
    other, other_ids, other_labels, other_loss = _network()
    eager = mf.Muon(mf.Graph(other_loss), 0.02, adam_params=[other.tokens.W, other.head.W])
    allowed = _example().allowed_words(torch.arange(40) % 2 == 0).cuda()
    for k in range(3):
        batch = torch.randint(-1, 40, (33,), generator=torch.Generator().manual_seed(20 + k)).cuda()
        ids.value.copy_(batch)
        other_ids.value.copy_(batch)
        for one in (step, eager):
            one.one_step()
            one.update()
        for a, b in zip(model.params, other.params):
            assert torch.equal(a.value, b.value)
        first, second = (_example().answer(m, torch.tensor([[1, 2], [3, 4]], device="cuda"), 6, allowed) for m in (model, other))
        assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
        assert bool((first[0][:, 2:] % 2 == 0).all())
        assert bool((first[1][:, 1::2] == float("-inf")).all())
        assert bool(logits.log_probs_forward(first[1]).entropy.isfinite().all())
