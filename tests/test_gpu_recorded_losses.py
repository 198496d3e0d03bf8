"""The losses over logits and the group norm in a RecordedStep: what a recorded pass reads is read in place, so
that a replay sees the labels, records and weights of the moment, and a pass that a replay could not repeat is
refused while it is recorded."""

import pytest
import torch

import myflows_amd as mf

pytestmark = pytest.mark.gpu

ROWS, CLASSES, POSITIONS = 96, 300, 12


def _constant(value):
    return mf.Variable(value, requires_grad=False)


def _network(make_loss):
    """(parameters, input, loss, optimiser) of Dense -> group norm -> Dense -> loss."""
    draw = mf.make_initializer(seed=1)
    mf.set_device("cuda")
    inner, head = mf.Dense(32, 64, initializer=draw), mf.Dense(64, CLASSES, initializer=draw)
    norm = mf.GroupNorm(8, 64, activation="silu", positions=POSITIONS)
    x = _constant(torch.zeros((ROWS, 32), device="cuda"))
    loss = make_loss(head(norm(inner(x))))
    return inner.params + norm.params + head.params, x, loss, mf.Adam(mf.Graph(loss), learning_rate=1e-2)


def _steps_agree(make_loss, refresh):
    """A network stepped eagerly and its twin stepped by replays, with inputs, and what refresh(i) writes, new
    before each step."""
    eager_params, eager_x, eager_loss, eager = _network(make_loss)
    params, x, loss, optimizer = _network(make_loss)
    step = mf.RecordedStep(optimizer)
    for i in range(4):
        batch = torch.randn((ROWS, 32), generator=torch.Generator().manual_seed(40 + i)).cuda()
        eager_x.value.copy_(batch)
        x.value.copy_(batch)
        refresh(torch.Generator().manual_seed(80 + i))
        eager.one_step()
        step.one_step()
        torch.cuda.synchronize()
        assert torch.equal(loss.value, eager_loss.value), f"loss of step {i}"
        for a, b in zip(params, eager_params):
            assert torch.equal(a.grad, b.grad), f"a gradient of step {i}"
        eager.update()
        step.update()
    step.close()


@pytest.mark.parametrize("dtype", (torch.int32, torch.int64))
def test_a_recorded_cross_entropy_reads_a_column_of_labels(dtype):
    """Labels that are a column of a teacher's alternatives, refreshed in place between the replays."""
    print("recorded cross entropy", dtype, flush=True)
    ids = torch.randint(-1, CLASSES, (ROWS, 20), generator=torch.Generator().manual_seed(2)).to(dtype).cuda()

    def refresh(g):
        ids.copy_(torch.randint(-1, CLASSES, (ROWS, 20), generator=g))

    _steps_agree(lambda out: mf.CrossEntropyLoss(out, _constant(ids[:, 0])), refresh)


def test_a_recorded_distillation_reads_slices_of_a_record():
    """The first six of twenty recorded alternatives, and row weights that are a column of a table."""
    print("recorded distillation", flush=True)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, CLASSES, (ROWS, 20), generator=g).int().cuda()
    teacher, weights = torch.randn((ROWS, 20), generator=g).cuda(), torch.rand((ROWS, 3), generator=g).cuda()

    def refresh(g):
        ids.copy_(torch.randint(-1, CLASSES, (ROWS, 20), generator=g))
        teacher.copy_(torch.randn((ROWS, 20), generator=g))
        weights.copy_(torch.rand((ROWS, 3), generator=g))

    _steps_agree(lambda out: mf.DistillationLoss(out, _constant(ids[:, :6]), _constant(teacher[:, :6]),
                                                 _constant(weights[:, 1]), temperature=1.5), refresh)


def _sum_of_losses(out):
    ids = torch.randint(0, CLASSES, (ROWS, 6), generator=torch.Generator().manual_seed(4)).cuda()
    teacher = torch.randn((ROWS, 6), generator=torch.Generator().manual_seed(5)).cuda()
    return mf.Add(mf.CrossEntropyLoss(out, _constant(ids[:, 0])), mf.DistillationLoss(out, _constant(ids), _constant(teacher)))


def _turned_record(out):
    ids = torch.randint(0, CLASSES, (6, ROWS), generator=torch.Generator().manual_seed(4)).cuda()
    teacher = torch.randn((6, ROWS), generator=torch.Generator().manual_seed(5)).cuda()
    return mf.DistillationLoss(out, _constant(ids.t()), _constant(teacher.t()))


@pytest.mark.parametrize("make_loss", (_sum_of_losses, _turned_record))
def test_work_of_another_library_is_refused_while_a_pass_is_recorded(make_loss):
    """Torch's own launches (an Add, a copy of a tensor whose rows are not contiguous) are no steps of the program: a
    replay would read what they left, or what has been written there since. The pass runs eagerly as ever."""
    print("refused in a recorded pass", make_loss.__name__, flush=True)
    _, _, loss, optimizer = _network(make_loss)
    with pytest.raises(RuntimeError, match="recorded"):
        mf.RecordedStep(optimizer)
    optimizer.one_step()
    assert bool(torch.isfinite(loss.value)) and bool(torch.ones(3, device="cuda").add(1.0).eq(2.0).all())
    labels = _constant(torch.zeros(ROWS, dtype=torch.int64, device="cuda"))
    mf.RecordedStep(_network(lambda out: mf.CrossEntropyLoss(out, labels))[3]).close()


@pytest.mark.parametrize("replayed", (mf.RecordedStep, mf.CapturedStep))
def test_a_classifier_of_images_trains_on_labels_through_replays(replayed):
    """ResNet18 with a cross entropy: the eager steps' loss and parameters, bit for bit, with new images and labels
    before each step."""
    print("resnet cross entropy", replayed.__name__, flush=True)
    table = torch.zeros((4, 3), dtype=torch.int64, device="cuda")

    def build():
        model = mf.ResNet18(output_dim=10, base_width=16, initializer=mf.make_initializer(seed=0), conv_backend="hip_native")
        x = _constant(torch.ones((4, 3, 48, 64), device="cuda"))
        loss = mf.CrossEntropyLoss(model(x), _constant(table[:, 1]))
        return model, x, loss, mf.Adam(mf.Graph(loss, optimize=True), learning_rate=1e-3)

    mf.set_device("cuda")
    eager_model, eager_x, eager_loss, eager = build()
    model, x, loss, optimizer = build()
    step = replayed(optimizer, warmup=1)
    for _ in range(1 + (replayed is mf.RecordedStep)):  # the passes so far moved the running statistics
        eager.graph.forward()
        eager.graph.backward()
    for i in range(3):
        g = torch.Generator().manual_seed(60 + i)
        images = torch.randn((4, 3, 48, 64), generator=g).cuda()
        eager_x.value.copy_(images)
        x.value.copy_(images)
        table.copy_(torch.randint(-1, 10, (4, 3), generator=g))
        eager.one_step()
        step.one_step()
        torch.cuda.synchronize()
        assert torch.equal(loss.value, eager_loss.value), f"loss of step {i}"
        eager.update()
        step.update()
        for a, b in zip(model.params, eager_model.params):
            assert torch.equal(a.value, b.value), f"a parameter after step {i}"
