"""The three operators as one program runs them: the example of a student that learns from a teacher's recorded
answers, and such a step recorded as a library program."""

import importlib.util
from pathlib import Path

import pytest
import torch

import myflows_amd as mf
from myflows_amd import logits

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def _example():
    spec = importlib.util.spec_from_file_location("distill_student", ROOT / "examples" / "distill_student.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_student_learns():
    history, agree = _example().main(steps=40, samples=16)
    for loss in zip(*history):  # both losses fall from each ten steps to the next
        tens = [sum(loss[i:i + 10]) for i in range(0, 40, 10)]
        assert tens == sorted(tens, reverse=True)
    assert agree > 0.5


def _student_step(seed=3):
    example = _example()
    mf.set_device("cuda")
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn((8 * 12, 32), generator=g).cuda()
    ids = torch.randint(0, 300, (96, 6), generator=g).cuda()
    teacher = torch.randn((96, 6), generator=g).cuda()
    student = example.Student(32, 64, 300, 12)
    x = mf.Variable(rows, requires_grad=False)
    loss = mf.DistillationLoss(student(x), example.constant(ids), example.constant(teacher), temperature=1.5)
    return student, x, loss, mf.Adam(mf.Graph(loss), learning_rate=1e-2)


def test_a_recorded_step_repeats_the_eager_one_bit_for_bit():
    eager_student, eager_x, eager_loss, eager = _student_step()
    student, x, loss, optimizer = _student_step()
    step = mf.RecordedStep(optimizer)
    for i in range(4):
        batch = torch.randn((96, 32), generator=torch.Generator().manual_seed(10 + i)).cuda()
        eager_x.value.copy_(batch)
        x.value.copy_(batch)
        eager.one_step()
        step.one_step()
        torch.cuda.synchronize()
        assert torch.equal(loss.value, eager_loss.value)
        for a, b in zip(student.params, eager_student.params):
            assert torch.equal(a.grad, b.grad)
        eager.update()
        step.update()


def test_the_operators_in_a_captured_graph():
    """A captured graph of split rows, the loss of few rows and its gradient, replayed with eager work between the
    replays: every replay gives the eager bits on the inputs of the moment."""
    g = torch.Generator().manual_seed(5)
    z = torch.randn((3, 60000), generator=g).cuda()
    tokens = torch.randint(0, 60000, (3,), generator=g).cuda()
    ids, teacher = torch.randint(0, 60000, (3, 8), generator=g).cuda(), torch.randn((3, 8), generator=g).cuda()
    seed = torch.ones((), device="cuda")
    x = torch.randn((2, 3000, 48), generator=g).cuda()
    gamma, beta = torch.rand(48, generator=g).cuda(), torch.rand(48, generator=g).cuda()

    def run():
        r = logits.log_probs_forward(z, tokens, top=30)
        d = logits.distill_loss_forward(z, ids, teacher)
        grad = logits.distill_loss_backward(z, ids, d, seed)
        y, mean, inv_std = mf.group_norm.group_norm_forward(x, gamma, beta, 6, activation="silu")
        return [*r, d.loss, d.row_loss, grad, y, mean, inv_std]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for i in range(3):
        z.copy_(torch.randn(z.shape, generator=g).cuda())
        x.mul_(1.25)
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


def test_captured_graphs_share_no_scratch_memory():
    """Two graphs of calls that join workgroups, captured one after the other: the second is replayed first, then
    both side by side on two streams. One of them forks to a second stream within its capture."""
    g = torch.Generator().manual_seed(6)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    rows = [torch.randn((4, 120000), generator=g).cuda() for _ in range(4)]
    ids, teacher = torch.randint(0, 120000, (4, 8), generator=g).cuda(), torch.randn((4, 8), generator=g).cuda()

    def run(z):
        r = logits.log_probs_forward(z, top=20)
        d = logits.distill_loss_forward(z, ids, teacher)
        return [r.entropy, r.log_sum, r.top_log_probs, r.top_ids, d.scale, d.row_loss]

    want = [run(z) for z in rows]
    torch.cuda.synchronize()
    graphs, captured = [], []
    for i in range(2):
        graph, outputs = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(graph):
            outputs.append(run(rows[2 * i]))
            if i == 1:
                sides[0].wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(sides[0]):
                    outputs.append(run(rows[2 * i + 1]))
                torch.cuda.current_stream().wait_stream(sides[0])
            else:
                outputs.append(run(rows[2 * i + 1]))
        graphs.append(graph)
        captured.append(outputs)

    def check(which):
        for i in which:
            for j in range(2):
                for a, b in zip(captured[i][j], want[2 * i + j]):
                    assert torch.equal(a, b)
                    a.zero_()
        torch.cuda.synchronize()

    graphs[1].replay()
    torch.cuda.synchronize()
    check([1])
    for _ in range(5):
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        check([0, 1])


def test_a_capture_keeps_no_memory_beyond_its_graph():
    """The scratch memory of a capture is given up by the first eager call after it that takes some itself. The graph
    keeps it for its replays (no later tensor gets it), and without the graph it is free."""
    g = torch.Generator().manual_seed(7)
    z = torch.randn((2, 120000), generator=g).cuda()
    ids, teacher = torch.randint(0, 120000, (2, 8), generator=g).cuda(), torch.randn((2, 8), generator=g).cuda()

    def run():
        r = logits.log_probs_forward(z, top=64)
        return [r.entropy, r.log_sum, r.top_log_probs, r.top_ids, logits.distill_loss_forward(z, ids, teacher).scale]

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
        during = len(mf.native._CAPTURE_BLOCKS)
        assert during >= 1
    want = run()
    assert not mf.native._CAPTURE_BLOCKS
    later = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in (512, 2048, 4100, 8192, 16384, 65536, 2 ** 20) * 8]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
    assert all(bool((t == 7).all()) for t in later)
