"""A student learns from a larger network's recorded answers.

A teacher (Dense networks over the positions of short sequences) answers once: ``log_probs_forward`` records the
ids and log probabilities of each position's most likely classes. A student, whose activations a group norm
normalises sample by sample, is trained on that record (``DistillationLoss``) and on the labels
(``CrossEntropyLoss``), and answers in turn: the labels' log probabilities, the entropy, the best classes.

    python examples/distill_student.py [--steps 60]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import myflows_amd as mf  # noqa: E402
from myflows_amd import logits  # noqa: E402


class Student(mf.Layer):
    """Dense -> group norm and SiLU -> Dense, over rows that are the positions of the samples in turn."""

    def __init__(self, features, width, classes, positions, groups=8, seed=1):
        super().__init__()
        draw = mf.make_initializer(seed=seed)
        self.inner = mf.Dense(features, width, initializer=draw)
        self.norm = mf.GroupNorm(groups, width, activation="silu", positions=positions)
        self.head = mf.Dense(width, classes, initializer=draw)
        self.params = self.inner.params + self.norm.params + self.head.params

    def forward(self, rows):
        return self.head(self.norm(self.inner(rows)))


def constant(value):
    return mf.Variable(value, requires_grad=False)


def answers(model, rows):
    """The logits of a model, without a backward pass."""
    node = model(constant(rows))
    mf.Graph(node).forward()
    return node.value


def main(steps=60, samples=64, positions=20, features=64, classes=1000, held=20, temperature=2.0):
    mf.set_device("cuda")
    generator = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.randn((samples * positions, features), generator=generator, device="cuda")

    teacher = Student(features, 512, classes, positions, seed=7)
    teacher.head.W.value = 3.0 * teacher.head.W.value  # answers that differ from one another
    record = logits.log_probs_forward(answers(teacher, rows), top=held)
    labels = record.top_ids[:, 0].clone()
    labels[::10] = -1  # a tenth of the positions has no label

    student = Student(features, 128, classes, positions)
    out = student(constant(rows))
    distillation = mf.DistillationLoss(out, constant(record.top_ids), constant(record.top_log_probs),
                                       temperature=temperature)
    cross_entropy = mf.CrossEntropyLoss(out, constant(labels))
    optimizer = mf.Adam(mf.Graph(mf.Add(distillation, cross_entropy)), learning_rate=3e-3)
    history = []
    for step in range(steps):
        optimizer.one_step()
        optimizer.update()
        history.append((float(distillation.value), float(cross_entropy.value)))
        if step % 10 == 0 or step == steps - 1:
            print(f"step {step:3d}  distillation {history[-1][0]:.4f}  cross entropy {history[-1][1]:.4f}", flush=True)

    answer = logits.log_probs_forward(answers(student, rows), labels, top=5)
    agree = float((answer.top_ids[:, 0] == record.top_ids[:, 0]).float().mean())
    print(f"agreement {agree:.3f}  entropy {float(answer.entropy.mean()):.3f}  "
          f"log prob of the labels {float(answer.log_prob[labels >= 0].mean()):.3f}")
    return history, agree


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    main(parser.parse_args().steps)
