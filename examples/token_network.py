"""A small network over tokens: trained with Muon, answering under a grammar.

Each position's token is looked up in an embedding; Dense networks with a group norm between them say which
token comes next. The matrices in the middle are updated by ``Muon``, the table and the head by its Adam. The
trained network then answers token by token: its logits lose the penalties of what the stream holds already and
what the grammar rules out (``adjust_logits``), and the most likely token left is taken (``log_probs_forward``).

    python examples/token_network.py [--steps 40]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import myflows_amd as mf  # noqa: E402
from myflows_amd import logits  # noqa: E402


class TokenNetwork(mf.Layer):
    """Embedding -> Dense -> group norm and SiLU -> Dense, a row for each position (its own group norm sample)."""

    def __init__(self, vocab, dim, width, groups=8, seed=1):
        super().__init__()
        draw = mf.make_initializer(seed=seed)
        self.tokens = mf.Embedding(vocab, dim, initializer=mf.make_initializer("normal", seed=seed, std=0.5), name="tokens")
        self.inner = mf.Dense(dim, width, initializer=draw, name="inner")
        self.norm = mf.GroupNorm(groups, width, activation="silu", positions=1)
        self.back = mf.Dense(width, dim, initializer=draw, name="back")
        self.head = mf.Dense(dim, vocab, initializer=draw, name="head")
        self.params = [p for layer in (self.tokens, self.inner, self.norm, self.back, self.head) for p in layer.params]

    def forward(self, ids):
        return self.head(self.back(self.norm(self.inner(self.tokens(ids)))))


def constant(value):
    return mf.Variable(value, requires_grad=False)


def answer(model, prompt, length, allowed):
    """(prompt with `length` tokens behind it, the last adjusted logits) of each row of a prompt, by the most likely token."""
    held, tokens = prompt.shape[1], prompt
    lengths = torch.full((prompt.shape[0],), held, device=prompt.device)
    ids = constant(prompt[:, -1].clone())
    node = model(ids)
    graph = mf.Graph(node)
    for _ in range(length):
        ids.value = tokens[:, -1].contiguous()
        graph.forward()
        adjusted = logits.adjust_logits(node.value, tokens=tokens, prompt_lengths=lengths, repetition=1.1, presence=0.5,
                                        frequency=0.25, allowed=allowed)
        best = logits.log_probs_forward(adjusted, top=1).top_ids
        tokens = torch.cat([tokens, best.to(tokens.dtype)], dim=1)
    return tokens, adjusted


def allowed_words(allowed):
    """The words of a mask from whether each token is allowed."""
    words = torch.zeros(-(-len(allowed) // 32) * 32, dtype=torch.int64)
    words[:len(allowed)] = allowed.long()
    packed = (words.view(-1, 32) << torch.arange(32)).sum(dim=1)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()


def main(steps=40, vocab=500, dim=64, width=192, batch=512, streams=4, length=12):
    mf.set_device("cuda")
    generator = torch.Generator().manual_seed(0)
    following = torch.randperm(vocab, generator=generator)  # what comes after each token
    model = TokenNetwork(vocab, dim, width)
    ids = constant(torch.zeros(batch, dtype=torch.int64, device="cuda"))
    labels = constant(torch.zeros(batch, dtype=torch.int64, device="cuda"))
    loss = mf.CrossEntropyLoss(model(ids), labels)
    optimizer = mf.Muon(mf.Graph(loss), 0.02, adam_params=[model.tokens.W, model.head.W], adam_learning_rate=1e-2)
    history = []
    for step in range(steps):
        drawn = torch.randint(0, vocab, (batch,), generator=generator)
        ids.value.copy_(drawn)
        labels.value.copy_(following[drawn])
        optimizer.one_step()
        optimizer.update()
        history.append(float(loss.value))
        if step % 10 == 0 or step == steps - 1:
            print(f"step {step:3d}  cross entropy {history[-1]:.4f}", flush=True)

    allowed = torch.arange(vocab) % 3 != 0
    prompt = torch.randint(0, vocab, (streams, 3), generator=generator).cuda()
    tokens, _ = answer(model, prompt, length, allowed_words(allowed).cuda())
    print("answers", tokens[:, 3:].tolist())
    return history, tokens.cpu(), allowed


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=40)
    main(parser.parse_args().steps)
