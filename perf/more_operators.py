"""The first layer, the update and the answers of a network over tokens, as cases to time and compare.

Three operators: the embedding lookup with scaling and its gradient by sorted tokens; the adjustment of
logits before they are answered with (penalties for tokens that were given before, biases, a grammar's
mask); the orthogonalisation of matrices by Newton-Schulz products, a list of them at a time, as an
optimiser's update takes its parameters.

``listed()`` gives the cases by name, ``draw(rng)`` one more of the same ranges, ``prepare`` makes what
a program has in hand before the call, ``run`` is one pass (the plain torch form, or with ``own`` the
framework's operators), ``work`` what a pass cannot do without and ``exact`` the definition in 64 bits.
"""

from __future__ import annotations

import torch

own = False
DEVICE = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}
NEG_INF = float("-inf")
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
# The weights of ResNet18 with two outputs: each convolution's kernel as (CO, CI * KH * KW), and the head's.
RESNET18 = "64x147,64x576*4,128x576,128x1152*3,128x64,256x1152,256x2304*3,256x128,512x2304,512x4608*3,512x256,512x2"


def listed():
    return [
        # One decoding step of 64 streams: their rows of the table; latency counts.
        {"name": "embedding_decode", "kind": "embedding", "tokens": 64, "vocab": 131072, "dim": 1024,
         "type": "bfloat16", "train": False, "missing": False},
        # A small network's training pass: a batch of 4096 tokens over 1000 classes of them.
        {"name": "embedding_small", "kind": "embedding", "tokens": 4096, "vocab": 1000, "dim": 512, "type": "float32",
         "train": True, "missing": False},
        # Odd sizes throughout, padded batches: one token in sixteen is none.
        {"name": "embedding_odd", "kind": "embedding", "tokens": 10007, "vocab": 50021, "dim": 771, "type": "float16",
         "train": True, "missing": True},
        # A large batch of text: some tokens come thousands of times, most of the table's rows never.
        {"name": "embedding_large", "kind": "embedding", "tokens": 65536, "vocab": 65536, "dim": 2048,
         "type": "bfloat16", "train": True, "missing": False},
        # One decoding step of one stream, a long answer behind it; latency counts.
        {"name": "adjust_one_row", "kind": "adjust", "rows": 1, "vocab": 131072, "held": 2048, "biases": 8,
         "mask": True, "pad": 0, "type": "bfloat16"},
        # Rows that are slices of a padded product, an odd vocabulary, short histories, no grammar.
        {"name": "adjust_odd", "kind": "adjust", "rows": 333, "vocab": 32771, "held": 257, "biases": 40, "mask": False,
         "pad": 61, "type": "float32"},
        # A large batch of streams under grammars: bandwidth counts.
        {"name": "adjust_batch", "kind": "adjust", "rows": 512, "vocab": 131072, "held": 4096, "biases": 16,
         "mask": True, "pad": 0, "type": "float16"},
        # The kernel of one 3x3 convolution of layer1: latency counts.
        {"name": "orthogonal_one", "kind": "orthogonal", "shapes": "64x576", "type": "float32"},
        # Every weight of ResNet18: one step of an optimiser.
        {"name": "orthogonal_resnet18", "kind": "orthogonal", "shapes": RESNET18, "type": "float32"},
        # Odd sizes, one matrix tall and one wide.
        {"name": "orthogonal_odd", "kind": "orthogonal", "shapes": "1999x517,771x1003", "type": "float16"},
        # A wide Dense layer's weight and the one behind it.
        {"name": "orthogonal_wide", "kind": "orthogonal", "shapes": "1024x4096,4096x1024", "type": "bfloat16"},
        # A large square weight: the matrix cores count.
        {"name": "orthogonal_large", "kind": "orthogonal", "shapes": "4096x4096", "type": "bfloat16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["embedding", "adjust", "orthogonal"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "embedding":
        dim, vocab = _spread(rng, 16, 4096), _spread(rng, 100, 131072)
        vocab = min(vocab, 2 ** 27 // dim)
        return {"kind": kind, "tokens": _spread(rng, 1, min(65536, 2 ** 27 // dim)), "vocab": vocab, "dim": dim,
                "type": dtype, "train": rng.random() < 0.7, "missing": rng.random() < 0.5}
    if kind == "adjust":
        vocab = _spread(rng, 100, 131072)
        return {"kind": kind, "rows": _spread(rng, 1, min(512, 2 ** 25 // vocab)), "vocab": vocab,
                "held": _spread(rng, 1, 4096), "biases": rng.choice([0, rng.randint(1, 64)]),
                "mask": rng.random() < 0.5, "pad": rng.choice([0, 0, rng.randint(1, 63)]), "type": dtype}
    shapes = []
    for _ in range(rng.choice([1, 1, 2, 4])):
        short = _spread(rng, 4, 1024)
        sides = short, _spread(rng, short, min(8 * short, 4096))
        shapes.append("%dx%d" % (sides if rng.random() < 0.5 else sides[::-1]))
    return {"kind": kind, "shapes": ",".join(shapes), "type": dtype}


def _shapes(case):
    """The (rows, columns) of each matrix of a case; "64x576*4" is four of them."""
    parts = [(part.split("*") + ["1"])[:2] for part in case["shapes"].split(",")]
    return [tuple(int(v) for v in shape.split("x")) for shape, count in parts for _ in range(int(count))]


def _ids(g, vocab, shape):
    """Tokens as text has them: the k-th most frequent has a share of about 1 / k."""
    u = torch.rand(shape, generator=g, device=DEVICE, dtype=torch.float64)
    return (torch.exp(u * torch.log(torch.tensor(vocab + 1.0, dtype=torch.float64))).long() - 1).clamp(0, vocab - 1)


def _inputs(case, seed):
    """The data of a case, made from the seed alone."""
    g, dtype = torch.Generator(device=DEVICE).manual_seed(seed), TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)  # noqa: E731
    if case["kind"] == "orthogonal":
        matrices = []
        for rows, columns in _shapes(case):
            # The momentum of gradients: a few strong directions over a noise that is not small.
            rank = max(1, min(rows, columns) // 8)
            strong = normal(rows, rank) * (0.5 + 3.0 * uniform(rank)) @ normal(rank, columns)
            matrices.append(((strong / rank ** 0.5 + normal(rows, columns)) * 1e-3).to(dtype))
        return {"matrices": matrices}
    vocab = case["vocab"]
    if case["kind"] == "embedding":
        tokens, dim = case["tokens"], case["dim"]
        ids = _ids(g, vocab, (tokens,))
        if case["missing"]:
            ids = torch.where(uniform(tokens) < 1 / 16, torch.full_like(ids, -1), ids)
        return {"table": normal(vocab, dim).to(dtype), "ids": ids, "scale": float(dim) ** 0.5,
                "grad": (normal(tokens, dim) * 0.1).to(dtype) if case["train"] else None}
    rows, held = case["rows"], case["held"]
    z = (normal(rows, vocab + case["pad"]) * 3.0).to(dtype)
    tokens = _ids(g, vocab, (rows, held))
    # Streams of unlike lengths, each a prompt and an answer; none behind their ends.
    length = (uniform(rows) * held).long() + 1
    tokens = torch.where(torch.arange(held, device=DEVICE) < length[:, None], tokens, torch.full_like(tokens, -1))
    data = {"logits": z[:, :vocab], "tokens": tokens, "prompt_lengths": (uniform(rows) * length).long(),
            "repetition": 1.0 + 0.5 * uniform(rows), "presence": uniform(rows) - 0.3, "frequency": 0.4 * uniform(rows),
            "bias_ids": None, "bias_values": None, "allowed": None}
    if case["biases"]:
        data.update(bias_ids=torch.randint(0, vocab, (rows, case["biases"]), generator=g, device=DEVICE),
                    bias_values=4.0 * normal(rows, case["biases"]))
    if case["mask"]:
        # A grammar leaves a row most tokens, or few of them.
        words = -(-vocab // 32)
        bits = (uniform(rows, words, 32) < torch.where(uniform(rows) < 0.5, 0.95, 0.02)[:, None, None]).long()
        packed = (bits << torch.arange(32, device=DEVICE)).sum(dim=2)
        data["allowed"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()
    return data


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


def _plain_embedding(s, case):
    ids, scale = s["ids"], s["scale"]
    given = (ids >= 0)[:, None]
    at = ids.clamp(min=0)
    out = {"y": torch.where(given, s["table"][at].float() * scale, 0.0).to(s["table"].dtype)}
    if case["train"]:
        grad = torch.zeros(s["table"].shape, dtype=torch.float32, device=ids.device)
        grad.index_add_(0, at, torch.where(given, s["grad"].float(), 0.0))
        out["grad"] = (grad * scale).to(s["table"].dtype)
    return out


def _plain_adjust(s, case):
    x, tokens = s["logits"].float(), s["tokens"]
    rows, vocab = x.shape
    given = tokens >= 0
    at = tokens.clamp(min=0)
    answer = given & (torch.arange(case["held"], device=x.device) >= s["prompt_lengths"][:, None])
    counts = torch.zeros((rows, vocab), dtype=torch.float32, device=x.device)
    seen = counts.scatter_add(1, at, given.float()) > 0
    counts.scatter_add_(1, at, answer.float())
    x = torch.where(seen, torch.where(x > 0, x / s["repetition"][:, None], x * s["repetition"][:, None]), x)
    x = x - s["frequency"][:, None] * counts - s["presence"][:, None] * (counts > 0)
    if s["bias_ids"] is not None:
        x.scatter_add_(1, s["bias_ids"], s["bias_values"])
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.reshape(rows, -1)[:, :vocab] == 1, x, NEG_INF)
    return {"logits": x.to(s["logits"].dtype)}


def _plain_orthogonal(matrix):
    a, b, c = COEFFICIENTS
    x = matrix.float()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.square().sum().sqrt() + EPS)
    for _ in range(STEPS):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.T if tall else x).to(matrix.dtype).contiguous()


def _own_embedding(s, case):
    from myflows_amd import embedding as ops
    out = {"y": ops.embedding_forward(s["table"], s["ids"], scale=s["scale"])}
    if case["train"]:
        out["grad"] = ops.embedding_backward(s["grad"], s["ids"], case["vocab"], scale=s["scale"])
    return out


def _own_adjust(s, case):
    from myflows_amd import logits as ops
    return {"logits": ops.adjust_logits(
        s["logits"], tokens=s["tokens"], prompt_lengths=s["prompt_lengths"], repetition=s["repetition"],
        presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
        allowed=s["allowed"])}


def run(state):
    case = state["case"]
    if case["kind"] == "embedding":
        return (_own_embedding if own else _plain_embedding)(state, case)
    if case["kind"] == "adjust":
        return (_own_adjust if own else _plain_adjust)(state, case)
    if own:
        from myflows_amd import orthogonal as ops
        return ops.orthogonalize_many(state["matrices"])
    return [_plain_orthogonal(matrix) for matrix in state["matrices"]]


def work(case):
    """Inputs and outputs once each. A lookup is one product an element, its gradient a sum; an adjustment a
    comparison an element. With the sides s <= l of a matrix, a step is a symmetric product over l, one over s
    and one of s x s with s x l, or, over all steps, the same polynomial formed from the s x s products alone
    but for two passes over the matrix's own sides: the lesser of the two is counted."""
    size = SIZES[case["type"]]
    if case["kind"] == "embedding":
        count = case["tokens"] * case["dim"]
        total = {"bytes": 8 * case["tokens"] + 2 * size * count, "flops": count}
        if case["train"]:
            total = {"bytes": total["bytes"] + size * (count + case["vocab"] * case["dim"]), "flops": 2 * count}
        return total
    if case["kind"] == "adjust":
        rows, vocab = case["rows"], case["vocab"]
        mask = 4 * -(-vocab // 32) if case["mask"] else 0
        return {"bytes": rows * (2 * size * vocab + mask + 8 * case["held"] + 12 * case["biases"] + 20),
                "flops": rows * vocab}
    total = {"bytes": 0, "flops": 0}
    for shape in _shapes(case):
        s, l = sorted(shape)
        total["bytes"] += 2 * size * s * l
        total["flops"] += min(STEPS * (3 * s * s * l + s ** 3), 6 * s * s * l + 14 * s ** 3)
    return total


def exact(case, seed):
    """The definitions in 64 bits."""
    data = _inputs(case, seed)
    return {"embedding": _exact_embedding, "adjust": _exact_adjust, "orthogonal": _exact_orthogonal}[case["kind"]](data, case)


def _exact_embedding(data, case):
    ids, scale = data["ids"], data["scale"]
    there = torch.nonzero(ids >= 0)[:, 0]
    y = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device=ids.device)
    y[there] = data["table"].index_select(0, ids[there]).double().mul_(scale)
    out = {"y": y}
    if case["train"]:
        # Rows in the order of their tokens; each token's sum is the product of its ones with its rows.
        order = there[torch.sort(ids[there], stable=True).indices]
        tokens, counts = torch.unique_consecutive(ids[order], return_counts=True)
        grad = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device=ids.device)
        if len(tokens):
            grad[tokens] = torch.segment_reduce(data["grad"][order].double().mul_(scale), "sum", lengths=counts, axis=0)
        out["grad"] = grad
    return out


def _exact_adjust(data, case):
    rows, vocab = data["logits"].shape
    out = []
    for r in range(rows):
        z, tokens = data["logits"][r].double(), data["tokens"][r]
        answer = tokens[int(data["prompt_lengths"][r]):]
        counts = torch.bincount(answer[answer >= 0], minlength=vocab).double()
        before = torch.unique(tokens[tokens >= 0])
        factor = data["repetition"][r].double()
        z[before] = torch.maximum(z[before], z[before] * 0) / factor + torch.minimum(z[before], z[before] * 0) * factor
        z -= data["frequency"][r].double() * counts + data["presence"][r].double() * counts.clamp(max=1)
        if data["bias_ids"] is not None:
            z.index_put_((data["bias_ids"][r],), data["bias_values"][r].double(), accumulate=True)
        if data["allowed"] is not None:
            place = torch.arange(vocab, device=z.device)
            words = data["allowed"][r].long() & 0xFFFFFFFF
            z[(words[place // 32] >> (place % 32)) % 2 == 0] = NEG_INF
        out.append(z)
    return {"logits": torch.stack(out)}


def _exact_orthogonal(data, case):
    a, b, c = COEFFICIENTS
    out = []
    for matrix in data["matrices"]:
        x = matrix.double()
        x = x / (torch.linalg.matrix_norm(x) + EPS)
        for _ in range(STEPS):  # the shorter side's products, on the side that they belong to
            if x.shape[0] > x.shape[1]:
                gram = x.mT.contiguous() @ x
                x = torch.addmm(x, x, torch.addmm(gram, gram, gram, beta=b, alpha=c), beta=a)
            else:
                gram = x @ x.mT.contiguous()
                x = torch.addmm(x, torch.addmm(gram, gram, gram, beta=b, alpha=c), x, beta=a)
        out.append(x)
    return out
