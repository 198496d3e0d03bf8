"""The operators of a classifier's answers and of a student's training, as cases to time and compare.

Three operators: the log probabilities of given tokens (with the rows' entropy and their top
alternatives) and their gradient; the distillation loss of a student against a teacher's recorded top
logits and its gradient; group norm with an activation over channels-last activations and its
gradients.

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


def listed():
    return [
        # One decoding step of one stream: the answer's log probability and 20 alternatives; latency counts.
        {"name": "log_probs_one_row", "kind": "log_probs", "rows": 1, "vocab": 131072, "type": "bfloat16", "top": 20,
         "pad": 0, "train": False},
        # A batch of a 1000-class classifier's answers with the five best classes.
        {"name": "log_probs_classes", "kind": "log_probs", "rows": 256, "vocab": 1000, "type": "float32", "top": 5,
         "pad": 0, "train": False},
        # Scoring long inputs, a row for each position, over a large vocabulary: bandwidth counts.
        {"name": "log_probs_scoring", "kind": "log_probs", "rows": 2048, "vocab": 131072, "type": "bfloat16", "top": 20,
         "pad": 0, "train": False},
        # A teacher's top logits being recorded: 64 a row, rows that are slices of a padded product.
        {"name": "log_probs_record", "kind": "log_probs", "rows": 777, "vocab": 32771, "type": "float16", "top": 64,
         "pad": 61, "train": False},
        # A training pass on log probabilities and entropies, an odd vocabulary in float32.
        {"name": "log_probs_train", "kind": "log_probs", "rows": 1000, "vocab": 50021, "type": "float32", "top": 0,
         "pad": 0, "train": True},
        # A small student of a 1000-class teacher: the loss and the gradient of one batch.
        {"name": "distill_classes", "kind": "distill", "rows": 64, "vocab": 1000, "type": "float32", "top": 5,
         "temperature": 2.0, "weights": False},
        # Ragged teacher records over an odd vocabulary, with row weights and rows that do not count.
        {"name": "distill_ragged", "kind": "distill", "rows": 333, "vocab": 32771, "type": "float16", "top": 20,
         "temperature": 1.5, "weights": True},
        # A large student's training pass against 64 recorded logits a row.
        {"name": "distill_large", "kind": "distill", "rows": 2048, "vocab": 65536, "type": "bfloat16", "top": 64,
         "temperature": 2.0, "weights": True},
        # The last feature map of one image (4x5 positions, 512 channels): latency counts.
        {"name": "group_norm_one", "kind": "group_norm", "n": 1, "positions": 20, "channels": 512, "groups": 32,
         "type": "float32", "activation": "relu", "train": False},
        # Layer1 activations of a batch of 64 images (29x39 positions), forward and backward.
        {"name": "group_norm_batch", "kind": "group_norm", "n": 64, "positions": 1131, "channels": 64, "groups": 32,
         "type": "float32", "activation": "silu", "train": True},
        # Odd sizes: rows of channels off every vector width, 15 channels a group.
        {"name": "group_norm_odd", "kind": "group_norm", "n": 33, "positions": 405, "channels": 90, "groups": 6,
         "type": "float16", "activation": "silu", "train": True},
        # Long samples (128x128 positions) whose groups no single workgroup holds: bandwidth counts.
        {"name": "group_norm_long", "kind": "group_norm", "n": 16, "positions": 16384, "channels": 256, "groups": 32,
         "type": "bfloat16", "activation": "silu", "train": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["log_probs", "distill", "group_norm"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "group_norm":
        groups, per = rng.choice([1, 2, 3, 4, 6, 8, 16, 32]), _spread(rng, 2, 64)
        channels = groups * per
        positions = _spread(rng, 8, 16384)
        most = max(1, min(64, 2 ** 25 // (channels * positions)))
        train = rng.random() < 0.7
        # A rounding that takes a ReLU to its other side changes a gradient wholly: forward passes only.
        return {"kind": kind, "n": _spread(rng, 1, most), "positions": positions, "channels": channels,
                "groups": groups, "type": dtype, "activation": "silu" if train else rng.choice(["none", "relu", "silu"]),
                "train": train}
    vocab = _spread(rng, 100, 131072)
    rows = _spread(rng, 1, max(1, min(4096, 2 ** 26 // vocab)))
    if kind == "log_probs":
        train = rng.random() < 0.4
        return {"kind": kind, "rows": rows, "vocab": vocab, "type": dtype, "top": 0 if train else rng.randint(0, 64),
                "pad": rng.choice([0, 0, rng.randint(1, 63)]), "train": train}
    return {"kind": kind, "rows": rows, "vocab": vocab, "type": dtype, "top": rng.randint(1, 64),
            "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]), "weights": rng.random() < 0.5}


def _logits(g, case, pad=0):
    """Logits of a trained network: normal, with one clear winner in most rows."""
    rows, vocab = case["rows"], case["vocab"]
    z = torch.randn((rows, vocab + pad), generator=g, device=DEVICE) * 2.0
    winner = torch.randint(0, vocab, (rows, 1), generator=g, device=DEVICE)
    lift = torch.rand((rows, 1), generator=g, device=DEVICE) * 14.0
    z.scatter_add_(1, winner, lift)
    return z, winner[:, 0]


def _inputs(case, seed):
    """The data of a case, made from the seed alone."""
    g, dtype = torch.Generator(device=DEVICE).manual_seed(seed), TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device=DEVICE)  # noqa: E731
    if case["kind"] == "group_norm":
        n, positions, c = case["n"], case["positions"], case["channels"]
        # Channels of unlike scales and offsets, as a product's outputs are.
        x = normal(n, positions, c) * (0.5 + uniform(c)) + normal(c)
        return {"x": x.to(dtype), "dy": normal(n, positions, c).to(dtype) if case["train"] else None,
                "gamma": 1.0 + 0.2 * normal(c), "beta": 0.1 * normal(c)}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    if case["kind"] == "log_probs":
        z, winner = _logits(g, case, case["pad"])
        if rows > 1 and not case["train"]:  # constrained decoding: in one row of eight most tokens are ruled out
            ruled = (uniform(rows, 1) < 0.125) & (uniform(rows, vocab + case["pad"]) < 0.9)
            z.masked_fill_(ruled, NEG_INF)
        z = z.to(dtype)
        tokens = torch.where(uniform(rows) < 0.5, winner, torch.randint(0, vocab, (rows,), generator=g, device=DEVICE))
        if rows > 1:  # positions without a token
            tokens = torch.where(uniform(rows) < 0.1, torch.full_like(tokens, -1), tokens)
        data = {"logits": z[:, :vocab], "tokens": tokens}
        if case["train"]:
            data.update(log_prob_grad=normal(rows), entropy_grad=0.1 * normal(rows))
        return data
    z, _ = _logits(g, case)
    # Distinct ids in no order, logits falling from the first on, records of unlike lengths, some empty.
    ids = torch.randint(0, vocab - top + 1, (rows, top), generator=g, device=DEVICE).sort(dim=1).values
    ids = (ids + torch.arange(top, device=DEVICE)).gather(1, uniform(rows, top).argsort(dim=1))
    teacher = 12.0 + normal(rows, 1) - torch.cumsum(uniform(rows, top) * (8.0 / top) + 0.05, dim=1)
    z.scatter_add_(1, ids, 0.6 * teacher + normal(rows, top))
    held = torch.where(uniform(rows) < 0.5, top, torch.randint(1, top + 1, (rows,), generator=g, device=DEVICE))
    if rows > 1:  # the first row counts, whatever the others do
        held = torch.where((uniform(rows) < 0.05) & (torch.arange(rows, device=DEVICE) > 0), torch.zeros_like(held), held)
    ids = torch.where(torch.arange(top, device=DEVICE) < held[:, None], ids, torch.full_like(ids, -1))
    weights = None
    if case["weights"]:
        weights = 0.5 + uniform(rows)
        if rows > 1:
            weights = torch.where((uniform(rows) < 0.1) & (torch.arange(rows, device=DEVICE) > 0),
                                  torch.zeros_like(weights), weights)
    # The loss scale of half-precision training where the gradients are held in float16.
    scale = 4096.0 if dtype is torch.float16 else 1.0
    return {"logits": z.to(dtype), "ids": ids, "teacher": teacher, "weights": weights,
            "seed": torch.full((), scale, device=DEVICE)}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


def _plain_log_probs(s, case):
    x, tokens, top = s["logits"].float(), s["tokens"], case["top"]
    rows, vocab = x.shape
    most = x.max(dim=1, keepdim=True).values
    shift = torch.where(most == NEG_INF, torch.zeros_like(most), most)
    e = torch.exp(x - shift)
    total = e.sum(dim=1, keepdim=True)
    log_sum = shift + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * (x - shift), torch.zeros_like(e)).sum(dim=1, keepdim=True) / total
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    log_prob = torch.where(given, (x.gather(1, at) - log_sum)[:, 0], torch.zeros_like(log_sum[:, 0]))
    out = {"log_prob": log_prob, "entropy": entropy[:, 0], "log_sum": log_sum[:, 0]}
    if top:
        # The order of (logit, then the lower index) as that of whole numbers.
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        place = torch.arange(vocab, device=x.device)
        key = torch.topk(bits * 2 ** 32 + (2 ** 32 - 1 - place), top, dim=1).values
        ids = 2 ** 32 - 1 - (key & (2 ** 32 - 1))
        out.update(top_log_probs=x.gather(1, ids) - log_sum, top_ids=ids.int())
    if case["train"]:
        p = e / total
        log_p = torch.where(p > 0, x - log_sum, torch.zeros_like(x))
        g = torch.where(given, s["log_prob_grad"], torch.zeros_like(log_prob))[:, None]
        grad = -g * p - s["entropy_grad"][:, None] * p * (log_p + entropy)
        grad.scatter_add_(1, at, g)
        out["grad"] = grad.to(s["logits"].dtype)
    return out


def _plain_distill(s, case):
    t = case["temperature"]
    x = s["logits"].float() / t
    valid = s["ids"] >= 0
    at = s["ids"].clamp(min=0)
    teacher = torch.where(valid, s["teacher"] / t, torch.full_like(s["teacher"], NEG_INF))
    counts = valid.any(dim=1, keepdim=True)
    most = torch.where(counts, teacher.max(dim=1, keepdim=True).values, torch.zeros_like(teacher[:, :1]))
    u = torch.exp(teacher - most)
    total = torch.where(counts, u.sum(dim=1, keepdim=True), torch.ones_like(most))
    p = u / total
    log_p = torch.where(valid, teacher - most - torch.log(total), torch.zeros_like(teacher))
    shift = x.max(dim=1, keepdim=True).values
    e = torch.exp(x - shift)
    sums = e.sum(dim=1, keepdim=True)
    log_q = x.gather(1, at) - shift - torch.log(sums)
    weight = counts[:, 0].float() if s["weights"] is None else torch.where(counts[:, 0], s["weights"], torch.zeros_like(
        s["weights"]))
    row_loss = torch.where(weight > 0, t * t * (p * (log_p - log_q)).sum(dim=1), torch.zeros_like(weight))
    whole = weight.sum()
    loss = (weight * row_loss).sum() / whole
    scale = (s["seed"] * weight / whole * t)[:, None]
    grad = scale * (e / sums)
    grad.scatter_add_(1, at, -scale * p)
    return {"loss": loss, "row_loss": row_loss, "grad": grad.to(s["logits"].dtype)}


def _plain_group_norm(s, case):
    n, positions, c = s["x"].shape
    groups, act = case["groups"], case["activation"]
    x = s["x"].float().reshape(n, positions, groups, c // groups)
    gamma, beta = (s[k].reshape(groups, c // groups) for k in ("gamma", "beta"))
    mean = x.mean(dim=(1, 3), keepdim=True)
    inv_std = torch.rsqrt((x - mean).square().mean(dim=(1, 3), keepdim=True) + 1e-5)
    hat = (x - mean) * inv_std
    u = hat * gamma + beta
    gate = 1.0 / (1.0 + torch.exp(-u)) if act == "silu" else None
    y = u * gate if act == "silu" else u.clamp(min=0) if act == "relu" else u
    out = {"y": y.reshape(n, positions, c).to(s["x"].dtype), "mean": mean.reshape(n, groups),
           "inv_std": inv_std.reshape(n, groups)}
    if case["train"]:
        du = s["dy"].float().reshape(x.shape)
        if act == "silu":
            du = du * gate * (1.0 + u * (1.0 - gate))
        elif act == "relu":
            du = torch.where(u > 0, du, torch.zeros_like(du))
        dhat = du * gamma
        dx = inv_std * (dhat - dhat.mean(dim=(1, 3), keepdim=True) - hat * (dhat * hat).mean(dim=(1, 3), keepdim=True))
        out.update(dx=dx.reshape(n, positions, c).to(s["x"].dtype), dgamma=(du * hat).sum(dim=(0, 1)).reshape(c),
                   dbeta=du.sum(dim=(0, 1)).reshape(c))
    return out


def _own_log_probs(s, case):
    from myflows_amd import logits as ops
    r = ops.log_probs_forward(s["logits"], s["tokens"], top=case["top"])
    out = {"log_prob": r.log_prob, "entropy": r.entropy, "log_sum": r.log_sum}
    if case["top"]:
        out.update(top_log_probs=r.top_log_probs, top_ids=r.top_ids)
    if case["train"]:
        out["grad"] = ops.log_probs_backward(s["logits"], s["tokens"], r, log_prob_grad=s["log_prob_grad"],
                                             entropy_grad=s["entropy_grad"])
    return out


def _own_distill(s, case):
    from myflows_amd import logits as ops
    r = ops.distill_loss_forward(s["logits"], s["ids"], s["teacher"], temperature=case["temperature"],
                                 row_weights=s["weights"])
    grad = ops.distill_loss_backward(s["logits"], s["ids"], r, s["seed"], temperature=case["temperature"])
    return {"loss": r.loss, "row_loss": r.row_loss, "grad": grad}


def _own_group_norm(s, case):
    from myflows_amd import group_norm as ops
    act = None if case["activation"] == "none" else case["activation"]
    y, mean, inv_std = ops.group_norm_forward(s["x"], s["gamma"], s["beta"], case["groups"], eps=1e-5, activation=act)
    out = {"y": y, "mean": mean, "inv_std": inv_std}
    if case["train"]:
        dx, dgamma, dbeta = torch.empty_like(s["x"]), torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
        ops.group_norm_backward(s["x"], s["dy"], s["gamma"], s["beta"], mean, inv_std, activation=act, x_grad=dx,
                                gamma_grad=dgamma, beta_grad=dbeta, accumulate=(False, False, False))
        out.update(dx=dx, dgamma=dgamma, dbeta=dbeta)
    return out


def run(state):
    case = state["case"]
    forms = {"log_probs": (_plain_log_probs, _own_log_probs), "distill": (_plain_distill, _own_distill),
             "group_norm": (_plain_group_norm, _own_group_norm)}
    return forms[case["kind"]][1 if own else 0](state, case)


def work(case):
    """Inputs and outputs once each; for an element of the logits a comparison, a difference, an exp and
    two sums forward and five operations more backward; for an activation about eight forward (its two
    sums, the affine form, the activation) and sixteen more backward."""
    size = SIZES[case["type"]]
    if case["kind"] == "group_norm":
        count = case["n"] * case["positions"] * case["channels"]
        small = 4 * (2 * case["channels"] + 2 * case["n"] * case["groups"])
        if case["train"]:
            return {"bytes": 4 * size * count + small + 8 * case["channels"], "flops": 24 * count}
        return {"bytes": 2 * size * count + small, "flops": 8 * count}
    rows, count, top = case["rows"], case["rows"] * case["vocab"], case["top"]
    if case["kind"] == "log_probs":
        train = case["train"]
        return {"bytes": (2 if train else 1) * size * count + rows * (20 + 8 * top + (8 if train else 0)),
                "flops": (10 if train else 5) * count}
    return {"bytes": 2 * size * count + rows * (12 * top + 4 + (4 if case["weights"] else 0)), "flops": 9 * count}


def exact(case, seed):
    """The definitions in 64 bits, a few rows (or one sample) at a time."""
    data = _inputs(case, seed)
    if case["kind"] == "group_norm":
        return _exact_group_norm(data, case)
    rows = max(1, 2 ** 25 // case["vocab"])
    parts = [(_exact_log_probs if case["kind"] == "log_probs" else _exact_distill)(
        {k: v[i:i + rows] if isinstance(v, torch.Tensor) and v.ndim else v for k, v in data.items()}, case)
        for i in range(0, case["rows"], rows)]
    out = {k: torch.cat([part[k] for part in parts]) for k in parts[0]}
    if case["kind"] == "distill":
        weight, grad = out.pop("weight"), out["grad"]
        out = {"loss": (weight * out["row_loss"]).sum() / weight.sum(), "row_loss": out["row_loss"],
               "grad": grad.mul_((data["seed"].double() * weight / weight.sum())[:, None])}
    return out


def _exact_log_softmax(z):
    """log softmax of each row in 64 bits; -inf where the logit is."""
    z = z.double()
    z = z - z.amax(dim=1, keepdim=True)
    return z - z.exp().sum(dim=1, keepdim=True).log()


def _exact_log_probs(data, case):
    z = data["logits"].double()
    log_p = _exact_log_softmax(z)
    p = log_p.exp()
    plogp = torch.nan_to_num(log_p, neginf=0.0).mul_(p)
    entropy = -plogp.sum(dim=1)
    r = torch.arange(z.shape[0], device=z.device)
    tokens, given = data["tokens"], data["tokens"] >= 0
    out = {"log_prob": torch.where(given, log_p[r, tokens * given], 0.0), "entropy": entropy,
           "log_sum": torch.logsumexp(z, dim=1)}
    if case["top"]:
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out.update(top_log_probs=log_p.gather(1, order), top_ids=order.int())
    if case["train"]:
        g = data["log_prob_grad"].double() * given
        grad = -g[:, None] * p - data["entropy_grad"].double()[:, None] * (plogp + p * entropy[:, None])
        grad[r, tokens * given] += g
        out["grad"] = grad
    return out


def _exact_distill(data, case):
    t, ids = case["temperature"], data["ids"]
    log_q = _exact_log_softmax(data["logits"].double() / t)
    held = ids >= 0
    u = torch.where(held, (data["teacher"].double() / t).exp(), 0.0)  # logits near 12: no overflow
    p = u / u.sum(dim=1, keepdim=True).clamp(min=1e-300)
    counts = held.any(dim=1).double()
    weight = counts if data["weights"] is None else counts * data["weights"].double()
    at = ids * held
    terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - log_q.gather(1, at)), 0.0)
    grad = log_q.exp_()
    r = torch.arange(ids.shape[0], device=ids.device)
    for k in range(ids.shape[1]):
        grad[r, at[:, k]] -= p[:, k]
    return {"row_loss": torch.where(weight > 0, t * t * terms.sum(dim=1), 0.0), "weight": weight, "grad": grad.mul_(t)}


def _exact_group_norm(data, case):
    n, groups, c = case["n"], case["groups"], case["channels"]
    gamma, beta = data["gamma"].double(), data["beta"].double()
    out = {k: [] for k in ("y", "mean", "inv_std") + (("dx", "dgamma", "dbeta") if case["train"] else ())}
    for i in range(n):
        x = data["x"][i].double()
        grouped = x.reshape(-1, groups, c // groups)
        var, mean = torch.var_mean(grouped, dim=(0, 2), correction=0)
        inv_std = (var + 1e-5) ** -0.5
        spread = lambda v: v.repeat_interleave(c // groups)  # noqa: E731
        hat = (x - spread(mean)) * spread(inv_std)
        u = hat * gamma + beta
        sig = torch.sigmoid(u)
        out["y"].append({"silu": u * sig, "relu": u.relu(), "none": u}[case["activation"]])
        out["mean"].append(mean)
        out["inv_std"].append(inv_std)
        if case["train"]:
            du = data["dy"][i].double() * {"silu": sig + u * sig * (1 - sig), "relu": (u > 0).double(),
                                           "none": torch.ones_like(u)}[case["activation"]]
            d = du * gamma
            means = [spread(v.reshape(-1, groups, c // groups).mean(dim=(0, 2))) for v in (d, d * hat)]
            out["dx"].append(spread(inv_std) * (d - means[0] - hat * means[1]))
            out["dgamma"].append((du * hat).sum(dim=0))
            out["dbeta"].append(du.sum(dim=0))
    result = {k: torch.stack(v) for k, v in out.items()}
    for k in ("dgamma", "dbeta"):
        if k in result:
            result[k] = result[k].sum(dim=0)
    return result
