"""What a classifier answers and how a student learns from a teacher's answers, on libmfhip.

* ``log_probs_forward`` / ``log_probs_backward``: the log probabilities of given tokens, each row's
  entropy and its top alternatives, and the gradient of the log probabilities and entropies;
* ``adjust_logits``: penalties for tokens given before, biases and a grammar's mask, ahead of an answer;
* ``distill_loss_forward`` / ``distill_loss_backward``: the loss of a student against a teacher's
  recorded top logits (``log_probs_forward`` with ``top`` makes such a record), and its gradient;
* ``CrossEntropyLoss`` and ``DistillationLoss``: both as losses of a ``Graph``.

Logits are 2-D GPU tensors of float32, bfloat16 or float16 whose rows are contiguous; the rows may lie
apart (a slice of a padded product is read in place). Everything else is float32, tokens and ids are
int32 or int64, and a negative token or id is none; they are read in place too, at their own strides. All
arithmetic is float32, and a gradient is rounded once to the logits' type. There is no host path. The
reference has no counterpart: its only loss is the mean squared error.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import native
from .graph import GradientOp
from .memory import share_memory

_TYPE_CODES = native.TYPE_CODES
_WHOLE = {torch.int32: 0, torch.int64: 1}  # whether whole numbers are int64
TOP_MAX = 64            # alternatives of a row
DISTILL_HELD_MAX = 256  # teacher ids of a row
ROWS_LIMIT = 1 << 22
VOCAB_LIMIT = 1 << 24
HELD_LIMIT = (1 << 20) - 1  # tokens of a row's history
BIAS_MAX = 1024            # biases of a row


class LogProbs:
    """What ``log_probs_forward`` returns, and ``log_probs_backward`` takes back.

    log_prob (rows,), None without tokens; entropy (rows,); log_sum (rows,), ln sum e^z; top_log_probs
    (rows, top) and top_ids (rows, top) int32, None for top 0; stats (2, rows), the largest logit m and
    sum e^(z - m). Iterates over them in this order."""

    __slots__ = ("_floats", "_given", "top_log_probs", "top_ids")

    def __init__(self, floats, given, top_log_probs, top_ids):
        self._floats, self._given = floats, given  # (5, rows): stats, entropy, log_sum, log_prob
        self.top_log_probs, self.top_ids = top_log_probs, top_ids

    @property
    def log_prob(self):
        return self._floats[4] if self._given else None

    @property
    def entropy(self):
        return self._floats[2]

    @property
    def log_sum(self):
        return self._floats[3]

    @property
    def stats(self):
        return self._floats[:2]

    def __iter__(self):
        return iter((self.log_prob, self.entropy, self.log_sum, self.top_log_probs, self.top_ids, self.stats))


class DistillLoss:
    """What ``distill_loss_forward`` returns, and ``distill_loss_backward`` takes back.

    loss (), the weighted mean of row_loss over the rows that count; row_loss (rows,); weights (rows,), those
    that count; stats (2, rows), the largest logit m and sum e^((z - m) / temperature); targets (rows, held),
    the teacher's probability of each id; scale (2,), the loss and 1 / sum of the weights."""

    __slots__ = ("_floats", "_rows", "_held")

    def __init__(self, floats, rows, held):
        self._floats, self._rows, self._held = floats, rows, held  # scale, row_loss, weights, stats, targets

    def _part(self, first, count):
        return self._floats[first:first + count]

    @property
    def loss(self):
        return self._floats[0]

    @property
    def scale(self):
        return self._part(0, 2)

    @property
    def row_loss(self):
        return self._part(2, self._rows)

    @property
    def weights(self):
        return self._part(2 + self._rows, self._rows)

    @property
    def stats(self):
        return self._part(2 + 2 * self._rows, 2 * self._rows).view(2, self._rows)

    @property
    def targets(self):
        return self._part(2 + 4 * self._rows, self._rows * self._held).view(self._rows, self._held)


def _logits(value):
    """(tensor, type code, rows, vocab, row stride) of a 2-D tensor of logits."""
    code = _TYPE_CODES.get(value.dtype) if isinstance(value, torch.Tensor) and value.is_cuda else None
    if code is None:
        raise TypeError("logits must be a float32, bfloat16 or float16 torch tensor on the GPU")
    if value.ndim != 2:
        raise ValueError("logits must be 2-D (rows, vocabulary)")
    rows, vocab = value.shape
    if not 0 < vocab <= VOCAB_LIMIT or rows > ROWS_LIMIT:
        raise ValueError(f"logits take at most {ROWS_LIMIT} rows of 1 to {VOCAB_LIMIT} elements")
    row_stride, stride = value.stride()
    if (vocab > 1 and stride != 1) or (rows > 1 and row_stride < vocab):
        value = value.contiguous()
        row_stride = vocab
    return value, code, rows, vocab, row_stride if rows > 1 else vocab


def _whole(value, shape, name):
    """(tensor, whether it is int64, row stride) of GPU whole numbers of a shape, read in place: one a row at any
    stride, or rows side by side at any row stride (others are copied)."""
    wide = _WHOLE.get(value.dtype) if isinstance(value, torch.Tensor) and value.is_cuda else None
    if wide is None:
        raise TypeError(f"{name} must be an int32 or int64 torch tensor on the GPU")
    if value.shape != shape:
        raise ValueError(f"{name} must have shape {shape}")
    strides = value.stride()
    if strides[-1] != 1 and len(shape) == 2 and shape[1] > 1:
        return value.contiguous(), wide, shape[1]
    return value, wide, strides[0]


def _row_floats(value, rows, name):
    """(tensor, stride) of one float32 a row; any stride, 0 (a broadcast scalar) included."""
    if not (isinstance(value, torch.Tensor) and value.is_cuda and value.dtype is torch.float32):
        raise TypeError(f"{name} must be a float32 torch tensor on the GPU")
    if value.shape != (rows,):
        raise ValueError(f"{name} must have shape {(rows,)}")
    return value, value.stride(0)


def _gradient(out, add, like):
    """(tensor, row stride) that a gradient of the logits goes to."""
    if out is None:
        if add:
            raise ValueError("add needs an out tensor")
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
        return out, out.shape[1]
    if not (isinstance(out, torch.Tensor) and out.is_cuda and out.dtype is like.dtype and out.shape == like.shape
            and (out.shape[1] <= 1 or out.stride(1) == 1) and (out.shape[0] <= 1 or out.stride(0) >= out.shape[1])):
        raise ValueError("out must be a GPU tensor of the logits' type and shape with contiguous rows")
    return out, out.stride(0) if out.shape[0] > 1 else out.shape[1]


@lru_cache(maxsize=256)
def _log_probs_workspace(rows, vocab, code, top):
    return native.workspace_bytes("mfh_log_probs_workspace", rows, vocab, code, top)


@lru_cache(maxsize=256)
def _distill_workspace(rows, vocab, code):
    return native.workspace_bytes("mfh_distill_workspace", rows, vocab, code)


def log_probs_forward(logits, tokens=None, *, top=0):
    """``LogProbs`` of each row z of the logits: log_prob = z[token] - ln sum e^z (0 where the token is
    negative, NaN where it lies beyond the vocabulary), the entropy, ln sum e^z, and the ``top`` most likely
    ids with their log probabilities, equal logits in rising order of their ids.

    A logit of -inf (a ruled-out token) has probability 0. A row of nothing else has log probabilities
    -inf and entropy 0; a NaN or +inf makes its row's values NaN, and a NaN is no alternative (an id that
    is then missing is -1)."""
    logits, code, rows, vocab, stride = _logits(logits)
    top = int(top)
    if not 0 <= top <= min(TOP_MAX, vocab):
        raise ValueError(f"top must lie between 0 and {min(TOP_MAX, vocab)} (at most {TOP_MAX} and the vocabulary)")
    wide = tokens_stride = 0
    if tokens is not None:
        tokens, wide, tokens_stride = _whole(tokens, (rows,), "tokens")
    floats = logits.new_empty((5, rows), dtype=torch.float32)
    top_log_probs = logits.new_empty((rows, top), dtype=torch.float32) if top else None
    top_ids = logits.new_empty((rows, top), dtype=torch.int32) if top else None
    workspace, held = native.byte_workspace(_log_probs_workspace(rows, vocab, code, top))
    stats, row = floats.data_ptr(), 4 * rows
    native._call("mfh_log_probs", logits.data_ptr(), code, rows, vocab, stride, native._addr(tokens), wide,
                 tokens_stride, 0 if tokens is None else stats + 4 * row, stats + 2 * row, stats + 3 * row, stats, top,
                 native._addr(top_log_probs), native._addr(top_ids), workspace, held,
                 native.stream_counters() if held else 0, native._stream())
    return LogProbs(floats, tokens is not None, top_log_probs, top_ids)


def _log_probs_gradient(logits, tokens, saved, log_prob_grad, entropy_grad, factor, scale, out, add):
    logits, code, rows, vocab, stride = _logits(logits)
    if not isinstance(saved, LogProbs) or saved._floats.shape[1] != rows:
        raise ValueError("saved must be the LogProbs of these logits")
    wide = tokens_stride = lp_step = entropy_step = 0
    if log_prob_grad is not None:
        if tokens is None:
            raise ValueError("a gradient of the log probabilities needs their tokens")
        tokens, wide, tokens_stride = _whole(tokens, (rows,), "tokens")
        log_prob_grad, lp_step = _row_floats(log_prob_grad, rows, "log_prob_grad")
    if entropy_grad is not None:
        entropy_grad, entropy_step = _row_floats(entropy_grad, rows, "entropy_grad")
    out, out_stride = _gradient(out, add, logits)
    stats = saved._floats.data_ptr()
    native._call("mfh_log_probs_backward", logits.data_ptr(), code, rows, vocab, stride,
                 0 if log_prob_grad is None else tokens.data_ptr(), wide, tokens_stride, stats, stats + 8 * rows,
                 native._addr(log_prob_grad), lp_step, native._addr(entropy_grad), entropy_step,
                 native._addr(factor), scale, out.data_ptr(), out_stride, int(add), native._stream())
    return out


def log_probs_backward(logits, tokens, saved, *, log_prob_grad=None, entropy_grad=None, out=None, add=False):
    """The gradient of sum(log_prob_grad * log_prob) + sum(entropy_grad * entropy) by the logits, written to
    (or, with add, added to) out. ``saved`` is the LogProbs of the same logits; the gradients (rows,) may have
    any stride (an expanded scalar). A row whose gradients are 0 gets 0, whatever its logits hold and its token is; a
    token beyond the vocabulary makes its row NaN where its log_prob_grad is not 0."""
    return _log_probs_gradient(logits, tokens, saved, log_prob_grad, entropy_grad, None, 1.0, out, add)


def _penalty(value, rows, name, positive=False):
    """(tensor or None, stride, value for all rows) of a penalty: a number, or one float32 a row."""
    if isinstance(value, torch.Tensor):
        return *_row_floats(value, rows, name), 0.0
    value = native._float32(value)
    if not math.isfinite(value) or (positive and value <= 0.0):
        raise ValueError(f"{name} must be finite{' and positive' if positive else ''} in float32")
    return None, 0, value


def _rows_of(value, rows, name):
    """A 2-D view of a tensor with a row for each of `rows`; a 1-D one is every row's."""
    if isinstance(value, torch.Tensor) and value.ndim == 1:
        value = value.expand(rows, -1)
    if not isinstance(value, torch.Tensor) or value.ndim != 2 or value.shape[0] != rows:
        raise ValueError(f"{name} must be a (rows, n) tensor, or an (n,) one for all rows")
    return value


def adjust_logits(logits, *, tokens=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                  bias_ids=None, bias_values=None, allowed=None, out=None):
    """The logits as an answer is drawn from them, of their type; out may be the logits themselves, and shares no
    memory with anything else that the call reads.

    ``tokens`` (rows, held) are a row's history: its prompt, the first ``prompt_lengths[row]`` of them (none
    without), and its answer so far. A logit z of a token in the history becomes z / repetition where z > 0 and
    z * repetition else; one that is n > 0 times in the answer then loses frequency * n and presence. Each
    penalty is a number or one float32 a row. ``bias_values`` are added at ``bias_ids``, equal ids' values in
    their order. Where ``allowed`` (int32 words; bit v % 32 of word v // 32 is token v's) has no bit, the logit
    is -inf. Biases and masks are (rows, n), or (n,) for all rows. A negative token or id is none, one beyond the
    vocabulary counts nowhere. Computed in float32 and rounded once."""
    logits, code, rows, vocab, stride = _logits(logits)
    wide = tokens_stride = held = 0
    if tokens is not None:
        if not isinstance(tokens, torch.Tensor) or tokens.ndim != 2 or tokens.shape[1] > HELD_LIMIT:
            raise ValueError(f"tokens must be a (rows, held) tensor with at most {HELD_LIMIT} a row")
        held = tokens.shape[1]
        tokens, wide, tokens_stride = _whole(tokens, (rows, held), "tokens")
    prompt_wide = prompt_stride = 0
    if prompt_lengths is not None:
        if tokens is None:
            raise ValueError("prompt_lengths need their tokens")
        prompt_lengths, prompt_wide, prompt_stride = _whole(prompt_lengths, (rows,), "prompt_lengths")
    repetition, repetition_stride, repetition_all = _penalty(repetition, rows, "repetition", positive=True)
    presence, presence_stride, presence_all = _penalty(presence, rows, "presence")
    frequency, frequency_stride, frequency_all = _penalty(frequency, rows, "frequency")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    bias_wide = bias_ids_stride = bias_values_stride = biases = 0
    if bias_ids is not None:
        bias_ids, bias_values = _rows_of(bias_ids, rows, "bias_ids"), _rows_of(bias_values, rows, "bias_values")
        biases = bias_ids.shape[1]
        if biases > BIAS_MAX:
            raise ValueError(f"a row takes at most {BIAS_MAX} biases")
        bias_ids, bias_wide, bias_ids_stride = _whole(bias_ids, (rows, biases), "bias_ids")
        if not (bias_values.is_cuda and bias_values.dtype is torch.float32):
            raise TypeError("bias_values must be a float32 torch tensor on the GPU")
        if bias_values.shape != bias_ids.shape:
            raise ValueError("bias_values must have the shape of bias_ids")
        if bias_values.stride(1) != 1 and biases > 1:
            bias_values = bias_values.contiguous()
        bias_values_stride = bias_values.stride(0)
    allowed_stride = 0
    if allowed is not None:
        allowed = _rows_of(allowed, rows, "allowed")
        if not (allowed.is_cuda and allowed.dtype is torch.int32):
            raise TypeError("allowed must be an int32 torch tensor on the GPU")
        if allowed.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"allowed must have {(vocab + 31) // 32} words a row")
        if allowed.stride(1) != 1 and allowed.shape[1] > 1:
            allowed = allowed.contiguous()
        allowed_stride = allowed.stride(0)
    given = out is not None
    out, out_stride = _gradient(out, False, logits)
    read = (tokens, prompt_lengths, repetition, presence, frequency, bias_ids, bias_values, allowed)
    native._on_current_device(logits, out, *read)
    if given:
        if (out.data_ptr() != logits.data_ptr() or out_stride != stride) and share_memory(out, logits):
            raise ValueError("out must be the logits themselves or share no memory with them")
        if any(value is not None and share_memory(out, value) for value in read):
            raise ValueError("out must share no memory with what the logits are adjusted by")
    native._call("mfh_adjust_logits", logits.data_ptr(), code, rows, vocab, stride, native._addr(tokens), wide,
                 tokens_stride, held, native._addr(prompt_lengths), prompt_wide, prompt_stride, native._addr(repetition),
                 repetition_stride, repetition_all, native._addr(presence), presence_stride, presence_all,
                 native._addr(frequency), frequency_stride, frequency_all, native._addr(bias_ids), bias_wide,
                 bias_ids_stride, native._addr(bias_values), bias_values_stride, biases, native._addr(allowed),
                 allowed_stride, out.data_ptr(), out_stride, native._stream())
    return out


def _temperature(value):
    value = float(value)
    if not 2.0 ** -63 <= value <= 2.0 ** 63:  # its square and the square's inverse are normal floats
        raise ValueError("the temperature must lie between 2^-63 and 2^63")
    return value


def distill_loss_forward(logits, teacher_ids, teacher_logits, *, temperature=1.0, row_weights=None):
    """``DistillLoss`` of a student's logits against a teacher's record: ids (rows, held) and float32 logits
    (rows, held; log probabilities serve as well, a row's constant does not matter). With the teacher's
    p = softmax(teacher_logits / T) over the ids that are held and the student's q = softmax(logits / T),
    row_loss = T^2 sum p (ln p - ln q[id]) and loss is its mean by row_weights (1 each without them).

    A row without an id, with teacher logits of -inf alone or with weight 0 does not count: its loss and
    gradient are 0, whatever its logits hold, and without any row that counts the loss is 0. An id beyond the
    vocabulary makes a counting row NaN. The temperature lies between 2^-63 and 2^63."""
    logits, code, rows, vocab, stride = _logits(logits)
    temperature = _temperature(temperature)
    if not isinstance(teacher_ids, torch.Tensor) or teacher_ids.ndim != 2 or not 0 < teacher_ids.shape[1] <= DISTILL_HELD_MAX:
        raise ValueError(f"teacher_ids must be a (rows, held) tensor with held between 1 and {DISTILL_HELD_MAX}")
    shape = (rows, teacher_ids.shape[1])
    teacher_ids, wide, ids_stride = _whole(teacher_ids, shape, "teacher_ids")
    if not (isinstance(teacher_logits, torch.Tensor) and teacher_logits.is_cuda and teacher_logits.dtype is torch.float32):
        raise TypeError("teacher_logits must be a float32 torch tensor on the GPU")
    if teacher_logits.shape != shape:
        raise ValueError(f"teacher_logits must have shape {shape}")
    teacher_stride, stride_within = teacher_logits.stride()
    if stride_within != 1 and shape[1] > 1:
        teacher_logits, teacher_stride = teacher_logits.contiguous(), shape[1]
    weights_stride = 0
    if row_weights is not None:
        row_weights, weights_stride = _row_floats(row_weights, rows, "row_weights")
    floats = logits.new_empty((2 + rows * (4 + shape[1]),), dtype=torch.float32)
    workspace, held = native.byte_workspace(_distill_workspace(rows, vocab, code))
    scale, row = floats.data_ptr(), 4 * rows
    row_loss = scale + 8
    native._call("mfh_distill_loss", logits.data_ptr(), code, rows, vocab, stride, teacher_ids.data_ptr(), wide,
                 ids_stride, teacher_logits.data_ptr(), teacher_stride, shape[1], native._addr(row_weights),
                 weights_stride, temperature, row_loss, row_loss + row, row_loss + 2 * row, row_loss + 4 * row, scale,
                 workspace, held, native.stream_counters(), native._stream())
    return DistillLoss(floats, rows, shape[1])


def distill_loss_backward(logits, teacher_ids, saved, seed, *, temperature=1.0, out=None, add=False):
    """seed times the gradient of the loss by the logits, written to (or, with add, added to) out. ``saved`` is
    the DistillLoss of the same arguments and seed one float on the GPU."""
    logits, code, rows, vocab, stride = _logits(logits)
    temperature = _temperature(temperature)
    if not isinstance(saved, DistillLoss) or saved._rows != rows:
        raise ValueError("saved must be the DistillLoss of these logits")
    teacher_ids, wide, ids_stride = _whole(teacher_ids, (rows, saved._held), "teacher_ids")
    seed = native._device_f32(seed, "seed")
    if seed.numel() != 1:
        raise ValueError("seed must hold one value")
    out, out_stride = _gradient(out, add, logits)
    scale, row = saved._floats.data_ptr(), 4 * rows
    row_loss = scale + 8
    native._call("mfh_distill_loss_backward", logits.data_ptr(), code, rows, vocab, stride, teacher_ids.data_ptr(), wide,
                 ids_stride, saved._held, row_loss + 4 * row, row_loss + 2 * row, row_loss + row, scale, seed.data_ptr(), temperature,
                 out.data_ptr(), out_stride, int(add), native._stream())
    return out


def _on_gpu(value, op):
    if not (isinstance(value, torch.Tensor) and value.is_cuda):
        raise ValueError(f"{op} runs on libmfhip and needs a GPU tensor (device=cpu is not supported)")


class CrossEntropyLoss(GradientOp):
    """The mean of -log_prob of the labels (rows,) over the rows whose label is not negative (0 without
    any). A label beyond the vocabulary makes the loss NaN. ``log_probs`` holds the last forward's LogProbs,
    entropies included."""

    def __init__(self, logits, labels, name="CrossEntropyLoss"):
        super().__init__(logits, labels, name=name)
        self.log_probs = self._scale = None

    def forward(self, logits, labels):
        _on_gpu(logits, "CrossEntropyLoss")
        self.log_probs = log_probs_forward(logits, labels)
        labels, wide, stride = _whole(labels, (logits.shape[0],), "labels")
        self._scale = torch.empty((2,), dtype=torch.float32, device=logits.device)
        native._call("mfh_row_mean", self.log_probs.log_prob.data_ptr(), labels.data_ptr(), wide, stride, logits.shape[0],
                     -1.0, self._scale.data_ptr(), native._stream())
        self.value = self._scale[0]

    def backward(self):
        logits, labels = self.parents
        if not logits.requires_grad:
            return
        buffer, add = logits.grad_buffer()
        seed = native._device_f32(self.grad, "seed").reshape(()).expand(logits.value.shape[0])
        _log_probs_gradient(logits.value, labels.value, self.log_probs, seed, None, self._scale[1:], -1.0, buffer, add)


class DistillationLoss(GradientOp):
    """The distillation loss of a student's logits node against a teacher's record (ids and logits nodes, and
    optionally row weights); ``saved`` holds the last forward's DistillLoss."""

    def __init__(self, logits, teacher_ids, teacher_logits, row_weights=None, temperature=1.0, name="DistillationLoss"):
        super().__init__(logits, teacher_ids, teacher_logits, *([] if row_weights is None else [row_weights]), name=name)
        self.temperature = _temperature(temperature)
        self.saved = None

    def forward(self, logits, teacher_ids, teacher_logits, row_weights=None):
        _on_gpu(logits, "DistillationLoss")
        self.saved = distill_loss_forward(logits, teacher_ids, teacher_logits, temperature=self.temperature,
                                          row_weights=row_weights)
        self.value = self.saved.loss

    def backward(self):
        logits, teacher_ids = self.parents[:2]
        if not logits.requires_grad:
            return
        buffer, add = logits.grad_buffer()
        distill_loss_backward(logits.value, teacher_ids.value, self.saved, self.grad, temperature=self.temperature,
                              out=buffer, add=add)
