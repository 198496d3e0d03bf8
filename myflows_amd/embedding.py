"""Embeddings on libmfhip: rows of a table by token, scaled, and the table's gradient.

``embedding_forward`` / ``embedding_backward`` take float32, bfloat16 or float16 tables and int32 or int64
tokens of any shape; ``Embedding_Op`` is the operator of a ``Graph`` and ``Embedding`` the layer, the first of a
network over tokens as ``Dense`` is of one over features. A negative token is none: its row is zeros and it
adds to no gradient. There is no host path. The reference has no counterpart: its layers take floats.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import native
from .graph import GradientOp
from .init import make_initializer
from .layers import Layer, _count, _parameter
from .memory import share_memory

COUNT_LIMIT = 1 << 30
VOCAB_LIMIT = 1 << 24
DIM_LIMIT = 1 << 20
_WHOLE = {torch.int32: 0, torch.int64: 1}  # whether tokens are int64


def _rows(value, name):
    """A 2-D GPU tensor of contiguous rows of a type that embeddings take, and its row stride."""
    if not (isinstance(value, torch.Tensor) and value.is_cuda and value.dtype in native.TYPE_CODES):
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 torch tensor on the GPU")
    if value.ndim != 2:
        raise ValueError(f"{name} must be 2-D (rows, elements)")
    rows, dim = value.shape
    if (dim > 1 and value.stride(1) != 1) or (rows > 1 and value.stride(0) < dim):
        value = value.contiguous()
    return value, value.stride(0) if rows > 1 else dim


def _tokens(ids):
    """(flat ids, whether they are int64, their stride); a 1-D tensor is read in place at any stride."""
    wide = _WHOLE.get(ids.dtype) if isinstance(ids, torch.Tensor) and ids.is_cuda else None
    if wide is None:
        raise TypeError("ids must be an int32 or int64 torch tensor on the GPU")
    flat = ids if ids.ndim == 1 else ids.reshape(-1)
    if flat.numel() > COUNT_LIMIT:
        raise ValueError(f"an embedding takes at most {COUNT_LIMIT} tokens")
    return flat, wide, flat.stride(0)


def _table_sizes(vocab, dim):
    if not 0 < vocab <= VOCAB_LIMIT or not 0 < dim <= DIM_LIMIT:
        raise ValueError(f"a table has 1 to {VOCAB_LIMIT} rows of 1 to {DIM_LIMIT} elements")


def _scale(value):
    value = float(value)
    if not math.isfinite(native._float32(value)):
        raise ValueError("scale must be finite in float32")
    return value


@lru_cache(maxsize=256)
def _workspace(count, vocab, dim, code):
    return native.workspace_bytes("mfh_embedding_workspace", count, vocab, dim, code)


def embedding_forward(table, ids, *, scale=1.0):
    """scale times the table's row of each token: a tensor of ids' shape and one more dimension, of the table's
    type. table is (vocab, dim) with contiguous rows, which may lie apart. A negative token's row is zeros, that
    of a token beyond the vocabulary NaN."""
    table, table_stride = _rows(table, "table")
    vocab, dim = table.shape
    _table_sizes(vocab, dim)
    flat, wide, step = _tokens(ids)
    native._on_current_device(table, flat)
    out = torch.empty((*ids.shape, dim), dtype=table.dtype, device=table.device)
    native._call("mfh_embedding", table.data_ptr(), native.TYPE_CODES[table.dtype], vocab, dim, table_stride,
                 flat.data_ptr(), wide, step, flat.numel(), _scale(scale), out.data_ptr(), dim, native._stream())
    return out


def embedding_backward(grad, ids, vocab, *, scale=1.0, out=None, add=False):
    """The gradient (vocab, dim) of the table from that of embedding_forward's output (ids' shape, dim): scale
    times the sum of the rows of each token, in float32 and an order that is the same each time (that of the tokens for
    those that come at most 64 times; the others' rows are summed in pieces), rounded once. It is written to
    (or, with add, added to) out, of grad's type or float32 with contiguous rows, which shares no memory with grad
    and ids; a row that no token names is zeros (with add, left as it is). Tokens beyond the vocabulary count nowhere."""
    flat, wide, step = _tokens(ids)
    if not isinstance(grad, torch.Tensor) or grad.ndim != ids.ndim + 1 or grad.shape[:-1] != ids.shape:
        raise ValueError("grad must have the shape of ids and one more dimension")
    vocab, dim = int(vocab), int(grad.shape[-1])
    _table_sizes(vocab, dim)
    grad, grad_stride = _rows(grad if grad.ndim == 2 else grad.reshape(-1, dim), "grad")
    given = out is not None
    if not given:
        if add:
            raise ValueError("add needs an out tensor")
        out = torch.empty((vocab, dim), dtype=grad.dtype, device=grad.device)
    elif not (isinstance(out, torch.Tensor) and out.is_cuda and out.dtype in (grad.dtype, torch.float32)
              and tuple(out.shape) == (vocab, dim) and (dim <= 1 or out.stride(1) == 1)
              and (vocab <= 1 or out.stride(0) >= dim)):
        raise ValueError("out must be a (vocab, dim) GPU tensor of grad's type or float32 with contiguous rows")
    native._on_current_device(grad, flat, out)
    if given and (share_memory(out, grad) or share_memory(out, flat)):
        raise ValueError("out must share no memory with grad and ids")
    code = native.TYPE_CODES[grad.dtype]
    workspace, held = native.byte_workspace(_workspace(flat.numel(), vocab, dim, code))
    native._call("mfh_embedding_backward", grad.data_ptr(), code, flat.numel(), dim, grad_stride, flat.data_ptr(), wide,
                 step, vocab, _scale(scale), out.data_ptr(), native.TYPE_CODES[out.dtype],
                 out.stride(0) if vocab > 1 else dim, int(bool(add)), workspace, held, native._stream())
    return out


class Embedding_Op(GradientOp):
    """scale times the rows of a table (vocab, dim) by the tokens of a node (which has no gradient)."""

    def __init__(self, ids, table, scale=1.0, name=None):
        super().__init__(ids, table, name=name)
        self.scale = _scale(scale)

    def forward(self, ids, table):
        if not (isinstance(table, torch.Tensor) and table.is_cuda):
            raise ValueError("Embedding runs on libmfhip and needs a GPU tensor (device=cpu is not supported)")
        self.value = embedding_forward(table, ids, scale=self.scale)

    def backward(self):
        ids, table = self.parents
        if not table.requires_grad:
            return
        buffer, add = table.grad_buffer()
        embedding_backward(self.grad, ids.value, table.value.shape[0], scale=self.scale, out=buffer, add=add)


class Embedding(Layer):
    """A table of ``num_tokens`` rows of ``dim`` features, drawn from a normal distribution of standard deviation 1
    unless an initializer is given, and looked up by a node of tokens; ``scale`` multiplies the rows."""

    def __init__(self, num_tokens, dim, scale=1.0, name=None, initializer=None):
        super().__init__(name=name)
        self.num_tokens, self.dim, self.scale = _count(num_tokens, "num_tokens"), _count(dim, "dim"), _scale(scale)
        draw = make_initializer("normal", std=1.0) if initializer is None else make_initializer(initializer)
        self.W = _parameter(draw((self.num_tokens, self.dim)), name, "W")
        self.params = [self.W]

    def forward(self, input_node):
        return Embedding_Op(input_node, self.W, self.scale)
