"""Matrices orthogonalised by Newton-Schulz products, on libmfhip: the update that the ``Muon`` optimiser makes of a
parameter's momentum.

``orthogonalize`` and ``orthogonalize_many`` take float32, bfloat16 or float16 matrices; a tensor of more
dimensions (a convolution's kernel) is one of its first dimension by the others. All matrices of a call go
through their products together, one launch a product. There is no host path. The reference has no counterpart:
its only optimisers with a state are elementwise.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import native
from .memory import overlap

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # steep at 0, and within 0.7 .. 1.2 for what began above 0.002, in five steps
STEPS = 5
STEPS_MAX = 64
SIDE_LIMIT = 1 << 20
ELEMENTS_LIMIT = 2 ** 31 - 1
COUNT_LIMIT = 1 << 16  # matrices of a call


def _matrix(value, name):
    """A 2-D view (or copy) of contiguous rows of a GPU tensor of two or more dimensions."""
    if not (isinstance(value, torch.Tensor) and value.is_cuda and value.dtype in native.TYPE_CODES):
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 torch tensor on the GPU")
    if value.ndim < 2:
        raise ValueError(f"{name} must have two dimensions or more")
    if value.ndim > 2:
        value = value.reshape(value.shape[0], math.prod(value.shape[1:]))
    rows, cols = value.shape
    if max(rows, cols) > SIDE_LIMIT or rows * cols > ELEMENTS_LIMIT:
        raise ValueError(f"{name} may have sides of {SIDE_LIMIT} and {ELEMENTS_LIMIT} elements at most")
    if rows and cols and ((cols > 1 and value.stride(1) != 1) or (rows > 1 and value.stride(0) < cols)):
        value = value.contiguous()
    return value


@lru_cache(maxsize=64)
def _checked_polynomial(coefficients, steps):
    """The coefficients, once it is shown that the steps keep every singular value below 3.5 and b x^2 + c x^4 below
    15.9: the kernels hold X, G and B = b G + c G G 2^12 times as large in float16, which ends at 2^12 * 15.99. The
    values that a step meets are all of 0 .. top (a continuous image of 0 .. 1 that holds 0); they are sampled."""
    a, b, c = coefficients
    top = 1.0
    for _ in range(steps):
        values = [top * i / 4096 for i in range(4097)]
        factors = [b * x * x + c * x ** 4 for x in values]
        top = max(abs(x * (a + f)) for x, f in zip(values, factors))
        if not (max(map(abs, factors)) < 15.9 and top < 3.5):
            raise ValueError(f"the coefficients {coefficients} take singular values out of range in {steps} steps")
    return coefficients


def _polynomial(coefficients, steps):
    steps = int(steps)
    if not 1 <= steps <= STEPS_MAX:
        raise ValueError(f"steps must lie between 1 and {STEPS_MAX}")
    coefficients = tuple(float(v) for v in coefficients)
    if len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients):
        raise ValueError("coefficients must be three finite numbers")
    return _checked_polynomial(coefficients, steps), steps


def _eps(value):
    value, held = float(value), native._float32(value)
    if not (math.isfinite(held) and value >= 0.0 and (held > 0.0 or value == 0.0)):
        raise ValueError("eps must be 0, or positive and finite in float32")
    return held


@lru_cache(maxsize=256)
def _workspace(shapes):
    table = (native.OrthogonalMatrix * len(shapes))(*((0, 0, cols, cols, rows, cols) for rows, cols in shapes))
    return native.workspace_bytes("mfh_orthogonalize_workspace", table, len(shapes))


def orthogonalize_many(matrices, *, steps=STEPS, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """Each matrix M taken through ``steps`` Newton-Schulz steps, as a list of tensors of their shapes and types.

    With X = M / (|M| + eps), |M| the Frobenius norm, a step makes X = a X + (b G + c G G) X of X X^T = G (of the
    shorter side): each singular value x becomes x (a + b x^2 + c x^4), which the default coefficients bring near 1.
    The products are formed to float32's precision (with at most 8 rows or columns, to 64 bits') and the result is
    rounded once to the matrix's type; a matrix
    of zeros stays one (for an eps above 0), and one with an infinity or NaN becomes NaN. The same call
    gives the same bits each time; which order a matrix's sums are added in may depend on the call's other matrices.
    ``out`` takes the results (each a contiguous
    tensor of its matrix's shape and type, possibly the matrix itself but no other one's memory). Other coefficients must keep values of
    0 .. 1 below 3.5, and b x^2 + c x^4 below 15.9, at every step."""
    matrices = list(matrices)
    (a, b, c), steps = _polynomial(coefficients, steps)
    eps = _eps(eps)
    if len(matrices) > COUNT_LIMIT:
        raise ValueError(f"a call takes at most {COUNT_LIMIT} matrices")
    views = [_matrix(value, "a matrix") for value in matrices]
    if out is None:
        out = [torch.empty_like(value, memory_format=torch.contiguous_format) for value in matrices]
    else:
        out = list(out)
        if len(out) != len(matrices):
            raise ValueError("out must hold a tensor for each matrix")
        for value, to in zip(matrices, out):
            if not (isinstance(to, torch.Tensor) and to.is_cuda and to.dtype is value.dtype and to.shape == value.shape
                    and to.is_contiguous()):
                raise ValueError("out must hold contiguous GPU tensors of the matrices' shapes and types")
        if overlap(out, [(view, i) for i, view in enumerate(views)]):
            raise ValueError("out must share no memory but with its own matrix")
    native._on_current_device(*matrices, *out)
    rows = {}
    for view, to in zip(views, out):
        if view.numel():
            rows.setdefault(view.dtype, []).append((view, to))
    for dtype, pairs in rows.items():
        shapes = tuple(tuple(view.shape) for view, _ in pairs)
        table = (native.OrthogonalMatrix * len(pairs))(*(
            (view.data_ptr(), to.data_ptr(), view.stride(0) if view.shape[0] > 1 else view.shape[1], view.shape[1], *view.shape)
            for view, to in pairs))
        workspace, held = native.byte_workspace(_workspace(shapes))
        native._call("mfh_orthogonalize", table, len(pairs), native.TYPE_CODES[dtype], steps, a, b, c, eps, workspace, held,
                     native.stream_counters(), native._stream())
    return out


def orthogonalize(matrix, *, steps=STEPS, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """``orthogonalize_many`` of one matrix."""
    return orthogonalize_many([matrix], steps=steps, coefficients=coefficients, eps=eps, out=None if out is None else [out])[0]


@lru_cache(maxsize=64)
def _muon_workspace(shapes):
    table = (native.MuonTensor * len(shapes))(*((0, 0, 0, rows, cols, 0.0, 0.0) for rows, cols in shapes))
    return native.workspace_bytes("mfh_muon_workspace", table, len(shapes))


def muon_update_many(updates, *, momentum=0.95, nesterov=True, grad_scale=1.0, steps=STEPS, coefficients=COEFFICIENTS,
                     eps=1e-7):
    """One Muon step, in place, for (param, grad, buffer, rate, decay) tuples of float32 tensors of a shape with two
    dimensions or more: with g = grad * grad_scale, buffer = momentum * buffer + g; the parameter becomes
    (1 - decay) param - rate O, with O the orthogonalised g + momentum * buffer (buffer without nesterov). A strided
    param or buffer is updated through a contiguous copy that is written back; neither may overlap itself or another
    of the call's tensors."""
    (a, b, c), steps = _polynomial(coefficients, steps)
    eps = _eps(eps)
    updates = list(updates)
    rows, held, back = [], [], []  # held: the copies of strided tensors, until the call is issued
    for param, grad, buffer, rate, decay in updates:
        tensors = [native._device_f32(t, name) for t, name in ((param, "param"), (grad, "grad"), (buffer, "buffer"))]
        if any(t.shape != param.shape for t in tensors):
            raise ValueError("Muon updates tensors of the parameter's shape")
        shape = tuple(_matrix(tensors[0], "param").shape)
        native._on_current_device(*tensors)
        if not param.numel():
            continue
        held.append(tensors)
        back += [(old, new) for old, new in ((param, tensors[0]), (buffer, tensors[2])) if old is not new]
        rows.append((*(t.data_ptr() for t in tensors), *shape, 1.0 - decay, float(rate)))
    if not rows:
        return
    if len(rows) > COUNT_LIMIT:
        raise ValueError(f"a Muon step takes at most {COUNT_LIMIT} parameters")
    # The caller's tensors, not their copies: a copy is written back over what it was made of.
    if overlap([t for param, _, buffer, _, _ in updates for t in (param, buffer)], [(grad, None) for _, grad, *_ in updates]):
        raise ValueError("the params and buffers of a Muon step must not overlap, nor its gradients any of them")
    table = (native.MuonTensor * len(rows))(*rows)
    workspace, size = native.byte_workspace(_muon_workspace(tuple(row[3:5] for row in rows)))
    native._call("mfh_muon_step", table, len(rows), float(momentum), int(bool(nesterov)), float(grad_scale), steps, a, b, c,
                 eps, workspace, size, native.stream_counters(), native._stream())
    for old, new in back:
        old.copy_(new)
