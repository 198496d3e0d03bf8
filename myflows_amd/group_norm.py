"""Group norm with an activation over channels-last activations, on libmfhip.

A channels-last tensor (N, ..., C) holds a sample's positions one after the other, its channels together:
what a ``Dense`` layer makes of positions as rows. Its groups are C / groups neighbouring channels of one
sample over all its positions, normalised by their own mean and variance: unlike a batch norm's, a sample's
result depends on no other sample, in training and inference alike.

``group_norm_forward`` / ``group_norm_backward`` take float32, bfloat16 or float16 activations (gamma, beta and
all statistics are float32); ``GroupNorm_Op`` is the operator of a ``Graph`` and ``GroupNorm`` the layer. There is
no host path. The reference has no counterpart: its only norm is the batch norm.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import native
from .device import torch_device
from .graph import GradientOp, Variable
from .layers import Layer, _count

ACTIVATIONS = {None: 0, "relu": 1, "silu": 3}
POSITIONS_LIMIT = 1 << 30
CHANNELS_LIMIT = 1 << 16
COLUMNS_LIMIT = 1 << 28  # samples times channels


def _activations(value, name, like=None):
    """A contiguous GPU tensor of a type that group norm takes (and of like's type and shape)."""
    if not (isinstance(value, torch.Tensor) and value.is_cuda and value.dtype in native.TYPE_CODES):
        raise TypeError(f"{name} must be a float32, bfloat16 or float16 torch tensor on the GPU")
    if like is not None and (value.dtype is not like.dtype or value.shape != like.shape):
        raise ValueError(f"{name} must have x's type and shape")
    return value if value.is_contiguous() else value.contiguous()


@lru_cache(maxsize=256)
def _sizes(shape, groups):
    """(n, positions, channels, groups) of a channels-last shape."""
    if len(shape) < 2:
        raise ValueError("group norm expects a channels-last tensor (N, ..., C)")
    n, channels, positions = int(shape[0]), int(shape[-1]), 1
    for size in shape[1:-1]:
        positions *= int(size)
    groups = int(groups)
    if groups < 1 or channels < 1 or channels % groups:
        raise ValueError(f"the {channels} channels must divide into {groups} groups")
    if not 1 <= positions <= POSITIONS_LIMIT:
        raise ValueError(f"group norm takes 1 to {POSITIONS_LIMIT} positions")
    native._within_int32(sample=positions * channels)
    if channels > CHANNELS_LIMIT or n * channels > COLUMNS_LIMIT:
        raise ValueError(f"group norm takes at most {CHANNELS_LIMIT} channels and {COLUMNS_LIMIT} channels over all samples")
    return n, positions, channels, groups


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'relu' or 'silu', not {name!r}")
    return ACTIVATIONS[name]


def _per_channel(value, channels, name):
    value = native._device_f32(value, name)
    if tuple(value.shape) != (channels,):
        raise ValueError(f"{name} must have shape (C,)")
    return value


@lru_cache(maxsize=256)
def _workspace(sizes, code, backward):
    return native.workspace_bytes("mfh_group_norm_workspace", *sizes, code, int(backward))


def group_norm_forward(x, gamma, beta, groups, *, eps=1e-5, activation=None):
    """(y, mean, inv_std) of channels-last x (N, ..., C): y = act(gamma (x - mean) inv_std + beta) of x's type,
    with the biased variance in inv_std = (variance + eps)^(-1/2) and both statistics float32 (N, groups).
    activation is None, "relu" or "silu"."""
    x = _activations(x, "x")
    sizes = n, positions, channels, groups = _sizes(x.shape, groups)
    act, eps = _activation(activation), float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    gamma, beta = _per_channel(gamma, channels, "gamma"), _per_channel(beta, channels, "beta")
    y = torch.empty_like(x)
    mean, inv_std = gamma.new_empty((n, groups)), gamma.new_empty((n, groups))
    code = native.TYPE_CODES[x.dtype]
    workspace, held = native.byte_workspace(_workspace(sizes, code, False))
    native._call("mfh_group_norm_forward", x.data_ptr(), code, *sizes, gamma.data_ptr(), beta.data_ptr(), act, eps,
                 y.data_ptr(), mean.data_ptr(), inv_std.data_ptr(), workspace, held, native._stream())
    return y, mean, inv_std


def _gradient_buffer(value, like, name):
    if value is None:
        return None
    if not (isinstance(value, torch.Tensor) and value.is_cuda and value.dtype is like.dtype and value.is_contiguous()
            and value.shape == like.shape):
        raise ValueError(f"{name} must be a contiguous GPU tensor of its forward value's type and shape")
    return value


def group_norm_backward(x, dy, gamma, beta, mean, inv_std, *, activation=None, x_grad=None, gamma_grad=None,
                        beta_grad=None, accumulate=(True, True, True)):
    """Write (or add, per ``accumulate``) the requested gradients of group_norm_forward into x_grad (x's type),
    gamma_grad and beta_grad (float32), from the output's gradient dy and the forward's mean and inv_std."""
    x = _activations(x, "x")
    dy = _activations(dy, "dy", x)
    if not (isinstance(mean, torch.Tensor) and mean.ndim == 2):
        raise ValueError("mean must be the (N, groups) tensor from group_norm_forward")
    sizes = n, positions, channels, groups = _sizes(x.shape, mean.shape[1])
    act = _activation(activation)
    gamma, beta = _per_channel(gamma, channels, "gamma"), _per_channel(beta, channels, "beta")
    mean, inv_std = native._device_f32(mean, "mean"), native._device_f32(inv_std, "inv_std")
    if tuple(mean.shape) != (n, groups) or tuple(inv_std.shape) != (n, groups):
        raise ValueError("mean and inv_std must be the (N, groups) tensors from group_norm_forward")
    x_grad = _gradient_buffer(x_grad, x, "x_grad")
    gamma_grad = _gradient_buffer(gamma_grad, gamma, "gamma_grad")
    beta_grad = _gradient_buffer(beta_grad, gamma, "beta_grad")
    if x_grad is None and gamma_grad is None and beta_grad is None:
        return
    code = native.TYPE_CODES[x.dtype]
    workspace, held = native.byte_workspace(_workspace(sizes, code, True))
    add_x, add_gamma, add_beta = (int(bool(a)) for a in accumulate)
    native._call("mfh_group_norm_backward", x.data_ptr(), dy.data_ptr(), code, *sizes, gamma.data_ptr(), beta.data_ptr(),
                 mean.data_ptr(), inv_std.data_ptr(), act, native._addr(x_grad), native._addr(gamma_grad),
                 native._addr(beta_grad), add_x, add_gamma, add_beta, workspace, held, native._stream())


class GroupNorm_Op(GradientOp):
    """Group norm of a channels-last x with parameters gamma, beta (C,) and an activation. With ``positions``, x
    is 2-D, its rows the positions of the samples one sample after the other (a Dense layer's rows)."""

    def __init__(self, x, gamma, beta, groups, eps=1e-5, activation=None, positions=None, name=None):
        super().__init__(x, gamma, beta, name=name)
        self.groups, self.eps = int(groups), float(eps)
        _activation(activation)
        self.activation = activation
        self.positions = None if positions is None else _count(positions, "positions")
        self._stats = None

    def _samples(self, value):
        if self.positions is None:
            return value
        if value.ndim != 2 or value.shape[0] % self.positions:
            raise ValueError(f"x must be 2-D with a multiple of {self.positions} rows")
        return value.reshape(-1, self.positions, value.shape[1])

    def forward(self, x, gamma, beta):
        if not (isinstance(x, torch.Tensor) and x.is_cuda):
            raise ValueError("GroupNorm runs on libmfhip and needs a GPU tensor (device=cpu is not supported)")
        y, mean, inv_std = group_norm_forward(self._samples(x), gamma, beta, self.groups, eps=self.eps,
                                              activation=self.activation)
        self.value = y.reshape(x.shape)
        self._stats = (mean, inv_std) if self.requires_grad else None

    def backward(self):
        x, gamma, beta = self.parents
        buffers = [node.grad_buffer() if node.requires_grad else (None, False) for node in self.parents]
        x_grad = None if buffers[0][0] is None else self._samples(buffers[0][0])
        group_norm_backward(self._samples(x.value), self._samples(self.grad), gamma.value, beta.value, *self._stats,
                            activation=self.activation, x_grad=x_grad, gamma_grad=buffers[1][0],
                            beta_grad=buffers[2][0], accumulate=tuple(add for _, add in buffers))


class GroupNorm(Layer):
    """Group norm over ``groups`` groups of ``num_features`` channels with gamma = 1, beta = 0 and an activation
    ("relu", "silu" or None); the same in training and inference. ``positions`` as in GroupNorm_Op."""

    def __init__(self, groups, num_features, eps=1e-5, activation=None, positions=None, name=None):
        super().__init__(name=name)
        self.groups, self.num_features = _count(groups, "groups"), _count(num_features, "num_features")
        if self.num_features % self.groups:
            raise ValueError(f"the {self.num_features} channels must divide into {self.groups} groups")
        self.eps, self.activation, self.positions = float(eps), activation, positions
        device = torch_device()
        prefix = f"{name}_" if name else ""
        self.gamma = Variable(torch.ones(self.num_features, device=device), trainable=True, name=prefix + "gamma")
        self.beta = Variable(torch.zeros(self.num_features, device=device), trainable=True, name=prefix + "beta")
        self.params = [self.gamma, self.beta]

    def forward(self, input_node):
        return GroupNorm_Op(input_node, self.gamma, self.beta, self.groups, eps=self.eps, activation=self.activation,
                            positions=self.positions)
