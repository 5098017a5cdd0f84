"""Group norm with its activation over channels-last tensors, in one operation with its gradient."""
import torch
import torch.nn as nn

from .. import _C

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` with mean and variance of every image's groups of channels.

    Channels are the last dimension, as in the states that :func:`cross_attention` reads; a map of (N, C, D, H, W) in torch's
    channels-last memory is given as ``x.permute(0, 2, 3, 4, 1)``, which copies nothing.  Differentiable in x, weight and bias;
    results do not depend on the order in which the GPU's blocks run.

    Args:
        x (Tensor): (images, ..., channels), float32, float16 or bfloat16
        groups (int): must divide the channels; a group is a run of consecutive ones
        weight, bias (Tensor): (channels,), of x's type or float32, both alike; None stands for 1 and 0
        eps (float): added to the variance
        activation (str): None, "relu", "silu" (z times the logistic function) or "gelu" (z times the normal distribution's)

    Statistics and sums are held in float32, about values of their own, so that they keep their accuracy far from 0; the result is
    rounded once.  Returns a contiguous tensor of x's shape and type.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, but got {activation!r}")
    return _C._native.group_norm(x, groups, weight, bias, eps, ACTIVATIONS[activation])


class GroupNorm(nn.Module):
    """:func:`group_norm` as a layer, with weight and bias in float32 unless ``dtype`` says otherwise."""

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation=None, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, but got {activation!r}")
        if groups < 1 or channels % groups != 0:
            raise ValueError(f"groups ({groups}) must divide the channels ({channels})")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        if affine:
            self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, affine={self.weight is not None}, activation={self.activation!r}"

    def forward(self, x):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps, self.activation)
