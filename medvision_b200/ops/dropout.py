"""Dropout from a counter-based generator: the mask is a function of a seed, and never stored."""
import torch
import torch.nn as nn

from .. import _C


def dropout(x, p=0.5, seed=None, offset=0, residual=None, training=True):
    """``residual + (x / (1 - p) where kept, else 0)``, each element dropped with probability p.

    Whether an element is kept depends on (seed, offset, its place in the row-major order of x) alone: two calls with the same
    seed and offset drop the same places, and the gradient finds the mask again from them.  The generator is Philox 4x32-10
    with 16 bits per element, so p is taken as the nearest multiple of 2**-16 and the scale follows that.

    Args:
        x (Tensor): float32, float16 or bfloat16, of any shape
        p (float): between 0 and 1
        seed (int or Tensor): 64 bits, or an int64 tensor of one element on x's device, which a captured graph reads at every
            replay and which must not change between forward and backward; None draws one from torch's CPU generator (in a
            captured graph a replay repeats the mask drawn while it was captured)
        offset (int): 64 bits; calls that share a seed (the layers of a step) take different ones
        residual (Tensor): added to the result in the same pass; of x's shape and type
        training (bool): False gives x, or x + residual, of the same shapes and types (on the CPU as well)

    Differentiable in x and residual.  A dropped element gives 0 whatever it holds.
    """
    if not training:
        if residual is None:
            return x
        if not isinstance(residual, torch.Tensor):
            raise TypeError(f"residual must be a Tensor, not {type(residual).__name__}")
        if residual.device != x.device:
            raise RuntimeError("expected all tensors to be on the same CUDA device")
        if residual.dtype != x.dtype:
            raise RuntimeError(f"expected scalar type {x.dtype} but found {residual.dtype}")
        if residual.shape != x.shape:
            raise RuntimeError("dropout: x and residual must have the same shape")
        return x + residual
    if seed is None:
        seed = int(torch.randint(2 ** 63 - 1, (), device="cpu"))
    return _C._native.dropout(x, p, seed, offset, residual)


class Dropout(nn.Module):
    """:func:`dropout` as a layer: a seed per call from torch's CPU generator, or the one given to the call."""

    def __init__(self, p=0.5):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
        self.p = float(p)

    def extra_repr(self):
        return f"p={self.p}"

    def forward(self, x, residual=None, seed=None, offset=0):
        return dropout(x, self.p, seed, offset, residual, self.training)
