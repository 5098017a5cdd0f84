"""Rotary positions of several axes: queries and keys turned by where they stand."""
from .. import _C


def rotary_positions(query, positions, key=None, sections=None, base=10000.0, interleaved=False):
    """Turns pairs of columns of every head by angles that grow with the position along an axis.

    Pair i of an axis with n pairs turns by ``positions[..., axis] * base ** (-i / n)``:
    (u, v) becomes (u cos - v sin, u sin + v cos), so that a product of a query and a key depends on the distance of their
    positions along every axis (time, depth, rows, columns).  Goes before :func:`cross_attention` and :func:`window_attention`: the
    states of a map by their voxels, the queries of a region by the places of its bins.  Differentiable in query and key.

    Args:
        query (Tensor): (images, states, heads, dim), float32, float16 or bfloat16, of any strides (a part of a projection's rows is
            read where it lies)
        positions (Tensor): (images, states, axes), float32, int32 or int64, of any strides (one map's may be expanded over the
            images); 1 to 4 axes
        key (Tensor): (images, states, key_heads, dim) of the same type: turned in the same pass
        sections (sequence of int): number of pairs of each axis, together at most dim // 2 and 256; None divides dim // 2 evenly, the
            first axes taking what is left over
        base (float): at least 1; the slowest pair of a long section turns by about 1 / base
        interleaved (bool): pairs are columns (2i, 2i + 1); else (i, i + pairs), counted over all axes.  Columns behind the pairs
            are copied

    Angles are formed in 64 bits, and far positions turn as exactly as near ones (up to 2^31; a position that is not finite gives NaN).
    Returns the turned query, or (query, key): contiguous, of the same shapes and types.
    """
    return _C._native.rotary_positions(query, key, positions, sections, base, interleaved)
