"""Attention of region features, or any other queries, to an encoder's states of another length."""
from .. import _C


def cross_attention(query, key, value, batch_index=None, lengths=None, mask=None, scale=None):
    """softmax(scale * query . key) value over the states of each region's image.

    Stands beside RoIAlign: where that reads a feature map at the places of a region, this reads it wherever the region's
    queries find what they look for.  Differentiable in query, key and value; results do not depend on the order in which the
    GPU's blocks run.

    Args:
        query (Tensor): (regions, tokens, heads, dim), float32, float16 or bfloat16; dim at most 256
        key, value (Tensor): (images, states, key_heads, dim) of the same type; ``heads`` must be a multiple of
            ``key_heads``, query head h reads key head h // (heads // key_heads)
        batch_index (Tensor): image of every region, (regions,) of a floating or integer type, such as ``rois[:, 0]``;
            floating ones are cut towards zero.  A region whose image does not exist gives zeros and sets the status bit
            that the roi operations set.  None: region r reads image r
        lengths (Tensor): int32 or int64 (images,): only the first ``lengths[n]`` states of an image are read
        mask (Tensor): bool (images, states): only states whose element is true are read
        scale (float): None stands for dim ** -0.5

    A query for which no state is left gives zeros, and no gradients.  States that are not read may hold anything.
    Returns a contiguous tensor of the query's shape and type.  Sums, weights and statistics are held in float32 and the
    result is rounded once; for float16 and bfloat16 the weights are rounded to that type before they meet the values, and the
    gradients are formed with the rounded result.
    """
    return _C._native.cross_attention(query, key, value, batch_index, lengths, mask, scale)
