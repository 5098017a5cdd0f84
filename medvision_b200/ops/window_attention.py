"""Attention of a sequence's tokens to the states around their own place, and to the first ones."""
from .. import _C


def window_attention(query, key, value, before, after=0, sinks=0, offsets=None, lengths=None, scale=None, rounded_weights=False):
    """softmax(scale * query . key) value over a sliding window of states, and a few first states that stay visible.

    Token t of a sequence stands at place ``p = offset + t`` among its states and reads the states ``j <= p + after`` with
    ``j >= p - before`` or ``j < sinks``.  Stands beside :func:`cross_attention`, for states in an order: the slices of a study, the
    scan lines of a map.  Whole sequences have offset 0; new tokens at the end of a cache ``lengths - tokens``.  Differentiable in
    query, key and value; results do not depend on the order in which the GPU's blocks run.

    Args:
        query (Tensor): (sequences, tokens, heads, dim), float32, float16 or bfloat16; dim at most 256
        key, value (Tensor): (sequences, states, key_heads, dim) of the same type; ``heads`` must be a multiple of
            ``key_heads``, query head h reads key head h // (heads // key_heads)
        before, after (int): states before and behind a token's own place that it reads; after=0 reads none that come later
        sinks (int): the first states, which every token reads as far as they do not come later than ``p + after``
        offsets (int or Tensor): place of the first token, for all sequences or int32 or int64 (sequences,); None stands for 0
        lengths (Tensor): int32 or int64 (sequences,): only the first ``lengths[n]`` states of a sequence are read
        scale (float): None stands for dim ** -0.5
        rounded_weights (bool): float16 and bfloat16: True rounds the weights to that type before they meet the values (and, for the values'
            gradient, the incoming one).  Up to a quarter less time; errors are then 1.2 to 1.4 times what a result's own rounding leaves, up to 1.5
            times in the values' gradient

    A token that reads no state gives zeros, and no gradients, whatever it and its gradient hold.  States that no token of their sequence
    reads may hold anything; one that is not finite and read by some may spoil the tokens near them, and a query or gradient that is not finite
    the gradients of states near those that its token reads.
    Returns a contiguous tensor of the query's shape and type.  Sums and statistics are held in float32 and the result is rounded
    once; weights and, in the gradients, the scores' slopes meet the values (keys, queries) as float32 or as two numbers of the type.
    """
    return _C._native.window_attention(query, key, value, before, after, sinks, offsets, lengths, scale, rounded_weights)
