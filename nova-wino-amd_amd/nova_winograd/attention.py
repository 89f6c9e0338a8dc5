"""Attention to an encoder's states on the gfx950 library:
``nova_cross_attention`` and the module ``NovaCrossAttention``, forward and
backward.

No counterpart in the reference: in a UNet this is what stands behind a block's
convolutions, from the pixels (channels-last activations, as they are) to the
prompt's states; in a decoder, from new tokens to the encoder's.
"""

import torch.nn as nn

from nova_winograd.ops import native


def nova_cross_attention(query, key, value, key_mask=None, scale=None):
    """``softmax(scale * query key^T) value`` for every head, queries and keys
    of any two lengths.

    Args:
        query:    [B, Lq, H, D] float16 or bfloat16 tensor on the GPU, D up to
                  256; any strides with a dense last axis (others are copied).
        key:      [B, Lk, KV, D], KV a divisor of H (query head h reads key head
                  h // (H // KV)), or [1, Lk, KV, D] where one sequence of
                  states serves the whole batch. Halves of one projection are
                  read where they are.
        value:    shaped like ``key``.
        key_mask: optional [B, Lk] (or [1, Lk]) boolean tensor, False for keys
                  that take no part (padding); such keys may hold anything. A
                  query without any key gives zeros, and no gradient.
        scale:    default D ** -0.5.

    Returns a dense [B, Lq, H, D] tensor of the query's type. Scores, sums and
    outputs are accumulated in float32, the probabilities rounded to the
    inputs' type for their product. Differentiable (once, in reverse mode) with
    respect to query, key and value. Runs on PyTorch's current stream; results
    do not change from call to call.
    """
    return native().cross_attention(query, key, value, key_mask, scale)


class NovaCrossAttention(nn.Module):
    """Projections around ``nova_cross_attention``: queries from ``x``
    [B, L, query_dim], keys and values from ``context`` [B or 1, S,
    context_dim], the heads' outputs back to query_dim."""

    def __init__(self, query_dim, context_dim=None, heads=8, dim_head=64, kv_heads=None,
                 bias=False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads % kv_heads:
            raise ValueError(f"NovaCrossAttention: {kv_heads} key heads do not divide {heads}")
        context_dim = query_dim if context_dim is None else context_dim
        self.heads, self.kv_heads, self.dim_head = heads, kv_heads, dim_head
        self.to_q = nn.Linear(query_dim, heads * dim_head, bias=bias)
        self.to_k = nn.Linear(context_dim, kv_heads * dim_head, bias=bias)
        self.to_v = nn.Linear(context_dim, kv_heads * dim_head, bias=bias)
        self.to_out = nn.Linear(heads * dim_head, query_dim)

    def forward(self, x, context, key_mask=None):
        q = self.to_q(x).unflatten(-1, (self.heads, self.dim_head))
        k = self.to_k(context).unflatten(-1, (self.kv_heads, self.dim_head))
        v = self.to_v(context).unflatten(-1, (self.kv_heads, self.dim_head))
        return self.to_out(nova_cross_attention(q, k, v, key_mask).flatten(-2))

    def extra_repr(self):
        return f"heads={self.heads}, kv_heads={self.kv_heads}, dim_head={self.dim_head}"
