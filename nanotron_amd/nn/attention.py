from typing import Optional

import torch

from nanotron_amd import _ops


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
              causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """Attention `softmax(scale * q @ k.T) @ v` of every head over its own sequence, the scores never in memory.

    Either packed, sequences of any lengths end to end: q [tokens, heads, head_dim], k and v [tokens_k, kv_heads, head_dim], with
    cu_seqlens (int32 [sequences + 1], on the GPU: sequence s is the rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1) and, where keys differ
    from queries in number, cu_seqlens_k; without cu_seqlens it is one sequence.  Or a batch of equal lengths: q [batch, tokens, heads, head_dim], k and
    v [batch, tokens_k, kv_heads, head_dim], each possibly part of a larger tensor, as a cache's first positions are.  Lengths of zero and
    one are fine, and nothing is read back to the host.  A batched cache that is used up to lengths of its own is packed as well: cu_seqlens_k then names the part of
    each that is in use and, as sequences of no queries (cu_seqlens repeats an offset), the room behind it.  Calls with few queries are cut into runs of keys by the average
    length: caches of very different lengths take as long as their longest one does uncut.

    heads is a multiple of kv_heads: head h reads key head `h // (heads // kv_heads)`.  causal: of n queries and m keys of a sequence query i
    sees the keys 0 .. m - n + i, so the last ones belong together.  A query that sees no key has output 0 and no gradient, and so
    have rows before the first sequence and behind the last.  Whatever keys and values hold that a query does not see (NaN in padding,
    tokens to come) does not reach it.  A query whose keys all score minus infinity has NaN, as its softmax is 0 / 0: an overflow stays to be
    seen.  scale: 1 / sqrt(head_dim) by default.

    bfloat16 or float16, head_dim a multiple of 8 up to 128.  Products run on the matrix cores with fp32 sums; maxima and sums are fp32; the
    softmax's numerators, and in backward the scores' gradients, are rounded to the type of q for the products they go into.  Rows are read where they are
    if they lie on 16-byte boundaries, else from a copy.  The same inputs give the same bits, forward and backward.  In float16 the scores' gradients of a
    call share one power of two, from the largest finite gradient and value of all its sequences: what is 2^28 below 2 head_dim times their product loses bits.  Memory kept for
    the backward pass beside q, k, v and the result: a byte an element of the result and 4 bytes a query and head; freed on return, where queries are few or keys
    are in the backward pass, partial results of fp32.  At most 2^27 queries times heads and keys times kv_heads, 2^24 elements from row to row, and
    (rows / 128 + sequences + 2) * heads up to 2^22.  ValueError / TypeError for what does not fit, RuntimeError beyond these sizes; differentiable once."""
    return _ops.host.attention(q, k, v, cu_seqlens, cu_seqlens_k, causal, scale)
