"""Attention over plain 16-bit pages (kv16_attention): single tokens and drafts, split over the contexts and joined.

The pages are K and V tensors (num_blocks, block_size, H, D), fp16 or bf16, in any strides over whole rows: paged_decompress's
outputs, or pages that rope_kv16_store appends to.  The codebook and 8-bit caches have attention of their own.
"""
from __future__ import annotations

import torch

from .. import _lib

__all__ = ["kv16_attention"]


def kv16_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   sm_scale: float | None = None, causal: bool = True, cu_seqlens_q: torch.Tensor | None = None, max_q_len: int | None = None,
                   max_seq_len: int | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new query tokens q (num_tokens, H_Q, D) over plain 16-bit pages of q's dtype.

    H_Q is a multiple of the pages' heads and D a multiple of 8 up to 256; pages may have any number of slots.
    block_table (num_seqs, max_blocks) and seq_lens (num_seqs,), the contexts with the new tokens
    included, are int32.  cu_seqlens_q (num_seqs + 1,) int32 splits q among the sequences; without it each has one token
    (a decode step).  Query i of sequence b sits at position seq_lens[b] - q_len_b + i; a row that sees no key is zeros, and infinities and
    NaN count only where a row sees them.  Queries of many tokens are right but slow: the keys are read again for every 32
    (token, query head) pairs of a kv head.
    max_q_len and max_seq_len: host ints that bound the query and context lengths (default: all of q, and the
    block table's capacity); what lies past them is not read, and positions stay as above.  out: a buffer to fill, whose
    rows of such tokens and of no sequence stay as they are (without it they are not initialised).
    Rows of q start at multiples of 16 bytes and those of out of 8; others are refused.
    workspace: scratch (rq_kv16_attention_workspace_bytes bytes), by default of this call from torch's allocator; a graph
    captured without torch's graph classes needs it, since nothing else keeps the scratch for its replays.
    """
    return _lib.ops().kv16_attention(q, k_cache, v_cache, block_table, seq_lens, sm_scale, causal, cu_seqlens_q, max_q_len, max_seq_len, out, workspace)
