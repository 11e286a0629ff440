"""Attention over plain 16-bit pages (kv16_attention): single tokens and drafts, split over the contexts and joined.

The pages are K and V tensors (num_blocks, block_size, H, D), fp16 or bf16, in any strides over whole rows: paged_decompress's
outputs, or pages that rope_kv16_store appends to.  The codebook and 8-bit caches have attention of their own.
"""
from __future__ import annotations

import functools
import math

import torch

from .. import _lib
from .q8 import _call, _device_index, _index, _row_strides, _scratch
from .rope import _check_pages

__all__ = ["kv16_attention"]


@functools.lru_cache(maxsize=4096)
def _attention_bytes(dev: int, num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int, max_q_len: int, max_seq_len: int) -> int:
    with torch.cuda.device(dev):  # (the GPU's number of CUs sizes the partial sums)
        return _lib.load().rq_kv16_attention_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, max_seq_len)


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
    shape, dtype, H = q.shape, q.dtype, k_cache.shape[2] if k_cache.dim() == 4 else 0
    if len(shape) != 3 or H < 1 or shape[1] % H or k_cache.dtype is not dtype:
        raise ValueError(f"q must be (tokens, a multiple of the pages' heads, head_dim) of the pages' dtype, got {tuple(shape)} of {dtype}")
    dev = _device_index(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q, out, workspace)
    T, HQ, D = shape
    pages = _check_pages(k_cache, v_cache, H, D)
    BS = pages[1]
    bt = _index(block_table, "block_table", torch.int32, 2)
    sl = _index(seq_lens, "seq_lens", torch.int32, 1)
    B, (tables, max_blocks) = sl.numel(), bt.shape
    if tables != B:
        raise ValueError("block_table and seq_lens differ in the number of sequences")
    cu = None
    if cu_seqlens_q is None:
        if T != B:
            raise ValueError(f"{T} query tokens and {B} sequences: cu_seqlens_q is needed")
        max_q_len = 1
    else:
        cu = _index(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1)
        if cu.numel() != B + 1:
            raise ValueError(f"cu_seqlens_q must have {B + 1} entries, got {cu.numel()}")
        max_q_len = T if max_q_len is None else min(int(max_q_len), T)
    qs = q.stride()
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    out = torch.empty(shape, dtype=dtype, device=q.device) if out is None else out
    os = out.stride()
    if out.shape != shape or out.dtype is not dtype or os[2] != 1:
        raise ValueError("out must have q's shape and dtype and be contiguous over head_dim")
    if T == 1 or HQ == 1:
        qs, os = _row_strides(shape, qs), _row_strides(shape, os)
    capacity = max_blocks * BS
    max_seq_len = capacity if max_seq_len is None else min(int(max_seq_len), capacity)
    keep, ws, ws_bytes = _scratch(workspace, _attention_bytes(dev, B, HQ, H, D, max_q_len, max_seq_len), q)
    _call(_lib.load().rq_kv16_attention, "rq_kv16_attention", dev,
          (q.data_ptr(), _lib.dtype_code(dtype), T, HQ, qs[0], qs[1], None if cu is None else cu.data_ptr(), B, max_q_len, 1 if causal else 0,
           k_cache.data_ptr(), v_cache.data_ptr(), *pages, H, D, bt.data_ptr(), max_blocks, bt.stride(0), sl.data_ptr(), max_seq_len,
           1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), out.data_ptr(), os[0], os[1], ws, ws_bytes))
    return out
