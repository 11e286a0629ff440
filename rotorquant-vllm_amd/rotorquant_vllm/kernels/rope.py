"""Position rotation (rotary embedding) on the way into a cache: a layer's rotation and its store in one call.

rope_compress_store writes the codebook cache (compress_store), rope_q8_store the 8-bit cache (q8_store) and
rope_kv16_store plain 16-bit pages; each also returns the rotated queries.  No counterpart in the reference, whose model rotates
before the backend is called.

cos_sin is the table a model's rotary embedding keeps, (positions, rot_dim): the cosines of rot_dim / 2 angles, then their sines, fp32 or
of the rows' dtype.  Angle i turns the dims (i, i + rot_dim / 2) (neox=True) or (2 i, 2 i + 1) (neox=False), in fp32 with each product
and the sum rounded once; dims from rot_dim on stay.  Keys are not rounded to their dtype between rotation and codes: the cache holds what the
store of the fp32 result would.  A token whose position is outside the table is rotated by NaN.  rot_dim and
head_dim are multiples of 16.

Calls run on the current stream of the tensors' device, whichever device is current.
"""
from __future__ import annotations

import torch

from .. import _lib
from .q8 import _format

__all__ = ["rope_compress_store", "rope_q8_store", "rope_kv16_store"]


def rope_compress_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                        kv_cache: torch.Tensor, slot_mapping: torch.Tensor, rot_T_even: torch.Tensor, rot_T_odd: torch.Tensor,
                        k_boundaries: torch.Tensor, v_boundaries: torch.Tensor, neox: bool = True, out_q: torch.Tensor | None = None,
                        rot_block: int | None = None, dense3: bool = False) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and compress key and value into slots of the codebook cache.

    Returns the rotated queries (out_q, which may be query itself; None without query).  The cache's bytes are those of
    compress_store of the rotated fp32 keys and the values in fp32; its arguments are compress_store's.  Slots outside the cache are skipped, and
    a slot is given once.
    """
    if rot_block is None:
        from . import _rt_block
        rot_block = _rt_block(rot_T_even, rot_T_odd)
    return _lib.ops().rope_compress_store(query, key, value, positions, cos_sin, kv_cache, slot_mapping, rot_T_even, rot_T_odd, k_boundaries,
                                          v_boundaries, neox, out_q, rot_block, dense3)


def rope_q8_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                  kv_cache: torch.Tensor, slot_mapping: torch.Tensor, fmt: str = "int8", neox: bool = True, out_q: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and quantise key and value into slots of the 8-bit cache.

    Returns the rotated queries (out_q, which may be query itself; None without query).  The cache's bytes are those of
    q8_store of the rotated fp32 keys and the values; slots, groups, fmt and workspace are q8_store's.
    """
    return _lib.ops().rope_q8_store(query, key, value, positions, cos_sin, kv_cache, slot_mapping, _format(fmt), neox, out_q, workspace)


def rope_kv16_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, neox: bool = True,
                    out_q: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and append key and value to plain 16-bit pages.

    k_cache and v_cache are (num_blocks, block_size, H, D) of key's dtype, fp16 or bf16, contiguous over D (views of one tensor
    of both, or paged_decompress's, as they are).  Returns the rotated queries (out_q, which may be query itself; None without query).
    Slots outside the cache are skipped, and a slot is given once.
    """
    return _lib.ops().rope_kv16_store(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, neox, out_q)
