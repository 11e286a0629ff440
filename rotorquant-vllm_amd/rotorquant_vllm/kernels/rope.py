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
from .q8 import _call, _check_cache, _device_index, _format, _scratch, _store_bytes

__all__ = ["rope_compress_store", "rope_q8_store", "rope_kv16_store"]

_CODE, _I64, _F32 = _lib._DTYPE_CODE, torch.int64, torch.float32


# A decode step's call waits for the checks below (its kernel takes 4 us): each tensor's sizes and strides are fetched once, and what is wrong is
# only looked for where the checks fail.

def _operands(query, key, value, positions, cos_sin, slot_mapping, neox, out_q):
    """(rotated queries to return, tokens, kv heads, head_dim, the arguments that every call begins with)."""
    shape, dtype = key.shape, key.dtype
    if len(shape) != 3 or value.shape != shape or value.dtype is not dtype:
        raise ValueError("key and value must have the same (tokens, heads, head_dim) shape and dtype")
    N, H, D = shape
    kt, kh, kd = key.stride()
    vt, vh, vd = value.stride()
    if kd != 1 or vd != 1:
        raise ValueError("key and value must be contiguous over head_dim")
    for t, name in ((positions, "positions"), (slot_mapping, "slot_mapping")):
        if t.dtype is not _I64 or t.dim() != 1 or t.numel() < N or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int64 tensor of {N} tokens or more")
    table = cos_sin.dtype
    if cos_sin.dim() != 2 or table is not _F32 and table is not dtype:
        raise ValueError(f"cos_sin must be (positions, rot_dim), contiguous over rot_dim, of float32 or {dtype}")
    rows, rot = cos_sin.shape
    row, one = cos_sin.stride()
    if one != 1:
        raise ValueError(f"cos_sin must be (positions, rot_dim), contiguous over rot_dim, of float32 or {dtype}")
    if query is None:
        if out_q is not None:
            raise ValueError("out_q without query")
        HQ = qt = qh = ot = oh = 0
        q = o = None
    else:
        q_shape = query.shape
        if len(q_shape) != 3 or q_shape[0] != N or q_shape[2] != D or query.dtype is not dtype:
            raise ValueError(f"query must be ({N}, heads, {D}) of {dtype}, as key is")
        if out_q is None:
            out_q = torch.empty(q_shape, dtype=dtype, device=query.device)
        elif out_q.shape != q_shape or out_q.dtype is not dtype:
            raise ValueError("out_q must have query's shape and dtype")
        HQ = q_shape[1]
        qt, qh, qd = query.stride()
        ot, oh, od = out_q.stride()
        if qd != 1 or od != 1:
            raise ValueError("query and out_q must be contiguous over head_dim")
        if HQ == 1:
            qh = oh = 0
        q, o = query.data_ptr(), out_q.data_ptr()
    if N == 1:  # (strides over a single token or head may be any number in a view)
        kt = vt = qt = ot = 0
    if H == 1:
        kh = vh = 0
    try:
        code = _CODE[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}") from None
    return out_q, N, H, D, (q, key.data_ptr(), value.data_ptr(), code, N, HQ, qt, qh, kt, kh, vt, vh, H, D, positions.data_ptr(), cos_sin.data_ptr(),
                            2 if table is _F32 else code, rows, row, rot, 1 if neox else 0, o, ot, oh)


def rope_compress_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                        kv_cache: torch.Tensor, slot_mapping: torch.Tensor, rot_T_even: torch.Tensor, rot_T_odd: torch.Tensor,
                        k_boundaries: torch.Tensor, v_boundaries: torch.Tensor, neox: bool = True, out_q: torch.Tensor | None = None,
                        rot_block: int | None = None, dense3: bool = False) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and compress key and value into slots of the codebook cache.

    Returns the rotated queries (out_q, which may be query itself; None without query).  The cache's bytes are those of
    compress_store of the rotated fp32 keys and the values in fp32; its arguments are compress_store's.  Slots outside the cache are skipped, and
    a slot is given once.
    """
    from . import _f32, _layout, _rt_block

    dev = _device_index(key, value, query, positions, cos_sin, kv_cache, slot_mapping, out_q)
    out_q, N, H, D, args = _operands(query, key, value, positions, cos_sin, slot_mapping, neox, out_q)
    if kv_cache.dtype != torch.uint8 or kv_cache.dim() != 3 or kv_cache.stride(2) != 1:
        raise ValueError("kv_cache must be a (num_blocks, block_size, total_bytes) uint8 tensor")
    blk = rot_block if rot_block is not None else _rt_block(rot_T_even, rot_T_odd)
    NB, BS, TB = kv_cache.shape
    device = key.device
    kb, vb, even, odd = _f32(k_boundaries, device), _f32(v_boundaries, device), _f32(rot_T_even, device), _f32(rot_T_odd, device)
    if even.shape != (D, D // 2) or odd.shape != (D, D // 2):
        raise ValueError(f"rot_T_even and rot_T_odd must be ({D}, {D // 2})")
    _call(_lib.load().rq_rope_compress_store, "rq_rope_compress_store", dev,
          (*args, _layout(dense3), slot_mapping.data_ptr(), kv_cache.data_ptr(), NB, BS, kv_cache.stride(0), kv_cache.stride(1), TB, even.data_ptr(),
           odd.data_ptr(), blk, kb.data_ptr(), kb.numel(), vb.data_ptr(), vb.numel()))
    return out_q


def rope_q8_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                  kv_cache: torch.Tensor, slot_mapping: torch.Tensor, fmt: str = "int8", neox: bool = True, out_q: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and quantise key and value into slots of the 8-bit cache.

    Returns the rotated queries (out_q, which may be query itself; None without query).  The cache's bytes are those of
    q8_store of the rotated fp32 keys and the values; slots, groups, fmt and workspace are q8_store's.
    """
    dev = _device_index(key, value, query, positions, cos_sin, kv_cache, slot_mapping, out_q, workspace)
    out_q, N, H, D, args = _operands(query, key, value, positions, cos_sin, slot_mapping, neox, out_q)
    NB, BS, stride = _check_cache(kv_cache, H, D)
    code = _format(fmt)
    keep, ws, ws_bytes = _scratch(workspace, _store_bytes(N, NB, BS), kv_cache)
    _call(_lib.load().rq_rope_q8_store, "rq_rope_q8_store", dev,
          (*args, code, slot_mapping.data_ptr(), kv_cache.data_ptr(), NB, BS, stride, ws, ws_bytes))
    return out_q


def rope_kv16_store(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, neox: bool = True,
                    out_q: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate query (N, H_Q, D) and key (N, H, D) by positions (N,), and append key and value to plain 16-bit pages.

    k_cache and v_cache are (num_blocks, block_size, H, D) of key's dtype, fp16 or bf16, contiguous over D (views of one tensor
    of both, or paged_decompress's, as they are).  Returns the rotated queries (out_q, which may be query itself; None without query).
    Slots outside the cache are skipped, and a slot is given once.
    """
    dev = _device_index(key, value, query, positions, cos_sin, k_cache, v_cache, slot_mapping, out_q)
    out_q, N, H, D, args = _operands(query, key, value, positions, cos_sin, slot_mapping, neox, out_q)
    if k_cache.dtype is not key.dtype:
        raise ValueError(f"the pages must be of {key.dtype}, as key is")
    pages = _check_pages(k_cache, v_cache, H, D)
    _call(_lib.load().rq_rope_kv16_store, "rq_rope_kv16_store", dev, (*args, slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *pages))
    return out_q


def _check_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, num_kv_heads: int, head_dim: int) -> tuple:
    """(pages, block_size, strides of both over pages, slots and heads) of plain 16-bit pages; strides over a single one as 0."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not k_cache.dtype:
        raise ValueError("k_cache and v_cache must have the same (num_blocks, block_size, heads, head_dim) shape and dtype")
    NB, BS, H, D = shape
    ks, vs = k_cache.stride(), v_cache.stride()
    if H != num_kv_heads or D != head_dim or ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"the pages must hold {num_kv_heads} heads of {head_dim}, contiguous over head_dim")
    if NB == 1 or BS == 1 or H == 1:
        ks, vs = (tuple(0 if n == 1 else x for n, x in zip(shape, st)) for st in (ks, vs))
    return NB, BS, *ks[:3], *vs[:3]
