"""Op-level API of the 8-bit KV cache: write (q8_store), read back (q8_read), attention (q8_attention).

The cache is a (num_blocks, block_size, q8_slot_bytes(num_kv_heads, head_dim)) uint8 tensor whose
pages hold K and V as int8 or e4m3 codes (fmt "int8" or "fp8") with a power-of-two scale for each
group of 16 consecutive slots, kv head and side; include/rq_abi.h defines the bytes.  head_dim 64 or 128,
block_size a multiple of 16.  No counterpart in the reference, whose codecs stop at 4 bits.

As everywhere in this package, tensors are on one ROCm device and there is no CPU path; calls run on the
current stream of that device, whichever device is current, and are safe on several
streams at once (scratch comes from torch's allocator unless passed).
"""
from __future__ import annotations

import functools
import math

import torch

from .. import _lib

__all__ = ["q8_slot_bytes", "q8_store", "q8_read", "q8_attention"]

_FORMATS = {"int8": 0, "fp8": 1}


def _format(fmt: str) -> int:
    try:
        return _FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"fmt must be 'int8' or 'fp8', got {fmt!r}") from None


# Calls of a few microseconds wait for the checks below: device indices and plain comparisons, no device objects, and each
# tensor's sizes and strides fetched once.

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # (0.06 against 0.24 us)


def _device_index(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """Index of the device that all tensors are on."""
    dev = first.get_device()
    for t in others if dev >= 0 else (first,):
        if dev < 0 or t is not None and t.get_device() != dev:
            if not (first.is_cuda and t.is_cuda):
                raise RuntimeError("rotorquant_vllm.kernels runs only on ROCm device tensors (got a "
                                   f"{(t if first.is_cuda else first).device.type} tensor); there is no CPU path")
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return dev


def _call(fn, name: str, dev: int, args: tuple) -> None:
    """fn(*args, stream): a launch goes to the current device's context, so the tensors' own is made current."""
    if _current_device() == dev:
        rc = fn(*args, _lib.stream_ptr(torch.device("cuda", dev)) if _lib._raw_stream is None else _lib._raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream_ptr(torch.device("cuda", dev)))
    if rc:
        _lib.check(rc, name)


def q8_slot_bytes(num_kv_heads: int, head_dim: int) -> int:
    """Bytes of a cache slot: the last dimension of the cache tensor (2056 for 8 heads of 128)."""
    return -(-num_kv_heads * (2 * head_dim + 1) // 8) * 8


def _check_cache(kv_cache: torch.Tensor, num_kv_heads: int, head_dim: int) -> tuple[int, int, int]:
    """(pages, block_size, bytes between pages) of an 8-bit cache."""
    shape = kv_cache.shape
    if kv_cache.dtype != torch.uint8 or len(shape) != 3:
        raise ValueError("kv_cache must be a (num_blocks, block_size, q8_slot_bytes) uint8 tensor")
    NB, BS, SB = shape
    if SB < num_kv_heads * (2 * head_dim + 1):
        raise ValueError(f"cache slots of {SB} bytes; {num_kv_heads} heads of {head_dim} take {q8_slot_bytes(num_kv_heads, head_dim)}")
    page, slot, byte = kv_cache.stride()
    if byte != 1 or slot != SB:
        raise ValueError("the slots of a page must be contiguous")
    return NB, BS, page


def _row_strides(shape, strides) -> tuple:
    """Strides of calls with one token or one head: that over a single one, which may be any number in a view, as 0."""
    return (strides[0] if shape[0] > 1 else 0, strides[1] if shape[1] > 1 else 0, strides[2])


def _index(t: torch.Tensor, name: str, dtype: torch.dtype, dim: int) -> torch.Tensor:
    if t.dtype != dtype or t.dim() != dim:
        raise ValueError(f"{name} must be a {dim}-dimensional {dtype} tensor, got {t.dim()} dimensions of {t.dtype}")
    return t if t.is_contiguous() or t.stride(-1) == 1 else t.contiguous()


# Sizes of scratch, by sizes alone (0.1 against 0.5 us a call).
@functools.lru_cache(maxsize=4096)
def _store_bytes(n_tokens: int, num_blocks: int, block_size: int) -> int:
    return _lib.load().rq_q8_store_workspace_bytes(n_tokens, num_blocks, block_size)


# (The attention's also by the GPU, whose number of CUs sizes the partial sums: asked for with that one current.)
@functools.lru_cache(maxsize=4096)
def _attention_bytes(dev: int, num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int, max_q_len: int, max_seq_len: int) -> int:
    with torch.cuda.device(dev):
        return _lib.load().rq_q8_attention_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, max_seq_len)


def _scratch(workspace: torch.Tensor | None, need: int, like: torch.Tensor) -> tuple[torch.Tensor | None, int, int]:
    """(tensor to keep, address, bytes) of the caller's buffer, or of one of this call from the stream's allocator."""
    if workspace is None:
        if not need:
            return None, 0, 0
        workspace = torch.empty(need, dtype=torch.uint8, device=like.device)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor")
    return workspace, workspace.data_ptr(), workspace.numel()


def q8_store(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor, fmt: str = "int8",
             workspace: torch.Tensor | None = None) -> None:
    """Quantise key / value (N, H, D) fp16, bf16 or fp32 into the slots slot_mapping[:N] of an 8-bit cache.

    Slots outside the cache (vLLM's padding id -1) are skipped; of tokens with the same slot the last one counts.
    A write of a group's first slot begins the group anew (its rows that this call does not write
    become 0); other writes keep its rows and never lower its scale.  A store reads and writes whole groups: stores to one
    group, and reads of it, on several streams have to be ordered by the caller.
    Rows (and the cache) start at multiples of 16 bytes, as slices of a fused projection do; others are refused.
    workspace: scratch of calls of more than 512 tokens (rq_q8_store_workspace_bytes bytes),
    by default from torch's allocator; a graph captured without torch's graph classes needs it.
    """
    dev = _device_index(key, value, kv_cache, slot_mapping, workspace)
    shape = key.shape
    if len(shape) != 3 or value.shape != shape or value.dtype != key.dtype:
        raise ValueError("key and value must have the same (tokens, heads, head_dim) shape and dtype")
    N, H, D = shape
    ks, vs = key.stride(), value.stride()
    if N == 1 or H == 1:
        ks, vs = _row_strides(shape, ks), _row_strides(shape, vs)
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("key/value must be contiguous over head_dim")
    NB, BS, stride = _check_cache(kv_cache, H, D)
    sm = _index(slot_mapping, "slot_mapping", torch.int64, 1)
    if sm.numel() < N:
        raise ValueError("slot_mapping shorter than the number of tokens")
    code = _format(fmt)
    keep, ws, ws_bytes = _scratch(workspace, _store_bytes(N, NB, BS), kv_cache)
    _call(_lib.load().rq_q8_store, "rq_q8_store", dev,
          (key.data_ptr(), value.data_ptr(), _lib.dtype_code(key.dtype), N, ks[0], ks[1], vs[0], vs[1], H, D, code, sm.data_ptr(), kv_cache.data_ptr(), NB, BS, stride, ws, ws_bytes))


def q8_read(kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, starts: torch.Tensor, num_kv_heads: int,
            head_dim: int, dtype: torch.dtype, fmt: str = "int8", out_k: torch.Tensor | None = None, out_v: torch.Tensor | None = None,
            total: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of a batch's contexts as plain rows, (total, H, D) each: token i of sequence b in row starts[b] + i.

    block_table (num_seqs, max_blocks), seq_lens (num_seqs,) and starts (num_seqs or num_seqs + 1, rising by
    at least each length) are int32.  out_k / out_v: buffers to fill, whose rows of no sequence stay as they are;
    without them `total` rows are allocated (rows of no sequence are then not initialised).
    The layout is that of variable-length attention over plain K and V.
    """
    dev = _device_index(kv_cache, block_table, seq_lens, starts, out_k, out_v)
    NB, BS, stride = _check_cache(kv_cache, num_kv_heads, head_dim)
    bt = _index(block_table, "block_table", torch.int32, 2)
    sl, st = _index(seq_lens, "seq_lens", torch.int32, 1), _index(starts, "starts", torch.int32, 1)
    B, max_blocks = bt.shape
    if sl.numel() < B or st.numel() < B:
        raise ValueError("block_table, seq_lens and starts differ in the number of sequences")
    code = _format(fmt)
    if total is None:
        if out_k is None and out_v is None:
            raise ValueError("total (the number of rows) is needed without out_k and out_v")
        total = (out_v if out_k is None else out_k).shape[0]
    shape = (total, num_kv_heads, head_dim)
    for t in (out_k, out_v):
        if t is not None and (t.shape != shape or t.dtype != dtype or not t.is_contiguous()):
            raise ValueError(f"outputs must be contiguous {shape} tensors of {dtype}")
    out_k = torch.empty(shape, dtype=dtype, device=kv_cache.device) if out_k is None else out_k
    out_v = torch.empty(shape, dtype=dtype, device=kv_cache.device) if out_v is None else out_v
    _call(_lib.load().rq_q8_read, "rq_q8_read", dev,
          (kv_cache.data_ptr(), NB, BS, stride, num_kv_heads, head_dim, code, bt.data_ptr(), max_blocks, bt.stride(0), sl.data_ptr(),
           st.data_ptr(), B, total, out_k.data_ptr(), out_v.data_ptr(), _lib.dtype_code(dtype)))
    return out_k, out_v


def q8_attention(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, num_kv_heads: int,
                 head_dim: int, fmt: str = "int8", sm_scale: float | None = None, causal: bool = True,
                 cu_seqlens_q: torch.Tensor | None = None, max_q_len: int | None = None, max_seq_len: int | None = None,
                 out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new query tokens q (num_tokens, H_Q, D) fp16 or bf16 over an 8-bit cache.

    block_table (num_seqs, max_blocks) and seq_lens (num_seqs,), the contexts with the new tokens
    included, are int32.  cu_seqlens_q (num_seqs + 1,) int32 splits q among the sequences; without it each has one token
    (a decode step).  Query i of sequence b sits at position seq_lens[b] - q_len_b + i; a row that sees no key is zeros.
    max_q_len and max_seq_len: host ints that bound the query and context lengths (default: all of q, and the
    block table's capacity); what lies past them is not read, and positions stay as above.  out: a buffer to fill, whose
    rows of such tokens and of no sequence stay as they are (without it they are not initialised).
    Rows of q start at multiples of 16 bytes and those of out of 8; others are refused.
    workspace: scratch (rq_q8_attention_workspace_bytes bytes), by default of this call from torch's allocator; a graph
    captured without torch's graph classes needs it, since nothing else keeps the scratch for its replays.
    """
    shape = q.shape
    if len(shape) != 3 or shape[2] != head_dim or num_kv_heads < 1 or shape[1] % num_kv_heads:
        raise ValueError(f"q must be (tokens, a multiple of {num_kv_heads} heads, {head_dim}), got {tuple(shape)}")
    dev = _device_index(q, kv_cache, block_table, seq_lens, cu_seqlens_q, out, workspace)
    NB, BS, stride = _check_cache(kv_cache, num_kv_heads, head_dim)
    bt = _index(block_table, "block_table", torch.int32, 2)
    sl = _index(seq_lens, "seq_lens", torch.int32, 1)
    T, HQ, D = shape
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
    out = torch.empty_like(q) if out is None else out
    os = out.stride()
    if out.shape != shape or out.dtype != q.dtype or os[2] != 1:
        raise ValueError("out must have q's shape and dtype and be contiguous over head_dim")
    if T == 1 or HQ == 1:
        qs, os = _row_strides(shape, qs), _row_strides(shape, os)
    capacity = max_blocks * BS
    max_seq_len = capacity if max_seq_len is None else min(int(max_seq_len), capacity)
    code = _format(fmt)
    keep, ws, ws_bytes = _scratch(workspace, _attention_bytes(dev, B, HQ, num_kv_heads, D, max_q_len, max_seq_len), q)
    _call(_lib.load().rq_q8_attention, "rq_q8_attention", dev,
          (q.data_ptr(), _lib.dtype_code(q.dtype), T, HQ, qs[0], qs[1], None if cu is None else cu.data_ptr(), B, max_q_len,
           1 if causal else 0, kv_cache.data_ptr(), NB, BS, stride, num_kv_heads, D, code, bt.data_ptr(), max_blocks, bt.stride(0),
           sl.data_ptr(), max_seq_len, 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), out.data_ptr(), os[0],
           os[1], ws, ws_bytes))
    return out
