"""Attention over the 8-bit cache in 64 bits with a tolerance that small weights count in, and helpers of its GPU tests."""
from __future__ import annotations

import math

import numpy as np
import torch

import q8_testlib as Q
from rotorquant_vllm import kernels as K

DEV = "cuda"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def new_cache(pages, block, H, D, fill=0):
    return torch.full((pages, block, K.q8_slot_bytes(H, D)), fill, dtype=torch.uint8, device=DEV)


def store(cache, ref, k, v, slots, fmt):
    slots = np.asarray(slots, np.int64)
    K.q8_store(k.to(DEV), v.to(DEV), cache, torch.from_numpy(slots).to(DEV), fmt=fmt)
    ref.store(k, v, slots)


def filled(lens, block, H, D, fmt, dtype, seed):
    """(cache on the GPU, reference, table) of sequences of these lengths."""
    table, pages = Q.layout(lens, block, seed)
    ref, cache = Q.Cache(pages, block, H, D, fmt), new_cache(pages, block, H, D)
    k, v = Q.rows(sum(lens), H, D, seed, dtype)
    store(cache, ref, k, v, np.concatenate([Q.slots_of(table, b, 0, n, block) for b, n in enumerate(lens)]), fmt)
    return cache, ref, table


def attention(q, ref, table, lens, cu, causal=True, sm_scale=None):
    """(out, tolerance) in 64 bits; ref: the cache's plain implementation.

    Tolerance of a kernel with exact products, fp32 sums, weights w_j = 2^7 2^(u_j - M) rounded to fp16, u_j the base-2 logarithm of
    p_j 2^e_j (e_j the V exponent of token j's group) and M at most its maximum, and an output rounded once, per element:
      half a step of the output's type of |o|, in fp16 2^-25 at least (its numbers under 2^-14 lie 2^-24 apart);
      weights: rounded by 2^-11 each, and off by 2 ds, ds = a score's error in fp32: D + 8 roundings of 2^-24 of sum |q k|
        (the sum of D products, then the scaling and the subtraction of the maximum): (2^-11 + 2 ds) sum p |v|;
      fp32 sums of n terms: n 2^-24 sum p |v|;
      weights under fp16's normal range: 2^-25 each, in units of 2^7 / max_j p_j 2^e_j: 2^-32 max_j(p_j 2^e_j) sum |c_j|.
    """
    q64 = q.double().numpy()
    T, HQ, D = q64.shape
    kv, G, block = ref.values(), HQ // ref.H, ref.block
    step = np.where(ref.exps[1] == -1000, 0.0, 2.0 ** ref.exps[1].astype(float))  # (groups, H)
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    out, tol = np.zeros_like(q64), np.zeros_like(q64)
    for b, L in enumerate(lens):
        s0, s1 = int(cu[b]), int(cu[b + 1])
        L = min(int(L), table.shape[1] * block)
        pos = np.arange(max(L, 0))
        slots = table[b, pos // block].astype(np.int64) * block + pos % block
        for h in range(ref.H):
            K_, V_, C_, S_ = kv[0, slots, h], kv[1, slots, h], np.abs(ref.codes[1, slots, h]), step[slots // Q.GROUP, h]
            if s1 == s0 or L <= 0:
                continue
            qs = q64[s0:s1, h * G:h * G + G].reshape(-1, D)  # rows: (token, head)
            i = np.repeat(np.arange(s1 - s0), G)
            n = np.clip(int(lens[b]) - (s1 - s0) + i + 1, 0, L) if causal else np.full(len(i), L)
            sees = n > 0
            p = np.where(pos[None] < n[:, None], qs @ K_.T * scale, -np.inf)
            p = np.exp(p - np.where(sees, p.max(axis=1), 0.0)[:, None])
            p /= np.where(sees, p.sum(axis=1), 1.0)[:, None]
            o, a = p @ V_, p @ np.abs(V_)
            ds = (D + 8) * 2.0 ** -24 * abs(scale) * np.where(pos[None] < n[:, None], np.abs(qs) @ np.abs(K_).T, 0.0).max(axis=1)
            codes = np.concatenate([np.zeros((1, D)), np.cumsum(C_, axis=0)])[n]
            t = (np.maximum(Q.HALF_STEP[q.dtype] * np.abs(o), 2.0 ** -25 if q.dtype == torch.float16 else 0.0) + (2.0 ** -11 + 2 * ds + n * 2.0 ** -24)[:, None] * a * (1 + 2.0 ** -8)
                 + 2.0 ** -32 * (p * S_[None]).max(axis=1)[:, None] * codes * (1 + 2.0 ** -8))
            out[s0:s1, h * G:h * G + G], tol[s0:s1, h * G:h * G + G] = o.reshape(-1, G, D), t.reshape(-1, G, D)
    return out, tol


def check(got, out, tol):
    err = np.abs(got.double().cpu().numpy() - out)
    assert (err <= tol).all(), f"off by {float(np.nanmax(err - tol)):.2e} past the tolerance, {int((~(err <= tol)).sum())} elements"
