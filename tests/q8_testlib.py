"""A plain 64-bit implementation of the 8-bit KV cache (numpy, host): store, read back and attention.

Pages are dicts of numbers here -- codes as values, exponents as ints -- and bytes only where a test
compares them; the byte layout is written down once more, element by element.
"""
from __future__ import annotations

import math

import numpy as np
import torch

GROUP, EMIN, EMAX = 16, -40, 60
LARGEST = {"int8": 127.5, "fp8": 448.0}
CODE_MAX = {"int8": 127.0, "fp8": 448.0}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def slot_bytes(H, D):
    return (H * (2 * D + 1) + 7) // 8 * 8


def e4m3_values():
    """The value of each e4m3 byte (NaN for 0x7f and 0xff)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(b >= 128, -v, v)


_E4M3 = e4m3_values()
_E4M3_POS = _E4M3[:127]  # 0 .. 448, rising


def round_code(fmt, x):
    """The code's value nearest to x, ties to even, clamped; NaN as 0."""
    x = np.where(np.isnan(x), 0.0, x)
    x = np.clip(x, -CODE_MAX[fmt], CODE_MAX[fmt])
    if fmt == "int8":
        return np.rint(x)
    a = np.abs(x)
    i = np.clip(np.searchsorted(_E4M3_POS, a, side="right") - 1, 0, 125)
    lo, hi = _E4M3_POS[i], _E4M3_POS[i + 1]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 1))  # an even byte has an even significand
    return np.where(up, hi, lo) * np.where(np.signbit(x), -1.0, 1.0)


def exponent(fmt, amax):
    e = EMIN
    while amax > LARGEST[fmt] * 2.0 ** e and e < EMAX:
        e += 1
    return e


def code_bytes(fmt, c):
    if fmt == "int8":
        return (c + 128).astype(np.uint8)
    i = np.searchsorted(_E4M3_POS, np.abs(c)).astype(np.uint8)
    return np.where(np.signbit(c), i | 128, i).astype(np.uint8)


def byte_codes(fmt, b):
    return b.astype(np.float64) - 128 if fmt == "int8" else _E4M3[b]


def code_index(block, H, D):
    """Byte of a page that holds (side, slot, head, dim): two int arrays (block, H, D), K's and V's; and the float of a
    page that holds the K scale of (slot, head) (V's is the next one)."""
    t, h, d = np.arange(block)[:, None, None], np.arange(H)[None, :, None], np.arange(D)[None, None, :]
    tile = ((t // GROUP) * H + h) * 2 * GROUP * D
    r = t % GROUP
    k = tile + 1024 * (d // 64) + 256 * ((d // 16) % 4) + 16 * r + d % 16
    v = tile + GROUP * D + 1024 * (d // 64) + 256 * (r // 4) + 16 * (d % 16) + 4 * ((d // 16) % 4) + r % 4
    scale = (block // GROUP * H * 2 * GROUP * D + ((t // GROUP) * H + h)[..., 0] * 16) // 4
    return k, v, scale


class Cache:
    """codes (2, slots, H, D) as numbers and exponents (2, groups, H); None-like exponent -1000: never begun."""

    def __init__(self, pages, block, H, D, fmt):
        self.pages, self.block, self.H, self.D, self.fmt = pages, block, H, D, fmt
        self.codes = np.zeros((2, pages * block, H, D))
        self.exps = np.full((2, pages * block // GROUP, H), -1000)

    def store(self, key, value, slots):
        rows = {}
        for i, s in enumerate(slots):
            if 0 <= s < self.pages * self.block:
                rows[int(s)] = i  # the last one counts
        x = [t.double().numpy() for t in (key, value)]
        for g in sorted({s // GROUP for s in rows}):
            mine = [s for s in rows if s // GROUP == g]
            whole = np.arange(g * GROUP, (g + 1) * GROUP)
            for side in range(2):
                for h in range(self.H):
                    new = {s: x[side][rows[s], h] for s in mine}
                    amax = max(np.max(np.where(np.isfinite(r), np.abs(r), 0.0)) for r in new.values())
                    e, old = exponent(self.fmt, amax), self.exps[side, g, h]
                    if g * GROUP in rows or old == -1000:
                        self.codes[side, whole, h] = 0
                    elif old >= e:
                        e = old
                    else:
                        self.codes[side, whole, h] = round_code(self.fmt, self.codes[side, whole, h] * 2.0 ** float(old - e))
                    for s, r in new.items():
                        self.codes[side, s, h] = round_code(self.fmt, r * 2.0 ** -float(e))
                    self.exps[side, g, h] = e

    def values(self):
        """(K, V): (slots, H, D) each."""
        s = np.where(self.exps == -1000, 0.0, 2.0 ** self.exps.astype(float))
        return self.codes * np.repeat(s, GROUP, axis=1)[..., None]

    def to_bytes(self):
        out = np.zeros((self.pages, self.block * slot_bytes(self.H, self.D)), np.uint8)
        k, v, at = code_index(self.block, self.H, self.D)
        begun = np.repeat(self.exps != -1000, GROUP, axis=1)[..., None]
        for side, idx in enumerate((k, v)):
            b = np.where(begun[side], code_bytes(self.fmt, self.codes[side]), 0)
            out[:, idx.reshape(-1)] = b.reshape(self.pages, -1)
            s = np.where(self.exps[side] == -1000, 0.0, 2.0 ** self.exps[side].astype(float)).astype(np.float32)
            out.view(np.float32)[:, (at + side)[::GROUP].reshape(-1)] = s.reshape(self.pages, -1)
        return out.reshape(self.pages, self.block, -1)


def same_numbers(a, b, fmt):
    """Bytes of two caches, equal but for the sign of an e4m3 zero."""
    if fmt == "fp8":
        a, b = (np.where(x == 128, 0, x) for x in (a, b))
    return np.array_equal(a, b)


def attention(q, kv, table, lens, cu, block, causal=True, sm_scale=None):
    """(out, tolerance) in 64 bits.  q (T, HQ, D) tensor, kv (2, slots, H, D).

    Tolerance of a kernel with exact products, fp32 sums, weights rounded to fp16 and an output rounded once, per element:
      half a step of the output's type of |o|;
      weights: rounded by 2^-11 each, and off by 2 ds, ds = a score's error in fp32: D + 8 roundings of 2^-24 of sum |q k|
        (the sum of D products, then the scaling and the subtraction of the maximum): (2^-11 + 2 ds) sum p |v|;
      weights under fp16's normal range: 2^-25 absolute where the largest is 1 or more: n 2^-25 max |v|.
    """
    q64 = q.double().numpy()
    T, HQ, D = q64.shape
    H = kv.shape[2]
    G = HQ // H
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    out, tol = np.zeros_like(q64), np.zeros_like(q64)
    for b, L in enumerate(lens):
        s0, s1 = int(cu[b]), int(cu[b + 1])
        L = min(int(L), table.shape[1] * block)
        pos = np.arange(max(L, 0))
        slots = table[b, pos // block].astype(np.int64) * block + pos % block
        for i in range(s0, s1):
            n = min(L, int(lens[b]) - (s1 - s0) + (i - s0) + 1) if causal else L
            if n <= 0:
                continue
            for j in range(HQ):
                k, v = kv[0, slots[:n], j // G], kv[1, slots[:n], j // G]
                s = k @ q64[i, j] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                o, a = p @ v, p @ np.abs(v)
                ds = (D + 8) * 2.0 ** -24 * float((np.abs(k) @ np.abs(q64[i, j])).max()) * abs(scale)
                out[i, j] = o
                tol[i, j] = HALF_STEP[q.dtype] * np.abs(o) + (2.0 ** -11 + 2 * ds) * a * (1 + 2.0 ** -8) + n * 2.0 ** -25 * np.abs(v).max()
    return out, tol


def layout(lens, block, seed, spare=3):
    """Random pages for these lengths: (table int32, pages)."""
    rng = np.random.RandomState(seed)
    need = [-(-n // block) for n in lens]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table, at = np.zeros((len(lens), max(need + [1])), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, len(order)


def slots_of(table, b, first, last, block):
    pos = np.arange(first, last)
    return table[b, pos // block].astype(np.int64) * block + pos % block


def rows(n, H, D, seed, dtype, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, n, H, D, generator=g)
    if outliers:
        x[0] *= 1 + (torch.randn(H, D, generator=g) * 3).abs()
    x = x.to(dtype)
    return x[0], x[1]
