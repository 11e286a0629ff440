"""Plain implementations, in 64 bits, of position rotation and of attention over plain 16-bit pages (torch, host)."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}  # relative to the value


def gen(seed):
    return torch.Generator().manual_seed(seed)


def table(positions, rot, dtype, base=10000.0):
    """Cosines, then sines, of each position's rot / 2 angles."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))[None, :]
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(dtype)


def pairs(rot, neox):
    """Dims of the first and second member of each pair."""
    i = torch.arange(rot // 2)
    return (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)


def rotate(x, positions, cos_sin, neox, dtype=torch.float64):
    """x (tokens, heads, D) turned, computed in dtype: products, then their sum, as elementary operations.  Positions outside the table: NaN."""
    rot = cos_sin.shape[1]
    a, b = pairs(rot, neox)
    inside = (positions >= 0) & (positions < cos_sin.shape[0])
    row = torch.where(inside[:, None], cos_sin.to(dtype)[positions.clamp(0, cos_sin.shape[0] - 1)], math.nan)[:, None, :]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    x = x.to(dtype)
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def rotation_error(x, positions, cos_sin, neox):
    """Bound on what three roundings to fp32 do to a rotated value: half a step of each product, and of their sum."""
    rot = cos_sin.shape[1]
    a, b = pairs(rot, neox)
    c, s = (y[:, None, :] for y in cos_sin.double()[positions].abs().chunk(2, dim=-1))
    x = x.double().abs()
    e = torch.zeros_like(x)
    e[..., a] = x[..., a] * c + x[..., b] * s
    e[..., b] = x[..., b] * c + x[..., a] * s
    return e * (2.01 * 2.0 ** -24) + 2.0 ** -148  # (each product once, their sum once; subnormals)


def attention(q, k, v, lens, q_lens, scale=None, causal=True):
    """Rows of q (tokens, H_Q, D) over each sequence's K and V (lists of (length, H, D)): (results in 64 bits, bound on the error of one with
    exact products, fp32 sums, base-2 exponentials good to 2^-21 and weights of 16 bits or more, before its rounding)."""
    T, HQ, D = q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, err, at = torch.zeros(T, HQ, D, dtype=torch.float64), torch.zeros(T, HQ, D, dtype=torch.float64), 0
    for b, (L, n) in enumerate(zip(lens, q_lens)):
        H = k[b].shape[1]
        for i in range(n):
            end = min(L, L - n + i + 1) if causal else L
            if end <= 0:
                at += 1
                continue
            for j in range(HQ):
                kk, vv, qq = k[b][:end, j // (HQ // H)].double(), v[b][:end, j // (HQ // H)].double(), q[at, j].double()
                s = kk @ qq * scale
                p = torch.softmax(s, dim=0)
                out[at, j] = p @ vv
                # a sum of D exact products in any order: D roundings of at most the sum of magnitudes; the score times its factor, and less the maximum
                ds = abs(scale) * (D + 2) * 2.0 ** -24 * (kk.abs() @ qq.abs()) + 4 * 2.0 ** -24 * s.abs().max()
                # weights: off by twice that, 2^-21 (the exponential, 2^-23, and the additions of 14 before it) and 2^-16 (their two 16-bit parts), or by
                # 2^-38 of the largest where fp16 ends; sums of 32 products and the running sum, twice a tile, and of the waves and
                # workgroups, above and below the fraction
                rel = 2 * ds.max() + 2.0 ** -16 + 2.0 ** -21 + (120 + end / 8) * 2.0 ** -24
                err[at, j] = rel * (p @ vv.abs()) + end * 2.0 ** -38 * p.max() * vv.abs().max()
            at += 1
    return out, err


def check(got, out, err):
    """got within err and half a step of its type."""
    step = torch.finfo(got.dtype).smallest_normal * HALF_STEP[got.dtype] * 2  # (of subnormals)
    bound = out.abs() * HALF_STEP[got.dtype] * 1.0001 + err * 1.01 + step
    off = (got.double().cpu() - out).abs()
    assert bool(torch.isfinite(got).all()), "not finite"
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} more than the bound"


class Pages:
    """Random contexts in pages of shuffled order; what lies behind a context (and in pages of none) is `rubbish`."""

    def __init__(self, lens, block, H, D, dtype, seed, rubbish=math.nan, spare=3, layout="two"):
        rng, g = np.random.RandomState(seed), gen(seed)
        need = [-(-n // block) for n in lens]
        order = rng.permutation(sum(need) + spare).astype(np.int32)
        self.table = np.full((len(lens), max(max(need), 1)), -5, np.int32)
        shape = (2, len(order), block, H, D) if layout == "two" else (len(order), 2, block, H, D) if layout == "paired" else (len(order), H, block, 2, D)
        both = torch.full(shape, rubbish, dtype=dtype)
        view = {"two": lambda x: (x[0], x[1]), "paired": lambda x: (x[:, 0], x[:, 1]),
                "heads": lambda x: (x[:, :, :, 0].transpose(1, 2), x[:, :, :, 1].transpose(1, 2))}[layout]
        self.both, self.view, self.kv, at = both, view, ([], []), 0
        strong = 1 + (torch.randn(H, D, generator=g) * 3).abs()
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            for side, cache in enumerate(view(both)):
                x = (torch.randn(n, H, D, generator=g) * (strong if side == 0 else 1)).to(dtype)
                pos = torch.arange(n)
                cache[torch.from_numpy(self.table[b].astype(np.int64))[pos // block], pos % block] = x
                self.kv[side].append(x)

    def to(self, device):
        return self.view(self.both.to(device))
