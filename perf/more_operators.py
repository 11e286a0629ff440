"""Timing cases of a layer's step around the KV cache: position rotation on the way into it, and attention over plain pages.

A new token's queries and keys are rotated by its position (rotary embedding, from a table of cosines and sines) and its keys and
values appended to a paged cache, in one operator for each of the cache's formats:

"kv16"  plain 16-bit pages, K and V (pages, block, heads, head_dim) each;
"q8"    the 8-bit cache: codes with a power-of-two scale for each 16 tokens, head and side (K or V);
"rq"    the codebook cache: norm, rotation by small blocks, 3- or 4-bit indices of the nearest centroids.

Each returns the rotated queries and what the touched pages then hold, as values.  "attend" is attention of one new token, or
a draft's few, over plain 16-bit pages.

Pairs of dims are (i, i + rot / 2) ("halves") or (2 i, 2 i + 1) ("pairs"), rot the rotated dims of a head; in fp32, y1 = x1 cos - x2 sin and
y2 = x2 cos + x1 sin, each product and the sum rounded once.

Shapes are those of bench.py and the tests: head_dim 128 and 64 (96, 80 and 256 beside them, for pages of other models), pages of 16 to 64
tokens, 1 to 8 kv heads, 1 to 16 query heads per kv head, contexts of 1 to 32768 tokens.  Keys carry strong channels (a scale of
1 + |N(0, 3)| per head and channel); values and queries are N(0, 1).  Pages are in random order, as after some hours of serving.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

GROUP = 16         # tokens that share a scale of the 8-bit cache
POSITIONS = 40960  # rows of the table of angles
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
LARGEST = {"int8": 127.5, "fp8": 448.0}
# The centroids of least squared error for N(0, 1) (Max 1960), the positive half.
CENTROIDS = {3: [0.2451, 0.7560, 1.3439, 2.1520], 4: [0.1284, 0.3881, 0.6568, 0.9424, 1.2562, 1.6181, 2.0690, 2.7326]}


def listed():
    common = {"dtype": "bfloat16", "heads": 8, "group": 4, "head_dim": 128, "block": 16}
    rope = dict(common, table="float32", style="halves", rot=128, padded=0)
    return [
        # one decode step of 16 sequences behind contexts that end inside a page: the smallest call
        dict(rope, name="kv16_step", kind="kv16", seqs=16, queries=1, shortest=100, longest=30000),
        # a full batch of prompts
        dict(rope, name="kv16_prompts", kind="kv16", seqs=8, queries=4096, shortest=0, longest=0, table="bfloat16"),
        # drafts of a captured batch with padding, a quarter of the dims rotated in pairs
        dict(rope, name="kv16_drafts", kind="kv16", seqs=96, queries=5, shortest=20, longest=9000, padded=32, dtype="float16", heads=4, group=7,
             head_dim=64, style="pairs", rot=16, block=32),
        # one decode step of a serving batch into the 8-bit cache
        dict(rope, name="q8_step", kind="q8", seqs=64, queries=1, shortest=100, longest=30000, format="int8"),
        # prompt chunks of odd lengths behind a prefix, e4m3 codes
        dict(rope, name="q8_chunks", kind="q8", seqs=7, queries=1501, shortest=5, longest=8000, format="fp8", dtype="float16", table="float16", block=32),
        # one decode step into the codebook cache, 3 bits
        dict(rope, name="rq_step", kind="rq", seqs=64, queries=1, shortest=100, longest=30000, k_bits=3, v_bits=3, rot_block=4),
        # a full batch of prompts, 4-bit keys and 3-bit values, 2 x 2 rotations
        dict(rope, name="rq_prompts", kind="rq", seqs=8, queries=4096, shortest=0, longest=0, k_bits=4, v_bits=3, rot_block=2, table="bfloat16"),
        # one user's decode step: latency and launches
        dict(common, name="attend_one", kind="attend", seqs=1, shortest=777, longest=777, queries=1),
        # a serving batch of decodes (32 query / 8 kv heads)
        dict(common, name="attend_batch", kind="attend", seqs=64, shortest=1024, longest=8192, queries=1),
        # few long contexts (28 query / 4 kv heads)
        dict(common, name="attend_long", kind="attend", seqs=4, shortest=20000, longest=32768, queries=1, heads=4, group=7, dtype="float16", block=64),
        # drafts of up to 8 tokens verified over their contexts
        dict(common, name="attend_drafts", kind="attend", seqs=32, shortest=600, longest=8000, queries=8),
        # heads of 256, 16 query heads on one kv head
        dict(common, name="attend_256", kind="attend", seqs=24, shortest=300, longest=6000, queries=1, heads=1, group=16, head_dim=256, block=32),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    heads, group = rng.choice([(8, 4), (8, 4), (4, 7), (4, 8), (2, 4), (1, 4), (8, 1), (2, 7), (1, 8), (4, 2), (1, 16)])
    c = {"dtype": rng.choice(["bfloat16", "bfloat16", "float16"]), "heads": heads, "group": group, "block": rng.choice([16, 16, 32, 64])}
    kind = rng.choice(["kv16", "kv16", "q8", "q8", "rq", "rq", "attend", "attend", "attend", "attend"])
    c["kind"] = kind
    if kind == "attend":
        c["head_dim"] = rng.choice([128, 128, 64, 96, 80, 256])
        longest = log(1, 32768)
        c.update(longest=longest, shortest=max(1, int(longest * rng.choice([0.1, 0.5, 0.9]))), queries=rng.choice([1, 1, 1, rng.randint(2, 12)]))
        most = (300000 if c["queries"] == 1 else 100000) * 1024 // max(1024, heads * c["head_dim"])
        c["seqs"] = max(1, min(log(1, 128), most // longest))
        return c
    c["head_dim"] = rng.choice([128, 128, 64]) if kind != "kv16" else rng.choice([128, 128, 64, 96, 256])
    c["rot"] = rng.choice([c["head_dim"], c["head_dim"], c["head_dim"] // 2, 16])
    c.update(style=rng.choice(["halves", "halves", "pairs"]), table=rng.choice(["float32", c["dtype"]]))
    if kind == "q8":
        c["format"] = rng.choice(["int8", "fp8"])
    if kind == "rq":
        c["head_dim"], c["rot_block"] = 128, rng.choice([4, 4, 2])
        c["rot"] = rng.choice([128, 128, 64, 16])
        c["k_bits"], c["v_bits"] = rng.choice([(3, 3), (4, 4), (4, 3)])
    if rng.random() < 0.5:  # decode steps and drafts
        c.update(seqs=log(1, 512), queries=rng.choice([1, 1, rng.randint(2, 12)]), padded=rng.choice([0, 0, rng.randint(1, 40)]), shortest=0,
                 longest=log(1, 30000))
    else:
        queries = log(1, 4096)
        c.update(seqs=max(1, min(log(1, 64), 16384 // queries)), queries=queries, padded=0, shortest=0, longest=rng.choice([0, log(1, 20000)]))
    return c


# ---------------------------------------------------------------------------
# Position rotation, in plain torch
# ---------------------------------------------------------------------------

def _pairs(case, x):
    """The first and second dims of the rotated pairs of x (..., head_dim): views."""
    r = case["rot"]
    return (x[..., :r // 2], x[..., r // 2:r]) if case["style"] == "halves" else (x[..., 0:r:2], x[..., 1:r:2])


def _rotate(case, x, rows):
    """x (tokens, heads, head_dim) rotated by the table's rows (tokens, rot), in the type of both."""
    c, s = (y[:, None, :] for y in rows.chunk(2, dim=-1))
    x1, x2 = _pairs(case, x)
    out = x.clone()
    y1, y2 = _pairs(case, out)
    y1.copy_(x1 * c - x2 * s)
    y2.copy_(x2 * c + x1 * s)
    return out


# ---------------------------------------------------------------------------
# The caches, in plain torch
# ---------------------------------------------------------------------------

def _q8_slot_bytes(case):
    return -(-case["heads"] * (2 * case["head_dim"] + 1) // 8) * 8


def _q8_sides(case, cache):
    """Views of an 8-bit cache (pages, block, slot bytes): codes (pages, groups, heads, K or V, 16 D) and the groups' scales
    (pages, groups, heads, K or V)."""
    P, n, H, D = cache.shape[0], case["block"] // GROUP, case["heads"], case["head_dim"]
    flat = cache.view(P, -1)
    end = n * H * 2 * GROUP * D
    return flat[:, :end].view(P, n, H, 2, GROUP * D), flat[:, end:end + n * H * 16].view(torch.float32).view(P, n, H, 4)[..., :2]


def _q8_decode(case, codes):
    """Codes (..., K or V, 16 D) in the cache's order -> their values (..., K or V, 16, D), fp32, without the scale."""
    D = case["head_dim"]
    v = codes.float() - 128 if case["format"] == "int8" else codes.view(torch.float8_e4m3fn).float()
    lead = v.shape[:-2]
    # K: [64-dim chunk][16-dim part][token][dim]; V: [chunk][token / 4][dim][16-dim part][token % 4]
    k = v[..., 0, :].reshape(*lead, D // 64, 4, 16, 16).movedim(-2, -4).reshape(*lead, GROUP, D)
    w = v[..., 1, :].reshape(*lead, D // 64, 4, 16, 4, 4).movedim((-4, -1), (-5, -4)).transpose(-1, -2).reshape(*lead, GROUP, D)
    return torch.stack([k, w], dim=-3)


def _q8_encode(case, v):
    """The inverse of _q8_decode for values that are codes."""
    D, lead = case["head_dim"], v.shape[:-3]
    b = (v + 128).to(torch.uint8) if case["format"] == "int8" else v.to(torch.float8_e4m3fn).view(torch.uint8)
    k = b[..., 0, :, :].reshape(*lead, 16, D // 64, 4, 16).movedim(-4, -2)
    w = b[..., 1, :, :].reshape(*lead, 4, 4, D // 64, 4, 16).transpose(-1, -2).movedim((-5, -4), (-4, -1))
    return torch.stack([k.reshape(*lead, 16 * D), w.reshape(*lead, 16 * D)], dim=-2)


def _q8_exponent(case, amax):
    m, e = torch.frexp(amax)  # m in [0.5, 1)
    m127, e127 = math.frexp(LARGEST[case["format"]])
    return torch.where(amax > 0, e - e127 + (m > m127).to(e.dtype), -40).clamp(-40, 60)


def _q8_write(case, cache, slots, kv):
    """Stores the tokens kv (n, K or V, heads, D), fp32, at slots (n).  A group's first slot begins it anew."""
    codes, scales = (x.flatten(0, 1) for x in _q8_sides(case, cache))  # of every group
    at, inverse = torch.unique(slots // GROUP, return_inverse=True)
    rows = torch.zeros(at.numel(), GROUP, *kv.shape[1:], device=kv.device)
    rows[inverse, slots % GROUP] = kv
    new = torch.zeros(at.numel(), GROUP, dtype=torch.bool, device=kv.device)
    new[inverse, slots % GROUP] = True
    rows = rows.permute(0, 3, 2, 1, 4)  # (groups, heads, K or V, 16, D)
    e = _q8_exponent(case, rows.abs().amax(dim=(-1, -2)))
    old_scale = scales[at]
    begun = (~new[:, 0])[:, None, None] & (old_scale > 0)
    old_e = torch.where(begun, torch.frexp(old_scale)[1] - 1, -40)
    e = torch.maximum(e, old_e)
    old = torch.where(begun[..., None, None], _q8_decode(case, codes[at]), torch.zeros((), device=kv.device))
    x = torch.where(new[:, None, None, :, None], torch.ldexp(rows, -e[..., None, None]), torch.ldexp(old, (old_e - e)[..., None, None]))
    c = x.round().clamp(-127, 127) if case["format"] == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    pages, part = at // (case["block"] // GROUP), at % (case["block"] // GROUP)
    all_codes, all_scales = _q8_sides(case, cache)
    all_codes[pages, part] = _q8_encode(case, c)
    all_scales[pages, part] = torch.ldexp(torch.ones((), device=kv.device), e)


def _q8_values(case, cache):
    """K and V of every slot: fp32 (K or V, slots, heads, D)."""
    codes, scales = _q8_sides(case, cache)
    v = _q8_decode(case, codes) * scales[..., None, None]  # (pages, groups, heads, 2, 16, D)
    return v.permute(3, 0, 1, 4, 2, 5).flatten(1, 3)


def _rq_book(case, side):
    """(centroids, boundaries) of a side's codebook, for rows of norm 1."""
    half = CENTROIDS[case["k_bits"] if side == 0 else case["v_bits"]]
    c = torch.tensor([-x for x in reversed(half)] + half, dtype=torch.float64) / math.sqrt(case["head_dim"])
    c = c.float()
    return c.to(_dev()), ((c[1:].double() + c[:-1].double()) / 2).float().to(_dev())


def _rq_blocks(case, seed):
    """The diagonal blocks of the rotation: (head_dim / w, w, w) for width w, fp32."""
    n, w = case["head_dim"] // case["rot_block"], case["rot_block"]
    x = torch.randn(n, w, generator=_gen(seed, 3), device=_dev(), dtype=torch.float64)
    x = x / x.square().sum(dim=-1, keepdim=True).sqrt()
    if w == 2:
        return torch.stack([torch.stack([x[:, 0], -x[:, 1]], dim=-1), torch.stack([x[:, 1], x[:, 0]], dim=-1)], dim=-2).float()
    a, b, c, d = x.unbind(-1)  # the matrix of v -> q v
    rows = [[a, -b, -c, -d], [b, a, -d, c], [c, d, a, -b], [d, -c, b, a]]
    return torch.stack([torch.stack(r, dim=-1) for r in rows], dim=-2).float()


def _chain(total, x, y):
    """x y added to a running fp32 sum, rounded once."""
    return (total.double() + x.double() * y.double()).float()


def _rq_codes(case, x, blocks, bounds):
    """Rows x (..., D), fp32 -> (indices, norms).  The squares are summed in eight interleaved sums and then those in order, and a block's products in
    order, each step rounded to fp32: the cache's own definition, since an index on a border goes by the last bit."""
    D, w = case["head_dim"], case["rot_block"]
    parts = x.reshape(*x.shape[:-1], D // 8, 8)
    sums = torch.zeros_like(parts[..., 0, :])
    for k in range(D // 8):
        sums = _chain(sums, parts[..., k, :], parts[..., k, :])
    total = sums[..., 0]
    for k in range(1, 8):
        total = total + sums[..., k]
    norm = total.double().sqrt().float()
    unit = (x.double() / (norm + 1e-10).double()[..., None]).float().reshape(*x.shape[:-1], D // w, w)
    turned = (unit[..., :1].double() * blocks[:, :, 0].double()).float()
    for k in range(1, w):
        turned = _chain(turned, unit[..., k:k + 1], blocks[:, :, k])
    turned = turned.reshape(x.shape)
    index = torch.zeros_like(turned, dtype=torch.uint8)
    for b in bounds:
        index += b < turned
    return index, norm


def _rq_slot_bytes(case):
    per_head = case["head_dim"] + 8  # nibbles and a norm, of K and V
    return case["heads"] * (1 << (per_head - 1).bit_length())


def _rq_sides(case, cache):
    """Views of a codebook cache: nibbles (slots, K or V, heads, D / 2) and norms (slots, K or V, heads)."""
    H, half = case["heads"], case["head_dim"] // 2
    flat = cache.view(-1, cache.shape[-1])[:, :2 * H * (half + 4)].view(-1, 2, H * (half + 4))
    return flat[..., :H * half].unflatten(-1, (H, half)), flat[..., H * half:].unflatten(-1, (H, 4))


def _rq_write(case, cache, slots, kv, blocks):
    nibbles, norms = _rq_sides(case, cache)
    for side in range(2):
        index, norm = _rq_codes(case, kv[:, side], blocks, _rq_book(case, side)[1])
        nibbles[slots, side] = index[..., 0::2] << 4 | index[..., 1::2]
        norms[slots, side] = norm.contiguous()[..., None].view(torch.uint8)


def _rq_values(case, cache):
    """K and V of every slot before the rotation is undone: fp32 (K or V, slots, heads, D)."""
    nibbles, norms = _rq_sides(case, cache)
    index = torch.stack([nibbles >> 4, nibbles & 15], dim=-1).flatten(-2).long()
    norm = norms.contiguous().view(torch.float32)
    return torch.stack([_rq_book(case, side)[0][index[:, side]] * norm[:, side] for side in range(2)])


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _dev():
    return torch.device("cuda")


def _gen(seed, stream):
    return torch.Generator(device=_dev()).manual_seed(1000 * int(seed) + stream)


def _i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=_dev())


def _table(case):
    """Cosines and sines of each position's angles, in the table's type."""
    half = case["rot"] // 2
    position, i = (torch.arange(n, dtype=torch.float64, device=_dev()) for n in (POSITIONS, half))
    angle = position[:, None] * 10000.0 ** (-i / half)[None, :]
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(DTYPES[case["table"]])


def _tokens(case, n, seed, stream):
    """n tokens' K and V: (n, K or V, heads, D)."""
    H, D = case["heads"], case["head_dim"]
    x = torch.randn(n, 2, H, D, generator=_gen(seed, stream), device=_dev())
    x[:, 0] *= 1 + (torch.randn(H, D, generator=_gen(seed, 2), device=_dev()) * 3).abs()
    return x.to(DTYPES[case["dtype"]])


def _held(case):
    """Tokens of each sequence before the call: part of the case, they do not change with its data."""
    return np.random.RandomState(4).randint(case["shortest"], case["longest"] + 1, case["seqs"])


def _prepare_append(case, seed):
    H, D, block, n = case["heads"], case["head_dim"], case["block"], case["queries"]
    held, dtype = _held(case), DTYPES[case["dtype"]]
    first, last = held // block, (held + n - 1) // block  # the pages that the new tokens are in
    pages = int((last - first + 1).sum()) + 3
    order = np.random.RandomState(1000 * int(seed) % (1 << 31) + 5).permutation(pages).astype(np.int64)
    old, slots, positions, begin = [], [], [], 0
    for h, f, e in zip(held, first, last):
        mine = order[begin:begin + e - f + 1]
        begin += e - f + 1
        at = np.arange(f * block, h + n)
        at = mine[at // block - f] * block + at % block
        old.append(at[:h - f * block])
        slots.append(at[h - f * block:])
        positions.append(np.arange(h, h + n))
    slots.append(np.full(case["padded"], -1))
    positions.append(np.zeros(case["padded"], np.int64))
    old, slots, positions = (torch.from_numpy(np.concatenate(x).astype(np.int64)).to(_dev()) for x in (old, slots, positions))
    kv, before = _tokens(case, slots.numel(), seed, 10), _tokens(case, old.numel(), seed, 11).float()
    s = {"case": case, "slots": slots, "positions": positions, "table": _table(case), "k": kv[:, 0].contiguous(), "v": kv[:, 1].contiguous(),
         "q": torch.randn(slots.numel(), H * case["group"], D, generator=_gen(seed, 6), device=_dev()).to(dtype)}
    s["out_q"] = torch.zeros_like(s["q"])
    if case["kind"] == "kv16":
        s["cache"] = torch.zeros(2, pages, block, H, D, dtype=dtype, device=_dev())
        s["cache"].view(2, -1, H, D)[:, old] = before.transpose(0, 1).to(dtype)
        return s
    # every page, in order, as one context: what the pages hold is read back that way
    s["all"], s["all_lens"] = _i32(np.arange(pages))[None], _i32([pages * block])
    s["back"] = [torch.zeros(pages * block, H, D, dtype=dtype, device=_dev()) for _ in range(2)]
    if case["kind"] == "q8":
        s["cache"] = torch.zeros(pages, block, _q8_slot_bytes(case), dtype=torch.uint8, device=_dev())
        s["starts"] = _i32([0, pages * block])
        if old.numel():
            _q8_write(case, s["cache"], old, before)
        return s
    s["cache"] = torch.zeros(pages, block, _rq_slot_bytes(case), dtype=torch.uint8, device=_dev())
    s["blocks"] = _rq_blocks(case, seed)
    turn = torch.block_diag(*s["blocks"]).T.contiguous()  # what a row is multiplied by
    s["turn"] = [turn[:, 0::2].contiguous(), turn[:, 1::2].contiguous()]
    s["books"] = [_rq_book(case, side) for side in range(2)]
    if old.numel():
        _rq_write(case, s["cache"], old, before, s["blocks"])
    return s


def _lens(case):
    """(context lengths, query lengths): part of the case."""
    rng = np.random.RandomState(4)
    lens = rng.randint(case["shortest"], case["longest"] + 1, case["seqs"])
    lens[0] = case["longest"]
    queries = rng.randint(1, case["queries"] + 1, case["seqs"])
    queries[0] = case["queries"]
    queries = np.minimum(queries, lens)
    return [int(x) for x in lens], [int(x) for x in queries]


def _prepare_attend(case, seed):
    H, D, block = case["heads"], case["head_dim"], case["block"]
    lens, queries = _lens(case)
    need = [-(-n // block) for n in lens]
    order = np.random.RandomState(1000 * int(seed) % (1 << 31) + 5).permutation(sum(need) + 7).astype(np.int32)
    table, begin = np.zeros((len(lens), max(need)), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[begin:begin + n]
        begin += n
    dtype = DTYPES[case["dtype"]]
    cache = torch.empty(2, len(order), block, H, D, dtype=dtype, device=_dev())
    strong = 1 + (torch.randn(H, D, generator=_gen(seed, 2), device=_dev()) * 3).abs()
    for p in range(0, len(order), 4096):  # (fp32 only in part)
        for side in range(2):
            part = cache[side, p:p + 4096]
            x = torch.randn(part.shape, generator=_gen(seed, 100 + p // 4096 * 2 + side), device=_dev())
            part.copy_(x * strong if side == 0 else x)
    q = torch.randn(sum(queries), H * case["group"], D, generator=_gen(seed, 6), device=_dev()).to(dtype)
    return {"case": case, "cache": cache, "table": _i32(table), "lens": _i32(lens), "starts": _i32(np.concatenate([[0], np.cumsum(queries)])),
            "most": max(queries), "longest": max(lens), "q": q, "out": torch.zeros_like(q)}


def prepare(case, seed):
    return _prepare_attend(case, seed) if case["kind"] == "attend" else _prepare_append(case, seed)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _kernels():
    path = os.path.join(os.getcwd(), "rotorquant-vllm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from rotorquant_vllm import kernels
    return kernels


def _run_own(s):
    kernels, case = _kernels(), s["case"]
    kind, H, D = case["kind"], case["heads"], case["head_dim"]
    if kind == "attend":
        return kernels.kv16_attention(s["q"], s["cache"][0], s["cache"][1], s["table"], s["lens"], cu_seqlens_q=None if s["most"] == 1 else s["starts"],
                                      max_q_len=s["most"], max_seq_len=s["longest"], out=s["out"])
    args, neox = (s["q"], s["k"], s["v"], s["positions"], s["table"]), case["style"] == "halves"
    if kind == "kv16":
        q = kernels.rope_kv16_store(*args, s["cache"][0], s["cache"][1], s["slots"], neox=neox, out_q=s["out_q"])
        return {"q": q, "kv": s["cache"]}
    if kind == "q8":
        q = kernels.rope_q8_store(*args, s["cache"], s["slots"], fmt=case["format"], neox=neox, out_q=s["out_q"])
        k, v = kernels.q8_read(s["cache"], s["all"], s["all_lens"], s["starts"], H, D, s["q"].dtype, fmt=case["format"], out_k=s["back"][0],
                               out_v=s["back"][1])
        return {"q": q, "k": k, "v": v}
    (kc, kb), (vc, vb) = s["books"]
    q = kernels.rope_compress_store(*args, s["cache"], s["slots"], *s["turn"], kb, vb, neox=neox, out_q=s["out_q"], rot_block=case["rot_block"])
    k, v = (x.view(s["cache"].shape[0], case["block"], H, D) for x in s["back"])
    kernels.paged_decompress(s["cache"], s["all"], s["all_lens"], H, D, kc, vc, s["q"].dtype, out_k=k, out_v=v)
    return {"q": q, "k": s["back"][0], "v": s["back"][1]}


def _attend(s):
    case, q = s["case"], s["q"]
    H, G, D = case["heads"], case["group"], case["head_dim"]
    k, v = (x[s["table"].long()].flatten(1, 2).float().transpose(1, 2).contiguous() for x in s["cache"])  # (B, H, L, D)
    B, L, T = k.shape[0], k.shape[2], s["most"]
    n = s["starts"].diff()
    rows = torch.arange(T, device=q.device)[None, :] < n[:, None]
    qp = torch.zeros(B, T, H * G, D, device=q.device)
    qp[rows] = q.float()
    qp = qp.view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    scores = torch.matmul(qp, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(D)).view(B, H, T, G, L)
    pos = (s["lens"] - n)[:, None] + torch.arange(T, device=q.device)[None, :]  # of each query
    hidden = torch.arange(L, device=q.device)[None, None, :] > torch.minimum(pos, s["lens"][:, None] - 1)[:, :, None]
    scores.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    scores -= scores.amax(dim=-1, keepdim=True)
    scores.exp_()
    total = scores.sum(dim=-1)
    out = torch.matmul(scores.view(B, H, T * G, L), v).view(B, H, T, G, D) / total[..., None]
    return out.permute(0, 2, 1, 3, 4).reshape(B, T, H * G, D)[rows].to(q.dtype)


def run(s):
    if own:
        return _run_own(s)
    case, kind = s["case"], s["case"]["kind"]
    if kind == "attend":
        return _attend(s)
    rows = s["table"][s["positions"]].float()
    dtype = s["q"].dtype
    q = _rotate(case, s["q"].float(), rows).to(dtype)
    kv = torch.stack([_rotate(case, s["k"].float(), rows), s["v"].float()], dim=1)
    keep = s["slots"] >= 0
    slots, kv = s["slots"][keep], kv[keep]
    if kind == "kv16":
        s["cache"].view(2, -1, *s["cache"].shape[3:])[:, slots] = kv.transpose(0, 1).to(dtype)
        return {"q": q, "kv": s["cache"]}
    if kind == "q8":
        _q8_write(case, s["cache"], slots, kv)
        k, v = _q8_values(case, s["cache"])
    else:
        _rq_write(case, s["cache"], slots, kv, s["blocks"])
        k, v = _rq_values(case, s["cache"])
    return {"q": q, "k": k.to(dtype), "v": v.to(dtype)}


# ---------------------------------------------------------------------------
# Work, and results in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    """Bytes: inputs once, outputs once; operations: 3 for each rotated value, 8 for each one quantised to 8 bits, 2 rot_block + 8 to a codebook,
    2 read back, and two for each product of Q K^T and P V."""
    H, D, HQ = case["heads"], case["head_dim"], case["heads"] * case["group"]
    if case["kind"] == "attend":
        lens, queries = _lens(case)
        pairs = sum(n * L - n * (n - 1) // 2 for n, L in zip(queries, lens))
        return {"bytes": sum(lens) * 4 * H * D + sum(-(-n // case["block"]) for n in lens) * 4 + sum(queries) * HQ * D * 4, "flops": pairs * HQ * D * 4}
    held, n, block = _held(case), case["queries"], case["block"]
    tokens = case["seqs"] * n + case["padded"]
    far = {int(p) for h in held for p in range(h, h + n)}  # rows of the table
    moved = tokens * (HQ * D * 4 + 2 * H * D * 2 + 16) + len(far) * case["rot"] * (4 if case["table"] == "float32" else 2)
    flops = tokens * (HQ + H) * case["rot"] * 3
    if case["kind"] == "kv16":
        return {"bytes": moved + case["seqs"] * n * 4 * H * D, "flops": flops}
    slot = 2 * H * D + H if case["kind"] == "q8" else H * (D + 8)
    back = int(((held + n - 1) // block - held // block + 1).sum()) * block  # slots of the touched pages
    per = 8 if case["kind"] == "q8" else 2 * case["rot_block"] + 8
    return {"bytes": moved + case["seqs"] * n * slot + back * (slot + 4 * H * D), "flops": flops + (case["seqs"] * n * per + back * 2) * 2 * H * D}


def _exact_q8(case, s, slots, kv):
    """Values of every slot after the tokens kv (n, K or V, heads, D) are written, from the format's definition."""
    cache, H, D, block = s["cache"], case["heads"], case["head_dim"], case["block"]
    P, n = cache.shape[0], block // GROUP
    flat = cache.view(P, -1)
    t, h, d = (torch.arange(m, device=cache.device) for m in (block, H, D))
    t, h, d = t[:, None, None], h[None, :, None], d[None, None, :]
    r, chunk = t % GROUP, (d // 64) * 1024
    tile = ((t // GROUP) * H + h) * 2 * GROUP * D
    k_at = tile + chunk + (d % 64 // 16) * 256 + r * 16 + d % 16
    v_at = tile + GROUP * D + chunk + (r // 4) * 256 + (d % 16) * 16 + (d % 64 // 16) * 4 + r % 4
    s_at = (n * H * 2 * GROUP * D + ((t // GROUP) * H + h)[..., 0] * 16).reshape(-1) // 4
    words = flat.view(torch.float32)
    x, scales = [], []
    for at, side in ((k_at, 0), (v_at, 1)):
        b = flat[:, at.reshape(-1)].view(P * block, H, D)
        if case["format"] == "int8":
            c = b.double() - 128
        else:
            e, m = ((b >> 3) & 15).double(), (b & 7).double()
            c = torch.where(e > 0, (8 + m) * torch.exp2(e - 10), m * 2.0 ** -9) * torch.where(b > 127, -1.0, 1.0)
        scales.append(words[:, s_at + side].view(P * block, H).double())
        x.append(c * scales[-1][..., None])
    x, scales = torch.stack(x, dim=1), torch.stack(scales, dim=1)  # (slots, 2, H, D), (slots, 2, H)
    is_new = torch.zeros(x.shape[0], dtype=torch.bool, device=cache.device)
    is_new[slots] = True
    fresh = torch.zeros_like(x)
    fresh[slots] = kv
    is_new, fresh, x, scales = (y.view(-1, GROUP, *y.shape[1:]) for y in (is_new, fresh, x, scales))
    hit, begins = is_new.any(dim=1), is_new[:, 0]
    big = fresh.abs().amax(dim=(1, 4))
    e = torch.where(big > 0, torch.ceil(torch.log2((big / LARGEST[case["format"]]).clamp(min=2.0 ** -200))), torch.full_like(big, -40.0)).clamp(-40, 60)
    scale = torch.maximum(torch.exp2(e), torch.where(begins[:, None, None], 0.0, scales[:, 0]))[:, None, :, :, None]
    y = torch.where(is_new[..., None, None, None], fresh, torch.where(begins[:, None, None, None, None], 0.0, x)) / scale
    if case["format"] == "int8":
        y = y.round().clamp(-127, 127)
    else:
        y = y.clamp(-448, 448)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # between e4m3 values near y
        y = ((y / step).round() * step).clamp(-448, 448)
    x = torch.where(hit[:, None, None, None, None], y * scale, x)
    return x.flatten(0, 1).transpose(0, 1)


def _exact_append(case, s):
    r, half = case["rot"], case["rot"] // 2
    angle = s["table"][s["positions"]].double()
    z = torch.complex(angle[:, :half], angle[:, half:])[:, None, :]

    def turn(x):  # as products of complex numbers
        x = x.double()
        y = x[..., :r].unflatten(-1, (2, half)).transpose(-1, -2) if case["style"] == "halves" else x[..., :r].unflatten(-1, (half, 2))
        y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * z)
        y = y.transpose(-1, -2).flatten(-2) if case["style"] == "halves" else y.flatten(-2)
        return torch.cat([y, x[..., r:]], dim=-1)

    q, keep = turn(s["q"]), s["slots"] >= 0
    slots = s["slots"][keep]
    kv = torch.stack([turn(s["k"])[keep], s["v"].double()[keep]], dim=1)
    if case["kind"] == "kv16":
        cache = s["cache"].double()
        cache.view(2, -1, *cache.shape[3:])[:, slots] = kv.transpose(0, 1)
        return {"q": q, "kv": cache}
    if case["kind"] == "q8":
        k, v = _exact_q8(case, s, slots, kv)
        return {"q": q, "k": k, "v": v}
    H, D = case["heads"], case["head_dim"]
    rows = s["cache"].view(-1, s["cache"].shape[-1])
    out = []
    for side in range(2):
        c, b = (x.double() for x in s["books"][side])
        begin = side * H * (D // 2 + 4)
        nibbles = rows[:, begin:begin + H * D // 2].unflatten(-1, (H, D // 2))
        norm = rows[:, begin + H * D // 2:begin + H * (D // 2 + 4)].contiguous().view(torch.float32).double()
        value = torch.empty(rows.shape[0], H, D, dtype=torch.float64, device=rows.device)
        value[..., 0::2], value[..., 1::2] = c[(nibbles >> 4).long()], c[(nibbles & 15).long()]
        value *= norm[..., None]
        x = kv[:, side]
        n = x.square().sum(dim=-1, keepdim=True).sqrt()
        turned = (x / (n + 1e-10)) @ torch.block_diag(*s["blocks"]).double().T.contiguous()
        value[slots] = c[torch.searchsorted(b, turned.contiguous())] * n
        out.append(value)
    return {"q": q, "k": out[0], "v": out[1]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "attend":
        return _exact_append(case, s)
    H, G, D, block = case["heads"], case["group"], case["head_dim"], case["block"]
    out, begin = torch.zeros(s["q"].shape, dtype=torch.float64, device=_dev()), 0
    for b, (L, n) in enumerate(zip(s["lens"].tolist(), s["starts"].diff().tolist())):
        at = s["table"][b, :-(-L // block)].long()
        k, v = (x[at].flatten(0, 1)[:L].double() for x in s["cache"])
        hidden = torch.arange(L, device=_dev())[None, :] > L - n + torch.arange(n, device=_dev())[:, None]
        for j in range(H * G):
            w = s["q"][begin:begin + n, j].double() @ k[:, j // G].T.contiguous() / math.sqrt(D)
            out[begin:begin + n, j] = w.masked_fill_(hidden, -math.inf).softmax(dim=-1) @ v[:, j // G]
        begin += n
    return out
