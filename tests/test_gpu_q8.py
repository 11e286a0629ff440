"""The 8-bit KV cache on the GPU: codes and values exactly those of the format, attention against 64 bits."""
import numpy as np
import pytest
import torch

import q8_testlib as Q
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
FMTS = ["int8", "fp8"]


def new_cache(pages, block, H, D, fill=0):
    return torch.full((pages, block, K.q8_slot_bytes(H, D)), fill, dtype=torch.uint8, device=DEV)


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def store(cache, ref, k, v, slots, fmt, **kw):
    slots = np.asarray(slots, np.int64)
    K.q8_store(k.to(DEV), v.to(DEV), cache, torch.from_numpy(slots).to(DEV), fmt=fmt, **kw)
    ref.store(k, v, slots)


def agree(cache, ref, fmt):
    assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), fmt)


def filled(lens, block, H, D, fmt, dtype, seed, **kw):
    """(cache on the GPU, reference, table) of sequences of these lengths."""
    table, pages = Q.layout(lens, block, seed)
    ref, cache = Q.Cache(pages, block, H, D, fmt), new_cache(pages, block, H, D)
    k, v = Q.rows(sum(lens), H, D, seed, dtype, **kw)
    slots = np.concatenate([Q.slots_of(table, b, 0, n, block) for b, n in enumerate(lens)] or [np.zeros(0, np.int64)])
    store(cache, ref, k, v, slots, fmt)
    return cache, ref, table


# ---- store -------------------------------------------------------------------


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,H,block,dtype", [(128, 2, 16, torch.bfloat16), (128, 3, 48, torch.float16), (64, 5, 32, torch.bfloat16),
                                             (64, 1, 16, torch.float32), (128, 8, 16, torch.float32)])
def test_store_token_by_token_and_in_one_call(fmt, D, H, block, dtype):
    """Appending with growing scales rounds the codes that stay again; a call with whole groups does not."""
    n = 37
    k, v = Q.rows(n, H, D, 5, dtype)
    k *= torch.linspace(0.01, 40, n)[:, None, None].to(dtype)  # scales that grow within a group
    ref, cache = Q.Cache(4, block, H, D, fmt), new_cache(4, block, H, D)
    slots = np.arange(n) + block  # from page 1 on
    for i in range(n):
        store(cache, ref, k[i:i + 1], v[i:i + 1], slots[i:i + 1], fmt)
    agree(cache, ref, fmt)
    ref, cache = Q.Cache(4, block, H, D, fmt), new_cache(4, block, H, D)
    store(cache, ref, k, v, slots, fmt)
    agree(cache, ref, fmt)
    store(cache, ref, k[:7] * 100, v[:7] * 0.01, slots[20:27], fmt)  # rewritten inside a group
    agree(cache, ref, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [1, 5, 63, 64, 257, 512, 513, 1500])
def test_store_any_order_duplicates_and_padding(fmt, n):
    """Slots in random order, some twice or more, some outside the cache: one launch or three, the last token counts."""
    H, D, block, pages = 2, 64, 32, 16
    rng = np.random.RandomState(n)
    ref, cache = Q.Cache(pages, block, H, D, fmt), new_cache(pages, block, H, D)
    for round_ in range(2):  # the second over what the first left
        k, v = Q.rows(n, H, D, 10 * n + round_, torch.float16)
        slots = rng.randint(-3, pages * block + 3, n)
        slots[slots == -2] = np.iinfo(np.int64).min
        store(cache, ref, k, v, slots, fmt)
        agree(cache, ref, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_store_extremes(fmt):
    """Zeros, the smallest and largest values of a type, infinities and NaN."""
    H, D = 2, 128
    k, v = Q.rows(48, H, D, 3, torch.float32)
    k[0] = 0.0
    v[:16] = 0.0
    v[16, 0, 5] = float("inf")
    v[17, 1, 6] = -float("inf")
    v[18, 0, 7] = float("nan")
    k[20] = float("nan")
    k[32:48] *= 1e-20
    k[40, 0] = 3e38
    v[32:48, 1] = 2.0 ** -41
    ref, cache = Q.Cache(3, 16, H, D, fmt), new_cache(3, 16, H, D)
    store(cache, ref, k, v, np.arange(48), fmt)
    agree(cache, ref, fmt)
    big = torch.full((16, H, D), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    tiny = torch.full((16, H, D), 1e-38, dtype=torch.bfloat16)
    store(cache, ref, big, tiny, np.arange(16), fmt)
    agree(cache, ref, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_every_code_and_every_tie(fmt):
    """All codes, the midpoints between them and their neighbours, at a scale of 1 (a value of 127 or 448 in the group)."""
    c = np.arange(-127, 128.0) if fmt == "int8" else np.unique(Q.e4m3_values()[np.isfinite(Q.e4m3_values())])
    mid = (c[1:] + c[:-1]) / 2
    x = np.concatenate([c, mid, np.nextafter(mid, 1e9, dtype=np.float32), np.nextafter(mid, -1e9, dtype=np.float32)])
    D, H = 128, 1
    n = -(-len(x) // (D * 15)) * 15
    flat = np.zeros(n * D)
    flat[:len(x)] = x
    t = torch.from_numpy(flat.reshape(n, H, D)).float()
    rows, slots = [], []
    for g in range(n // 15):  # the group's first row holds the largest code
        rows += [torch.full((1, H, D), float(c.max())), t[15 * g:15 * g + 15]]
        slots += list(range(16 * g, 16 * g + 16))
    t = torch.cat(rows)
    ref, cache = Q.Cache(n // 15, 16, H, D, fmt), new_cache(n // 15, 16, H, D)
    store(cache, ref, t, t, slots, fmt)
    assert (ref.exps == 0).all()
    agree(cache, ref, fmt)


def test_store_leaves_other_pages_and_strided_inputs():
    """K and V as views of one projection, a cache with a gap between its pages and old bytes in it."""
    H, D, block, n = 4, 128, 16, 21
    qkv = torch.randn(n, (8 + 2 * H) * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    k, v = qkv[:, 8 * D:(8 + H) * D].view(n, H, D), qkv[:, (8 + H) * D:].view(n, H, D)
    sb = K.q8_slot_bytes(H, D)
    raw = torch.full((5, 2, block, sb), 171, dtype=torch.uint8, device=DEV)
    cache = raw[:, 0]
    slots = torch.arange(n, device=DEV) + 2 * block
    K.q8_store(k, v, cache, slots)
    ref = Q.Cache(5, block, H, D, "int8")
    ref.store(k.cpu(), v.cpu(), slots.cpu().numpy())
    got, want = cache.cpu().numpy(), ref.to_bytes()
    payload = block // 16 * H * (32 * D)
    got2, want2 = got.reshape(5, -1), want.reshape(5, -1)
    assert np.array_equal(got2[2:4, :payload], want2[2:4, :payload])
    sc = slice(payload, payload + 16 * H)
    assert np.array_equal(got2[2:4, sc].copy().view(np.float32).reshape(2, H, 4)[..., :2], want2[2:4, sc].copy().view(np.float32).reshape(2, H, 4)[..., :2])
    assert (got2[[0, 1, 4]] == 171).all() and bool((raw[:, 1] == 171).all())


# ---- read back ------------------------------------------------------------------


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,H,block,dtype", [(128, 2, 16, torch.bfloat16), (64, 3, 32, torch.float16), (128, 1, 64, torch.float32)])
def test_read(fmt, D, H, block, dtype):
    lens = [0, 1, 15, 16, 17, 0, 130, 64, 3]
    cache, ref, table = filled(lens, block, H, D, fmt, torch.float16, 7)
    kv = ref.values()
    gaps = [0, 2, 0, 5, 0, 1, 0, 0, 4]  # rows between sequences that stay as they were
    starts = np.cumsum([0] + [n + g for n, g in zip(lens, gaps)])
    total = int(starts[-1]) + 6
    out = [torch.full((total, H, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    got = K.q8_read(cache, i32(table), i32(lens), i32(starts), H, D, dtype, fmt=fmt, out_k=out[0], out_v=out[1])
    for side in range(2):
        want = torch.full((total, H, D), 7.0, dtype=dtype)
        for b, n in enumerate(lens):
            want[starts[b]:starts[b] + n] = torch.from_numpy(kv[side][Q.slots_of(table, b, 0, n, block)]).to(dtype)
        assert got[side].data_ptr() == out[side].data_ptr()
        assert torch.equal(out[side].cpu(), want)


def test_read_many_sequences_and_cut_rows():
    """More sequences than one step of the search takes; rows past the outputs are not written."""
    H, D = 1, 64
    rng = np.random.RandomState(0)
    lens = list(rng.randint(0, 40, 300))
    cache, ref, table = filled(lens, 16, H, D, "int8", torch.bfloat16, 9)
    starts = np.concatenate([[0], np.cumsum(lens)])
    total = int(starts[-1])
    kv = ref.values()
    at = np.concatenate([Q.slots_of(table, b, 0, n, 16) for b, n in enumerate(lens)])
    k, v = K.q8_read(cache, i32(table), i32(lens), i32(starts), H, D, torch.bfloat16, total=total)
    for got, side in ((k, 0), (v, 1)):
        assert torch.equal(got.cpu(), torch.from_numpy(kv[side][at]).to(torch.bfloat16))
    whole = torch.zeros(total, H, D, dtype=torch.bfloat16, device=DEV)
    K.q8_read(cache, i32(table), i32(lens), i32(starts), H, D, torch.bfloat16, out_k=whole[:total - 50], out_v=torch.zeros_like(whole[:total - 50]))
    assert torch.equal(whole[:total - 50].cpu(), k[:total - 50].cpu()) and not whole[total - 50:].any()


def test_bad_pages_read_page_zero():
    """Page ids outside the cache, as in the other kernels, stand for page 0."""
    H, D, block = 2, 128, 16
    cache, ref, table = filled([40], block, H, D, "int8", torch.bfloat16, 3)
    bad, good = table.copy(), table.copy()
    bad[0, 1], good[0, 1] = 1 << 30, 0
    bad[0, 2], good[0, 2] = -7, 0
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    outs = []
    for t in (bad, good):
        outs.append(list(K.q8_read(cache, i32(t), i32([40]), i32([0]), H, D, torch.float32, total=40)) + [K.q8_attention(q, cache, i32(t), i32([40]), H, D)])
    for x, y in zip(*outs):
        assert torch.equal(x, y)


# ---- attention ------------------------------------------------------------------


def attend(lens, queries, block, H, G, D, fmt, dtype, seed, causal=True, sm_scale=None, prepare=None, **kw):
    cache, ref, table = filled([max(n, 0) for n in lens], block, H, D, fmt, dtype, seed)
    cu = np.concatenate([[0], np.cumsum(queries)])
    q = torch.randn(int(cu[-1]), H * G, D, generator=torch.Generator().manual_seed(seed)).to(dtype)
    if prepare:
        q = prepare(q)
    out, tol = Q.attention(q, ref.values(), table, lens, cu, block, causal, sm_scale)
    got = K.q8_attention(q.to(DEV), cache, i32(table), i32(lens), H, D, fmt=fmt, cu_seqlens_q=i32(cu), max_q_len=max(queries), causal=causal,
                         sm_scale=sm_scale, **kw)
    err = np.abs(got.double().cpu().numpy() - out)
    assert (err <= tol).all(), f"off by {float((err - tol).max()):.2e} past the tolerance"
    return got


SHAPES = [(2, 4, 128, 16), (1, 8, 128, 32), (4, 7, 64, 16), (2, 1, 128, 48), (1, 17, 64, 64), (3, 2, 128, 16)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,D,block", SHAPES)
def test_decode(fmt, dtype, H, G, D, block):
    lens = [1, 16, 17, 31, 32, 33, 129, 0, 500]
    got = attend(lens, [1] * len(lens), block, H, G, D, fmt, dtype, 11)
    assert not got[7].any()  # no keys: zeros
    table, _ = Q.layout(lens, block, 11)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,G,D,block", SHAPES[:4])
def test_drafts(fmt, causal, H, G, D, block):
    """A few tokens per sequence, none, and more than the sequence has keys."""
    lens, queries = [40, 1, 100, 5, 64, 3, 0, 333], [5, 1, 0, 5, 9, 7, 2, 16]
    got = attend(lens, queries, block, H, G, D, fmt, torch.bfloat16, 12, causal=causal)
    if causal:
        at = sum(queries[:5])
        assert not got[at:at + 4].any()  # 7 queries over 3 keys: the first four see none


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,D,lens,queries", [(2, 4, 128, [70, 33, 200], [70, 33, 41]), (1, 3, 64, [130], [130]), (1, 1, 128, [64, 65, 63], [64, 65, 63]),
                                                (1, 8, 128, [300, 21], [21, 21])])
def test_prompts_and_chunks(fmt, dtype, H, G, D, lens, queries):
    attend(lens, queries, 16, H, G, D, fmt, dtype, 13)


@pytest.mark.parametrize("sm_scale", [0.0, -0.1, 1.0, 1e-6])
def test_scales(sm_scale):
    attend([77, 40], [1, 3], 16, 2, 4, 128, "int8", torch.bfloat16, 14, sm_scale=sm_scale)


@pytest.mark.parametrize("fmt", FMTS)
def test_large_and_small_rows(fmt):
    """Query rows far from 1 and a zero row; values of very different groups."""
    def prepare(q):
        q[0] *= 1e-30
        q[1] = 0
        q[2, :, 3] = 2000.0
        return q
    attend([50, 60, 70, 80], [1, 1, 1, 1], 16, 2, 4, 128, fmt, torch.bfloat16, 15, prepare=prepare)


@pytest.mark.parametrize("fmt", FMTS)
def test_groups_of_very_different_scales(fmt):
    """V groups 2^30 apart, and one of zeros: its tokens still count in the sum."""
    H, D, block, n = 1, 128, 16, 96
    k, v = Q.rows(n, H, D, 4, torch.float32, outliers=False)
    for g, e in enumerate((-20, 10, 0, -10, 5, 0)):
        v[16 * g:16 * g + 16] *= 2.0 ** e
    v[32:48] = 0
    k[16:32] *= 0.0
    k[16:32, :, 0] = -60.0  # the largest values under small weights
    table, pages = Q.layout([n], block, 2)
    ref, cache = Q.Cache(pages, block, H, D, fmt), new_cache(pages, block, H, D)
    store(cache, ref, k, v, Q.slots_of(table, 0, 0, n, block), fmt)
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(2)).to(torch.float16)
    q[:, :, 0] = 4.0
    out, tol = Q.attention(q, ref.values(), table, [n], [0, 1], block)
    got = K.q8_attention(q.to(DEV), cache, i32(table), i32([n]), H, D, fmt=fmt)
    assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,G,D,n,t", [(1, 4, 128, 96, 96), (2, 8, 64, 200, 30), (1, 1, 128, 193, 193), (1, 4, 128, 2100, 50)])
def test_prompts_of_very_different_scales(fmt, H, G, D, n, t):
    """As above, prompts: tokens whose weights fp16 does not hold (their V is 2^20 to 2^30 times smaller, or zero) keep their
    place in the sum of the softmax."""
    block = 16
    k, v = Q.rows(n, H, D, 4, torch.float32, outliers=False)
    k *= 0.25
    for g in range(-(-n // 16)):
        v[16 * g:16 * g + 16] *= (2.0 ** 10, 2.0 ** -20, 0.0, 1.0, 2.0 ** -10)[g % 5]
    table, pages = Q.layout([n], block, 2)
    ref, cache = Q.Cache(pages, block, H, D, fmt), new_cache(pages, block, H, D)
    store(cache, ref, k, v, Q.slots_of(table, 0, 0, n, block), fmt)
    q = torch.randn(t, H * G, D, generator=torch.Generator().manual_seed(2)).to(torch.float16)
    out, tol = Q.attention(q, ref.values(), table, [n], [0, t], block)
    got = K.q8_attention(q.to(DEV), cache, i32(table), i32([n]), H, D, fmt=fmt, cu_seqlens_q=i32([0, t]), max_q_len=t)
    assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_memory_behind_the_contexts_is_not_read_as_numbers(fmt):
    """Pages full of bytes that no store wrote (NaN codes, infinite scales) behind a context's end, and never-begun groups."""
    H, D, block, n = 2, 128, 64, 37
    k, v = Q.rows(n, H, D, 6, torch.bfloat16)
    table, pages = Q.layout([n], block, 2)
    ref = Q.Cache(pages, block, H, D, fmt)
    clean, dirty = new_cache(pages, block, H, D), new_cache(pages, block, H, D, fill=0xff)
    slots = Q.slots_of(table, 0, 0, n, block)
    store(clean, ref, k, v, slots, fmt)
    K.q8_store(k.to(DEV), v.to(DEV), dirty, torch.from_numpy(slots).to(DEV), fmt=fmt)
    # rows of the last group behind the context: NaN codes
    idx_k, idx_v, _ = Q.code_index(block, H, D)
    raw = dirty[table[0, 0]].view(-1)
    for idx in (idx_k, idx_v):
        raw[torch.from_numpy(idx[n:48].reshape(-1)).to(DEV)] = 0x7f
    for T in (1, 5):
        q = torch.randn(T, 8, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
        cu = i32([0, T])
        a, b = (K.q8_attention(q, c, i32(table), i32([n]), H, D, fmt=fmt, cu_seqlens_q=cu) for c in (clean, dirty))
        assert torch.equal(a, b)


def test_long_context_splits_agree():
    """A context over many workgroups, next to short ones; bounds on the lengths change the shares, not the result."""
    H, G, D, block = 2, 4, 128, 16
    lens = [9001, 3, 700]
    cache, ref, table = filled(lens, block, H, D, "int8", torch.bfloat16, 21)
    q = torch.randn(3, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, tol = Q.attention(q, ref.values(), table, lens, [0, 1, 2, 3], block)
    for bound in (None, 9001, 20000):
        got = K.q8_attention(q.to(DEV), cache, i32(table), i32(lens), H, D, max_seq_len=bound)
        assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()
    short = K.q8_attention(q.to(DEV), cache, i32(table), i32(lens), H, D, max_seq_len=500)  # keys past the bound are not read
    out, tol = Q.attention(q, ref.values(), table, [500, 3, 500], [0, 1, 2, 3], block)
    assert (np.abs(short.double().cpu().numpy() - out) <= tol).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,G,D,lens,queries,causal", [
    (2, 4, 128, [200, 64, 1, 0, 450], [200, 33, 1, 0, 130], True), (1, 8, 64, [300, 129], [65, 129], True), (3, 3, 128, [97], [97], False),
    (1, 1, 128, [2500], [160], True), (2, 5, 64, [1100, 40], [40, 40], True), (1, 4, 128, [30, 70], [90, 70], True)])
def test_prompts(fmt, H, G, D, lens, queries, causal):
    """Query lengths that take the prefill kernels: odd ones, none, more queries than keys, few queries over long contexts."""
    attend(lens, queries, 16, H, G, D, fmt, torch.float16, 31, causal=causal)
    attend(lens, queries, 32, H, G, D, fmt, torch.bfloat16, 32, causal=causal)


# ---- together ------------------------------------------------------------------


def _backend(monkeypatch, fmt, H, HQ, D):
    import math
    monkeypatch.setenv("RQ_CACHE_8BIT", fmt)
    monkeypatch.delenv("RQ_DENSE_3BIT", raising=False)
    from rotorquant_vllm.vllm import rq_backend as B
    return B, B.RQAttentionImpl(HQ, D, 1 / math.sqrt(D), num_kv_heads=H)


def _metadata(slots, table, lens, q_lens, host=True):
    import types
    md = types.SimpleNamespace(num_actual_tokens=sum(q_lens), max_query_len=max(q_lens), use_cascade=False, block_table=i32(table), seq_lens=i32(lens),
                               slot_mapping=torch.from_numpy(np.asarray(slots, np.int64)).to(DEV), query_start_loc=i32(np.concatenate([[0], np.cumsum(q_lens)])))
    if host:
        md.rq_seq_lens_cpu, md.rq_query_start_loc_cpu = md.seq_lens.cpu(), md.query_start_loc.cpu()
    return md


@pytest.mark.parametrize("fmt,H,G,D,block,dtype", [("int8", 2, 4, 128, 16, torch.bfloat16), ("fp8", 3, 2, 64, 32, torch.float16)])
def test_backend_steps(monkeypatch, fmt, H, G, D, block, dtype):
    """Prompts, then a mixed batch (decodes, a draft, a prompt chunk), then decodes, through the backend: the cache and every
    output against the plain implementation."""
    B, impl = _backend(monkeypatch, fmt, H, H * G, D)
    final = [75, 60, 40, 310]
    table, pages = Q.layout(final, block, 3)
    cache = torch.zeros(B.RQAttentionBackend.get_kv_cache_shape(pages, block, H, D), dtype=torch.uint8, device=DEV)
    ref = Q.Cache(pages, block, H, D, fmt)
    done = [0, 0, 0, 0]
    for step, q_lens in enumerate(([70, 50, 33, 0], [1, 1, 5, 300], [1, 1, 1, 1], [2, 7, 0, 3])):
        seqs = [b for b in range(4) if q_lens[b]]
        q_step = [q_lens[b] for b in seqs]
        slots = np.concatenate([Q.slots_of(table, b, done[b], done[b] + q_lens[b], block) for b in seqs])
        for b in seqs:
            done[b] += q_lens[b]
        lens = [done[b] for b in seqs]
        n = sum(q_step)
        k, v = Q.rows(n, H, D, 50 + step, dtype)
        q = torch.randn(n, H * G, D, generator=torch.Generator().manual_seed(step)).to(dtype)
        out = torch.full((n + 1, H * G, D), 9.0, dtype=dtype, device=DEV)
        md = _metadata(slots, table[seqs], lens, q_step, host=step != 2)
        impl.forward(None, q.to(DEV), k.to(DEV), v.to(DEV), cache, md, output=out)
        ref.store(k, v, slots)
        agree(cache, ref, fmt)
        want, tol = Q.attention(q, ref.values(), table[seqs], lens, np.concatenate([[0], np.cumsum(q_step)]), block)
        assert (np.abs(out[:n].double().cpu().numpy() - want) <= tol).all(), step
        assert bool((out[n] == 9.0).all())


def test_backend_decode_graph(monkeypatch):
    """A captured decode step (store and attention) replayed over longer contexts, with eager work in between."""
    H, G, D, block, fmt = 2, 4, 128, 16, "int8"
    B, impl = _backend(monkeypatch, fmt, H, H * G, D)
    start, steps = [40, 700, 5], 20
    table, pages = Q.layout([n + steps for n in start], block, 8)
    cache, ref = new_cache(pages, block, H, D), Q.Cache(pages, block, H, D, fmt)
    k0, v0 = Q.rows(sum(start), H, D, 60, torch.bfloat16)
    store(cache, ref, k0, v0, np.concatenate([Q.slots_of(table, b, 0, n, block) for b, n in enumerate(start)]), fmt)
    buf = {"q": torch.zeros(3, H * G, D, dtype=torch.bfloat16, device=DEV), "k": torch.zeros(3, H, D, dtype=torch.bfloat16, device=DEV),
           "v": torch.zeros(3, H, D, dtype=torch.bfloat16, device=DEV), "out": torch.zeros(3, H * G, D, dtype=torch.bfloat16, device=DEV)}
    md = _metadata([-1, -1, -1], table, start, [1, 1, 1], host=False)
    step = lambda: impl.forward(None, buf["q"], buf["k"], buf["v"], cache, md, output=buf["out"])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (slots of -1: nothing is stored)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    lens = list(start)
    for i in range(steps):
        k, v = Q.rows(3, H, D, 70 + i, torch.bfloat16)
        q = torch.randn(3, H * G, D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
        slots = np.concatenate([Q.slots_of(table, b, n, n + 1, block) for b, n in enumerate(lens)])
        lens = [n + 1 for n in lens]
        buf["q"].copy_(q), buf["k"].copy_(k), buf["v"].copy_(v)
        md.slot_mapping.copy_(torch.from_numpy(slots)), md.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        ref.store(k, v, slots)
        got = buf["out"].clone()
        eager = K.q8_attention(buf["q"], cache, md.block_table, md.seq_lens, H, D, fmt=fmt)
        assert torch.equal(got, eager)
        if i % 6 == 0:
            torch.cuda.synchronize()
            agree(cache, ref, fmt)
            want, tol = Q.attention(q, ref.values(), table, lens, [0, 1, 2, 3], block)
            assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


def test_captured_prompt_and_long_store():
    """A store of more than 512 tokens, a prompt and a read-back in one graph: several replays with new inputs."""
    H, G, D, block, fmt, n = 2, 4, 128, 16, "fp8", 600
    table, pages = Q.layout([n], block, 4)
    cache = new_cache(pages, block, H, D)
    slots = torch.from_numpy(Q.slots_of(table, 0, 0, n, block)).to(DEV)
    bt, sl, cu = i32(table), i32([n]), i32([0, n])
    k, v = (x.to(DEV) for x in Q.rows(n, H, D, 1, torch.bfloat16))
    q = torch.zeros(n, H * G, D, dtype=torch.bfloat16, device=DEV)

    def work():
        K.q8_store(k, v, cache, slots, fmt=fmt)
        return K.q8_attention(q, cache, bt, sl, H, D, fmt=fmt, cu_seqlens_q=cu, max_q_len=n), K.q8_read(cache, bt, sl, cu, H, D, torch.bfloat16, fmt=fmt, total=n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, (rk, rv) = work()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        a, b = Q.rows(n, H, D, 90 + i, torch.bfloat16)
        k.copy_(a), v.copy_(b)
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        got = [x.clone() for x in (out, rk, rv)]
        eager_out, (ek, ev) = work()
        torch.cuda.synchronize()
        for x, y in zip(got, (eager_out, ek, ev)):
            assert torch.equal(x, y)


def test_two_streams_at_once():
    """Calls that overlap on two streams have scratch of their own."""
    H, G, D, block = 2, 4, 128, 16
    lens = [5000, 300, 4000]
    cache, ref, table = filled(lens, block, H, D, "int8", torch.bfloat16, 5)
    bt, sl = i32(table), i32(lens)
    qs = [torch.randn(3, H * G, D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    want = [K.q8_attention(q, cache, bt, sl, H, D) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(K.q8_attention(qs[i], cache, bt, sl, H, D))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_strided_and_expanded_inputs():
    """q as a view of a fused projection, an output row stride, a transposed block table, a shared prefix (the same pages twice)."""
    H, G, D, block = 2, 4, 128, 16
    lens = [90, 90]
    cache, ref, table = filled([90], block, H, D, "int8", torch.bfloat16, 6)
    table = np.concatenate([table, table])
    qkv = torch.randn(2, (H * G + 2 * H) * D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    q = qkv[:, :H * G * D].view(2, H * G, D)
    wide = torch.full((2, H * G, D + 8), 3.0, dtype=torch.bfloat16, device=DEV)
    bt = i32(np.ascontiguousarray(table.T)).t()
    got = K.q8_attention(q, cache, bt, i32(lens), H, D, out=wide[..., :D])
    want, tol = Q.attention(q.cpu(), ref.values(), table, lens, [0, 1, 2], block)
    assert got.data_ptr() == wide.data_ptr() and bool((wide[..., D:] == 3.0).all())
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    odd = torch.zeros(2 * H * G * D + 4, dtype=torch.bfloat16, device=DEV)[4:].view(2, H * G, D)  # 8 bytes off
    with pytest.raises(ValueError, match="16-byte aligned"):
        K.q8_attention(odd, cache, bt, i32(lens), H, D)
    with pytest.raises(ValueError, match="16-byte aligned"):
        K.q8_store(odd[:, :H], odd[:, :H], cache, torch.zeros(2, dtype=torch.int64, device=DEV))


def test_empty_calls():
    H, D = 2, 128
    cache = new_cache(2, 16, H, D)
    e = torch.zeros(0, H, D, dtype=torch.bfloat16, device=DEV)
    K.q8_store(e, e, cache, torch.zeros(0, dtype=torch.int64, device=DEV))
    k, v = K.q8_read(cache, i32(np.zeros((0, 1))), i32([]), i32([]), H, D, torch.bfloat16, total=0)
    assert k.shape == v.shape == (0, H, D)
    q = torch.zeros(0, 8, D, dtype=torch.bfloat16, device=DEV)
    assert K.q8_attention(q, cache, i32(np.zeros((0, 1))), i32([]), H, D).shape == (0, 8, D)
    # a zeroed page reads as zeros, and attends as zeros
    k, v = K.q8_read(cache, i32([[0]]), i32([5]), i32([0]), H, D, torch.float32, total=5)
    assert not k.any() and not v.any()
    q = torch.ones(1, 8, D, dtype=torch.bfloat16, device=DEV)
    assert K.q8_attention(q, cache, i32([[0]]), i32([5]), H, D).abs().max() < 1e-9
    # a table without pages: nothing to see
    out = K.q8_attention(q, cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), i32([5]), H, D)
    assert not out.any()


# ---- sizes that change the path -------------------------------------------------


@pytest.mark.parametrize("fmt", FMTS)
def test_many_sequences(fmt):
    """More than 64 sequences, some empty, shared out over the GPU (a long bound) and an item each (a short one)."""
    H, G, D, block = 1, 3, 64, 16
    rng = np.random.RandomState(3)
    lens = [int(n) for n in rng.randint(0, 50, 150)]
    lens[70], lens[140] = 700, 400
    cache, ref, table = filled(lens, block, H, D, fmt, torch.bfloat16, 17)
    q = torch.randn(150, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, tol = Q.attention(q, ref.values(), table, lens, range(151), block)
    wide = np.zeros((150, 200), np.int32)
    wide[:, :table.shape[1]] = table
    for t in (table, wide):
        got = K.q8_attention(q.to(DEV), cache, i32(t), i32(lens), H, D, fmt=fmt)
        assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()
    queries = [int(n) for n in rng.randint(0, 6, 150)]
    cu = np.concatenate([[0], np.cumsum(queries)])
    q = torch.randn(int(cu[-1]), H * G, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out, tol = Q.attention(q, ref.values(), table, lens, cu, block)
    for t in (table, wide):
        got = K.q8_attention(q.to(DEV), cache, i32(t), i32(lens), H, D, fmt=fmt, cu_seqlens_q=i32(cu), max_q_len=5)
        assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()


@pytest.mark.parametrize("D", [64, 128])
def test_prompts_in_several_passes(D):
    """A table so wide that the tile images of one kv head fill a pass: one launch pair per sequence and head."""
    H, G, block = 2, 4, 32
    lens, queries = [90, 0, 200], [90, 0, 70]
    cache, ref, table = filled(lens, block, H, D, "int8", torch.bfloat16, 18)
    cu = [0, 90, 90, 160]
    q = torch.randn(160, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, tol = Q.attention(q, ref.values(), table, lens, cu, block)
    wide = np.zeros((3, 16384), np.int32)
    wide[:, :table.shape[1]] = table
    for t, bound in ((wide, None), (table, None), (wide, 200)):
        got = K.q8_attention(q.to(DEV), cache, i32(t), i32(lens), H, D, cu_seqlens_q=i32(cu), max_q_len=90, max_seq_len=bound)
        assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()


def test_cache_past_32_bits():
    """Pages more than 4 GiB into a cache: written, read back and attended to."""
    H, G, D, block, n = 8, 2, 128, 16, 100
    pages = (5 << 30) // (block * K.q8_slot_bytes(H, D))
    cache = torch.empty(pages, block, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV)
    table = np.arange(pages - 7, pages, dtype=np.int32)[None]
    small, ref = np.arange(7, dtype=np.int32)[None], Q.Cache(7, block, H, D, "fp8")
    k, v = Q.rows(n, H, D, 8, torch.bfloat16)
    K.q8_store(k.to(DEV), v.to(DEV), cache, torch.from_numpy(Q.slots_of(table, 0, 0, n, block)).to(DEV), fmt="fp8")
    ref.store(k, v, Q.slots_of(small, 0, 0, n, block))
    kv = ref.values()
    got = K.q8_read(cache, i32(table), i32([n]), i32([0]), H, D, torch.float32, fmt="fp8", total=n)
    for side in range(2):
        assert np.array_equal(got[side].cpu().numpy(), kv[side][Q.slots_of(small, 0, 0, n, block)].astype(np.float32))
    for T in (1, 100):  # (the second by the prefill kernels)
        q = torch.randn(T, H * G, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        out, tol = Q.attention(q, kv, small, [n], [0, T], block)
        got = K.q8_attention(q.to(DEV), cache, i32(table), i32([n]), H, D, fmt="fp8", cu_seqlens_q=i32([0, T]))
        assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()


def test_nan_and_infinite_queries_stay_in_their_rows():
    H, G, D, block = 1, 4, 128, 16
    cache, ref, table = filled([60], block, H, D, "int8", torch.bfloat16, 19)
    for T in (1, 6, 60):  # item, columns of a block, prefill
        q = torch.randn(T, H * G, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        clean = K.q8_attention(q.to(DEV), cache, i32(table), i32([60]), H, D, cu_seqlens_q=i32([0, T]))
        bad = q.clone()
        bad[T // 2, 1, 5] = float("nan")
        bad[T // 2, 2, 6] = float("inf")
        got = K.q8_attention(bad.to(DEV), cache, i32(table), i32([60]), H, D, cu_seqlens_q=i32([0, T]))
        keep = torch.ones(T, H * G, dtype=torch.bool)
        keep[T // 2, 1:3] = False
        assert torch.equal(got[keep.to(DEV)], clean[keep.to(DEV)])
        assert not torch.isfinite(got[T // 2, 1:3]).any()


@pytest.mark.parametrize("fmt", FMTS)
def test_memory_behind_the_contexts_in_prompts(fmt):
    """As above, for the prefill kernels: the rows of the last group behind a prompt hold NaN's codes."""
    H, G, D, block, n = 1, 4, 128, 64, 69
    k, v = Q.rows(n, H, D, 6, torch.bfloat16)
    table, pages = Q.layout([n], block, 2)
    clean, dirty = new_cache(pages, block, H, D), new_cache(pages, block, H, D, fill=0xff)
    slots = torch.from_numpy(Q.slots_of(table, 0, 0, n, block)).to(DEV)
    for c in (clean, dirty):
        K.q8_store(k.to(DEV), v.to(DEV), c, slots, fmt=fmt)
    idx_k, idx_v, _ = Q.code_index(block, H, D)
    raw = dirty[table[0, 1]].view(-1)
    for idx in (idx_k, idx_v):
        raw[torch.from_numpy(idx[n - 64:16].reshape(-1)).to(DEV)] = 0x7f
    q = torch.randn(n, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    for causal in (True, False):
        a, b = (K.q8_attention(q, c, i32(table), i32([n]), H, D, fmt=fmt, causal=causal, cu_seqlens_q=i32([0, n])) for c in (clean, dirty))
        assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(seed):
    rng = np.random.RandomState(1000 + seed)
    H, G, D, block = int(rng.choice([1, 2, 3, 5])), int(rng.choice([1, 2, 4, 6, 9])), int(rng.choice([64, 128])), int(rng.choice([16, 32, 48, 128]))
    fmt, dtype = FMTS[seed % 2], [torch.bfloat16, torch.float16][(seed // 2) % 2]
    B = int(rng.randint(1, 7))
    lens = [int(n) for n in rng.randint(0, int(rng.choice([40, 300])), B)]
    queries = [int(rng.randint(0, int(rng.choice([2, 8, 90])) + 1)) for _ in range(B)]
    queries[0] = max(1, queries[0])
    attend(lens, queries, block, H, G, D, fmt, dtype, 40 + seed, causal=bool(rng.randint(0, 4)))
