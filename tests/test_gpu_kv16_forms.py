"""kv16_attention in the forms that long contexts and long queries take: a wave for each kv head, queries of a thousand tokens."""
import math

import numpy as np
import pytest
import torch

import kv16_testlib as P
from rotorquant_vllm import _lib
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
KEYS = 1 << 18  # what a wide table could hold


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def padded(table, block=16, keys=KEYS):
    """The table with columns up to a capacity of `keys`: pages that no sequence has, nor are they read."""
    wide = np.full((table.shape[0], keys // block), -5, np.int32)
    wide[:, :table.shape[1]] = table
    return wide


def assert_a_wave_for_each_head(seqs, HQ, H, D, max_q, keys=KEYS):
    """By the scratch of the call: with a head for each of its four waves, the GPU's resident workgroups take four times as many shares."""
    width = 64 if D <= 64 else 128 if D <= 128 else 256
    blocks = 2 if max_q * HQ // H > 16 else 1
    resident = (1 if width == 256 else 2) * torch.cuda.get_device_properties(0).multi_processor_count
    need = _lib.load().rq_kv16_attention_workspace_bytes(seqs, HQ, H, D, max_q, keys)
    assert need == 2 * (4 * resident // H) * H * blocks * 16 * (width + 2) * 4


def case(lens, q_lens, H, G, D, dtype, seed=1):
    pages = P.Pages(lens, 16, H, D, dtype, seed)
    return pages, torch.randn(sum(q_lens), H * G, D, generator=P.gen(seed + 1)).to(dtype)


def rewritten(pages):
    """The pages' tensors with what pages.kv holds."""
    for side, cache in enumerate(pages.view(pages.both)):
        for b, x in enumerate(pages.kv[side]):
            at = torch.arange(len(x))
            cache[torch.from_numpy(pages.table[b].astype(np.int64))[at // 16], at % 16] = x
    return pages.to(DEV)


def run(pages, q, lens, q_lens, table=None, causal=True, **kw):
    return K.kv16_attention(q.to(DEV), *rewritten(pages), i32(pages.table if table is None else table), i32(lens), causal=causal,
                            cu_seqlens_q=i32(np.concatenate([[0], np.cumsum(q_lens)])), max_q_len=max(q_lens), **kw)


# ---- a wave for each kv head -----------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [40, 64, 96, 128])
@pytest.mark.parametrize("H,G,q_lens", [(4, 1, [1, 1, 1, 1]), (8, 5, [1, 1, 1, 1]), (4, 3, [4, 1, 7, 5]), (4, 17, [1, 3, 1, 2]), (12, 2, [1, 2, 9, 1])])
def test_a_wave_for_each_head(H, G, q_lens, D, dtype):
    """Short contexts, an empty one and a long one that is cut into shares, one block of columns or two."""
    lens = [1, 260, 0, 9000]
    assert_a_wave_for_each_head(4, H * G, H, D, max(q_lens))
    for causal in (True, False):
        pages, q = case(lens, q_lens, H, G, D, dtype)
        P.check(run(pages, q, lens, q_lens, padded(pages.table), causal), *P.attention(q, *pages.kv, lens, q_lens, causal=causal))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [200, 256])
@pytest.mark.parametrize("H,G", [(4, 1), (8, 5), (4, 16)])
def test_a_wave_for_each_wide_head(H, G, D, dtype):
    lens = [1, 260, 0, 9000]
    assert_a_wave_for_each_head(4, H * G, H, D, 1)
    pages, q = case(lens, [1] * 4, H, G, D, dtype)
    P.check(run(pages, q, lens, [1] * 4, padded(pages.table)), *P.attention(q, *pages.kv, lens, [1] * 4))


def test_many_sequences_by_heads():
    """More than 64 of them, which the shares are walked through 64 at a time."""
    lens = [int(x) for x in np.random.RandomState(1).randint(0, 300, 150)]
    lens[70], lens[-1] = 5000, 1500
    assert_a_wave_for_each_head(150, 8, 4, 64, 1)
    pages, q = case(lens, [1] * 150, 4, 2, 64, BF)
    P.check(run(pages, q, lens, [1] * 150, padded(pages.table)), *P.attention(q, *pages.kv, lens, [1] * 150))


# ---- long queries ----------------------------------------------------------------------

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,H,G,dtype", [(64, 2, 4, BF), (128, 1, 3, FP), (256, 1, 2, BF), (96, 2, 1, FP)])
@pytest.mark.parametrize("keys", [2048, 4096, KEYS])
@pytest.mark.parametrize("lens,q_lens", [([1500, 40, 1100], [1500, 40, 1030]), ([2040, 1, 700], [1025, 1, 3])])
def test_prompts(lens, q_lens, keys, D, H, G, dtype, causal):
    """Queries of a thousand tokens: a workgroup for each item (2048 keys at most), and shares."""
    pages, q = case(lens, q_lens, H, G, D, dtype)
    got = run(pages, q, lens, q_lens, padded(pages.table, keys=keys), causal)
    P.check(got, *attention_by_heads(q, *pages.kv, lens, q_lens, causal))


def attention_by_heads(q, k, v, lens, q_lens, causal):
    """P.attention, a head's rows at a time."""
    T, HQ, D = q.shape
    scale, at = 1 / math.sqrt(D), 0
    out, err = torch.zeros(T, HQ, D, dtype=torch.float64), torch.zeros(T, HQ, D, dtype=torch.float64)
    for b, (L, n) in enumerate(zip(lens, q_lens)):
        end = (L - n + 1 + torch.arange(n)).clamp(0, L) if causal else torch.full((n,), L)
        hidden = torch.arange(L)[None, :] >= end[:, None]
        for j in range(HQ):
            kk, vv, qq = k[b][:, j // (HQ // k[b].shape[1])].double(), v[b][:, j // (HQ // k[b].shape[1])].double(), q[at:at + n, j].double()
            s = qq @ kk.T * scale
            p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1).nan_to_num(0.0)
            out[at:at + n, j] = p @ vv
            seen = lambda x: x.masked_fill(hidden, 0.0).amax(dim=1, keepdim=True)  # noqa: E731
            ds = scale * (D + 2) * 2.0 ** -24 * seen(qq.abs() @ kk.abs().T) + 4 * 2.0 ** -24 * seen(s.abs())
            rel = 2 * ds + 2.0 ** -16 + 2.0 ** -21 + (120 + end[:, None] / 8) * 2.0 ** -24
            top = torch.where(hidden[..., None], 0.0, vv.abs()).amax(dim=(1, 2))[:, None] if n * L * D < 1 << 24 else vv.abs().max()
            err[at:at + n, j] = rel * (p @ vv.abs()) + end[:, None] * 2.0 ** -38 * p.amax(dim=1, keepdim=True) * top
        at += n
    return out, err


def test_the_plain_form_by_heads():
    lens, q_lens = [9, 70, 3], [5, 33, 7]
    for causal in (True, False):
        pages, q = case(lens, q_lens, 2, 2, 64, BF)
        for a, b in zip(attention_by_heads(q, *pages.kv, lens, q_lens, causal), P.attention(q, *pages.kv, lens, q_lens, causal=causal)):
            assert torch.allclose(a, b, rtol=1e-9, atol=1e-15)
