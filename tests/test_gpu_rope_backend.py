"""The backend around rotation and plain pages: rope_and_store before forward, and layers whose shape the fused kernels do not take."""
import math
import types

import numpy as np
import pytest
import torch

import kv16_testlib as P
from rotorquant_vllm import kernels as K
from rotorquant_vllm.vllm import rq_backend as B

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS = 16


def impl(monkeypatch, HQ, H, D, **env):
    for name in ("RQ_MODE", "RQ_BITS", "RQ_ISO_MODE", "RQ_K_BITS", "RQ_V_BITS", "RQ_USE_FUSED_PAGED", "RQ_DENSE_3BIT", "RQ_CACHE_8BIT"):
        monkeypatch.delenv(name, raising=False)
    for name, value in env.items():
        monkeypatch.setenv(name, value)
    return B.RQAttentionImpl(HQ, D, 1.0 / math.sqrt(D), num_kv_heads=H)


def metadata(q_lens, lens, table):
    """One forward's metadata: the last q_lens[b] of lens[b] tokens are new."""
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    slots = [table[b, np.arange(n - t, n) // BS].astype(np.int64) * BS + np.arange(n - t, n) % BS for b, (t, n) in enumerate(zip(q_lens, lens))]
    return types.SimpleNamespace(
        num_actual_tokens=sum(q_lens), max_query_len=max(q_lens), use_cascade=False, slot_mapping=torch.from_numpy(np.concatenate(slots)).to(DEV),
        block_table=i32(table), seq_lens=i32(lens), query_start_loc=i32(np.concatenate([[0], np.cumsum(q_lens)])), max_seq_len=max(lens))


def new_cache(H, D, pages):
    return torch.zeros(B.RQAttentionBackend.get_kv_cache_shape(pages, BS, H, D), dtype=torch.uint8, device=DEV)


def tokens(n, HQ, H, D, seed, dtype=torch.bfloat16):
    g = P.gen(seed)
    return [torch.randn(n, h, D, generator=g).to(dtype).to(DEV) for h in (HQ, H, H)]


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("env", [dict(), dict(RQ_USE_FUSED_PAGED="1", RQ_BITS="4"), dict(RQ_DENSE_3BIT="1"), dict(RQ_CACHE_8BIT="int8"), dict(RQ_CACHE_8BIT="fp8")],
                         ids=["iso3", "fused4", "dense3", "int8", "fp8"])
def test_prompt_then_decodes(monkeypatch, env, neox):
    """Each step: the cache's bytes and the outputs of a forward that is given the rotated fp32 keys (and values in fp32) to store."""
    HQ, H, D, prompts = 8, 2, 128, [40, 7]
    layer, table, cos_sin = impl(monkeypatch, HQ, H, D, **env), np.arange(8, dtype=np.int32).reshape(2, 4)[::-1].copy(), P.table(100, 64, torch.float32).to(DEV)
    ours, theirs, lens = new_cache(H, D, 8), new_cache(H, D, 8), [0, 0]
    for step, new in enumerate((prompts, [1, 1], [1, 1], [3, 2])):
        lens = [a + b for a, b in zip(lens, new)]
        md = metadata(new, lens, table)
        q, k, v = tokens(sum(new), HQ, H, D, step)
        positions = torch.cat([torch.arange(n - t, n) for t, n in zip(new, lens)]).to(DEV)
        turned_q = P.rotate(q.cpu(), positions.cpu(), cos_sin.cpu(), neox, torch.float32).to(q.dtype).to(DEV)
        turned_k = P.rotate(k.cpu(), positions.cpu(), cos_sin.cpu(), neox, torch.float32).to(DEV)
        out, want = torch.zeros_like(q), torch.zeros_like(q)
        got_q = layer.rope_and_store(q, k, v, positions, cos_sin, neox, ours, md.slot_mapping)
        layer.forward(None, got_q, None, None, ours, md, output=out)
        layer.forward(None, turned_q, turned_k, v.float(), theirs, md, output=want)
        assert torch.equal(got_q, turned_q) and torch.equal(ours, theirs) and torch.equal(out, want)
        assert bool(out.any())


def test_padded_steps_and_refusals(monkeypatch):
    layer, cache = impl(monkeypatch, 4, 2, 128), new_cache(2, 128, 3)
    q, k, v = tokens(9, 4, 2, 128, 1)
    cos_sin, positions = P.table(50, 128, torch.float32).to(DEV), torch.arange(9, device=DEV)
    slots = torch.tensor([5, -1, 7, -1, -1], device=DEV)
    got = layer.rope_and_store(q, k, v, positions, cos_sin, True, cache, slots)
    assert got.shape == (5, 4, 128) and torch.equal(got.cpu(), P.rotate(q.cpu()[:5], torch.arange(5), cos_sin.cpu(), True, torch.float32).to(q.dtype))
    assert sorted(cache.view(48, -1).any(-1).nonzero().flatten().tolist()) == [5, 7]
    same = layer.rope_and_store(q[:5], k, v, positions, cos_sin, True, cache, slots, out_q=q[:5])
    assert same.data_ptr() == q.data_ptr() and torch.equal(q[:5], got)
    q, cache = tokens(9, 4, 2, 128, 1)[0], new_cache(2, 128, 3)
    behind = q[5:].clone()
    same = layer.rope_and_store(q, k, v, positions, cos_sin, True, cache, slots, out_q=q)  # (the whole padded batch, in place)
    assert torch.equal(same, got) and torch.equal(q[:5], got) and torch.equal(q[5:], behind)
    with pytest.raises(ValueError, match="encoder"):
        layer.attn_type = B.AttentionType.ENCODER_ONLY
        layer.rope_and_store(q, k, v, positions, cos_sin, True, cache, slots)
    q8 = impl(monkeypatch, 4, 2, 128, RQ_CACHE_8BIT="int8")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        q8.rope_and_store(q.float(), k.float(), v.float(), positions, cos_sin, True, new_cache(2, 128, 3), slots)


# (query heads, kv heads, head size): shapes that the fused kernels do not take
SHAPES = [(8, 2, 64), (6, 3, 96), (4, 1, 256), (20, 1, 128), (34, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_layers_of_other_shapes(monkeypatch, shape, dtype):
    """Prompts, decodes, drafts and mixed batches through kv16_attention against the device matmuls, both within a rounding of the rotated output's type."""
    HQ, H, D = shape
    layer, pages = impl(monkeypatch, HQ, H, D), 40
    table, cache = np.random.RandomState(1).permutation(pages).astype(np.int32).reshape(4, 10), new_cache(H, D, pages)
    calls, real = [], B._kv16_attention_fn
    monkeypatch.setattr(B, "_kv16_attention_fn", lambda *a, **kw: calls.append(a[0].shape[0]) or real(*a, **kw))
    lens = [0, 0, 0, 0]
    for step, new in enumerate(([100, 64, 3, 130], [1, 1, 1, 1], [2, 1, 2, 1], [1, 1, 5, 20])):
        lens = [a + b for a, b in zip(lens, new)]
        md = metadata(new, lens, table)
        q, k, v = tokens(sum(new), HQ, H, D, step, dtype)
        got, want = torch.full_like(q, 7.0), torch.zeros_like(q)
        calls.clear()
        layer.forward(None, q, k, v, cache, md, output=got)
        assert calls == [sum(new)]
        monkeypatch.setattr(layer, "_plain_kernel", lambda *a: False)
        layer.forward(None, q, None, None, cache, md, output=want)
        monkeypatch.undo()
        monkeypatch.setattr(B, "_kv16_attention_fn", lambda *a, **kw: calls.append(a[0].shape[0]) or real(*a, **kw))
        # the rotated output is rounded once by each, so that it may differ by a step where both are within half of one; turned back by an
        # orthogonal 4 x 4 block, and rounded again
        step_of = torch.finfo(dtype).eps
        blocks = want.float().reshape(*want.shape[:-1], D // 4, 4).norm(dim=-1, keepdim=True).expand(*want.shape[:-1], D // 4, 4).reshape(want.shape)
        assert bool(((got.float() - want.float()).abs() <= 2 * step_of * blocks + step_of * want.float().abs() + 1e-6).all())
        same = (got == want).float().mean()
        assert float(same) > 0.9, float(same)


def test_other_shapes_hidden_rows(monkeypatch):
    """Rows whose queries begin before their context: zeros, and no NaN."""
    HQ, H, D = 4, 2, 64
    layer, cache = impl(monkeypatch, HQ, H, D), new_cache(H, D, 4)
    q, k, v = tokens(4, HQ, H, D, 3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    md = types.SimpleNamespace(num_actual_tokens=4, max_query_len=3, use_cascade=False, slot_mapping=torch.tensor([-1, 0, 1, 32], device=DEV),
                               block_table=i32([[0, 1], [2, 3]]), seq_lens=i32([2, 1]), query_start_loc=i32([0, 3, 4]), max_seq_len=2)
    out = torch.full_like(q, 7.0)
    layer.forward(None, q, k, v, cache, md, output=out)
    assert bool((out[0] == 0).all()) and bool(torch.isfinite(out).all()) and bool(out[1:].any(-1).all())


def test_other_shapes_padded_batch(monkeypatch):
    """Rows behind the last sequence are zeros, as the matmuls leave them."""
    HQ, H, D = 4, 2, 64
    layer, cache = impl(monkeypatch, HQ, H, D), new_cache(H, D, 4)
    q, k, v = tokens(5, HQ, H, D, 3)
    md = metadata([2, 1], [2, 1], np.arange(4, dtype=np.int32).reshape(2, 2))
    md.slot_mapping = torch.cat([md.slot_mapping, md.slot_mapping.new_full((2,), -1)])
    md.num_actual_tokens = 5
    out = torch.full_like(q, 7.0)
    layer.forward(None, q, k, v, cache, md, output=out)
    assert bool(out[:3].any(-1).all()) and not out[3:].any()
