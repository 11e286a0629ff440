"""Layers of other shapes over prompts of a thousand tokens, which kv16_attention takes by workgroups for items or by shares."""
import numpy as np
import pytest
import torch

from rotorquant_vllm.vllm import rq_backend as B
from test_gpu_rope_backend import impl, metadata, new_cache, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("HQ,H,D", [(8, 2, 64), (4, 2, 256), (20, 1, 128)])
def test_long_prompts(monkeypatch, HQ, H, D, dtype):
    """Prompts beside decodes, then a chunk behind its prefix, against the device matmuls: the rotated outputs are rounded once by each, so that they differ by a step
    at most where both are within half of one, are turned back by orthogonal 4 x 4 blocks and rounded again."""
    layer, pages = impl(monkeypatch, HQ, H, D), 300
    table, cache = np.random.RandomState(2).permutation(pages).astype(np.int32).reshape(2, 150), new_cache(H, D, pages)
    calls, real = [], B._kv16_attention_fn
    lens = [0, 0]
    for step, new in enumerate(([1100, 5], [1, 1030], [1200, 1])):
        lens = [a + b for a, b in zip(lens, new)]
        md = metadata(new, lens, table)
        q, k, v = tokens(sum(new), HQ, H, D, step, dtype)
        got, want = torch.full_like(q, 7.0), torch.zeros_like(q)
        calls.clear()
        with monkeypatch.context() as m:
            m.setattr(B, "_kv16_attention_fn", lambda *a, **kw: calls.append(a[0].shape[0]) or real(*a, **kw))
            layer.forward(None, q, k, v, cache, md, output=got)
        assert calls == [sum(new)]
        with monkeypatch.context() as m:
            m.setattr(layer, "_plain_kernel", lambda *a: False)
            layer.forward(None, q, None, None, cache, md, output=want)
        step_of, want32 = torch.finfo(dtype).eps, want.float()
        blocks = want32.reshape(*want.shape[:-1], D // 4, 4).norm(dim=-1, keepdim=True).expand(*want.shape[:-1], D // 4, 4).reshape(want.shape)
        assert bool(((got.float() - want32).abs() <= 2 * step_of * blocks + step_of * want32.abs() + 1e-6).all())
