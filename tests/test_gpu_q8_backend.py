"""RQ_CACHE_8BIT in the backend on the GPU: refusals before a store, scratch, batches with idle sequences."""
import math
import types

import numpy as np
import pytest
import torch

import q8_bounds as X
import q8_testlib as Q

pytestmark = pytest.mark.gpu


def backend(monkeypatch, fmt, H, HQ, D):
    monkeypatch.setenv("RQ_CACHE_8BIT", fmt)
    monkeypatch.delenv("RQ_DENSE_3BIT", raising=False)
    from rotorquant_vllm.vllm import rq_backend as B
    return B, B.RQAttentionImpl(HQ, D, 1 / math.sqrt(D), num_kv_heads=H)


def metadata(slots, table, lens, q_lens, host=True):
    md = types.SimpleNamespace(num_actual_tokens=sum(q_lens), max_query_len=max(q_lens), use_cascade=False, block_table=X.i32(table), seq_lens=X.i32(lens),
                               slot_mapping=torch.from_numpy(np.asarray(slots, np.int64)).to(X.DEV), query_start_loc=X.i32(np.concatenate([[0], np.cumsum(q_lens)])))
    if host:
        md.rq_seq_lens_cpu, md.rq_query_start_loc_cpu = md.seq_lens.cpu(), md.query_start_loc.cpu()
    return md


def test_queries_of_32_bits_are_refused_before_the_store(monkeypatch):
    H, HQ, D, block = 2, 8, 128, 16
    _, impl = backend(monkeypatch, "int8", H, HQ, D)
    cache = X.new_cache(2, block, H, D)
    k, v = (x.to(X.DEV) for x in Q.rows(1, H, D, 1, torch.float32))
    q = torch.zeros(1, HQ, D, device=X.DEV)
    with pytest.raises(ValueError, match="float16 or bfloat16 model"):
        impl.forward(None, q, k, v, cache, metadata([16], [[1]], [1], [1]), output=torch.empty_like(q))
    assert not cache.any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("host", [True, False])
def test_decodes_beside_idle_sequences(monkeypatch, fmt, host):
    H, HQ, D, block = 2, 8, 128, 16
    _, impl = backend(monkeypatch, fmt, H, HQ, D)
    lens, q_lens = [40, 25, 33, 60], [1, 0, 1, 0]
    cache, ref, table = X.filled(lens, block, H, D, fmt, torch.bfloat16, 9)
    q = torch.randn(2, HQ, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    want, tol = X.attention(q, ref, table, lens, cu)
    out = torch.zeros_like(q, device=X.DEV)
    impl.forward(None, q.to(X.DEV), None, None, cache, metadata([-1, -1], table, lens, q_lens, host), output=out)
    X.check(out, want, tol)


def test_profiling_sets_the_scratch_of_the_largest_call_aside(monkeypatch):
    """The run without metadata reaches the memory that a call over the longest context then needs."""
    H, HQ, D = 8, 32, 128
    _, impl = backend(monkeypatch, "int8", H, HQ, D)
    q = torch.zeros(16, HQ, D, dtype=torch.bfloat16, device=X.DEV)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    impl.forward(None, q, q[:, :H], q[:, :H], None, None, output=out)
    assert not out.any()
    from rotorquant_vllm import _lib
    aside = torch.cuda.max_memory_allocated() - before
    assert torch.cuda.memory_allocated() == before
    for seqs, queries, keys in ((1, 8192, 8192), (8, 1000, 4000), (64, 100, 8192), (256, 1, 8192), (5, 40, 8192)):
        assert _lib.load().rq_q8_attention_workspace_bytes(seqs, HQ, H, D, queries, keys) <= aside
