"""Layers of other shapes around kv16_attention, with fake kernels (no GPU): which batches go to it and what it is given."""
import math
from types import SimpleNamespace

import pytest
import torch

from rotorquant_vllm.vllm import rq_backend as B

HQ, H, D, BS = 4, 2, 64, 16


@pytest.fixture
def layer(monkeypatch):
    """A 16-bit layer with heads of 64; its calls of kv16_attention, which writes ones, are in layer.calls."""
    for name in ("RQ_MODE", "RQ_BITS", "RQ_ISO_MODE", "RQ_K_BITS", "RQ_V_BITS", "RQ_USE_FUSED_PAGED", "RQ_DENSE_3BIT", "RQ_CACHE_8BIT"):
        monkeypatch.delenv(name, raising=False)
    layer = B.RQAttentionImpl(HQ, D, 1.0 / math.sqrt(D), num_kv_heads=H)
    layer.calls = []

    def decompress(kv_cache, block_table, seq_lens, heads, head_dim, kc, vc, dtype, out_k, out_v, **kw):
        return out_k.zero_(), out_v.zero_(), block_table, None

    def attend(q, k_cache, v_cache, block_table, seq_lens, out, cu_seqlens_q, **kw):
        layer.calls.append(SimpleNamespace(table=block_table, lens=seq_lens, cu=cu_seqlens_q, **kw))
        assert block_table.shape[0] == seq_lens.numel() == cu_seqlens_q.numel() - 1
        out[:int(cu_seqlens_q[-1])] = 1

    monkeypatch.setattr(B, "_paged_decompress_fn", decompress)
    monkeypatch.setattr(B, "_kv16_attention_fn", attend)
    monkeypatch.setattr(layer, "_plain_kernel", lambda *a: True)
    return layer


def metadata(q_lens, lens, tokens, **host):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return SimpleNamespace(num_actual_tokens=tokens, max_query_len=max(q_lens, default=0), use_cascade=False, block_table=i32([[2 * b, 2 * b + 1] for b in range(len(lens))]).view(len(lens), 2),
                           seq_lens=i32(lens), query_start_loc=torch.cat([i32([0]), i32(q_lens).cumsum(0, dtype=torch.int32)]), **host)


def forward(layer, md):
    q = torch.randn(md.num_actual_tokens, HQ, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    cache = torch.zeros(B.RQAttentionBackend.get_kv_cache_shape(8, BS, H, D), dtype=torch.uint8)
    assert layer.forward(None, q, None, None, cache, md, output=out) is out
    return out


def test_a_batch_of_no_sequences(layer):
    """Zeros for the padding, and no call."""
    assert not forward(layer, metadata([], [], 3)).any() and not layer.calls


def test_a_batch_with_padding(layer):
    out = forward(layer, metadata([2, 1], [20, 1], 5))
    assert bool(out[:3].any(-1).all()) and not out[3:].any()
    (call,) = layer.calls
    assert call.max_q_len == 2 and call.max_seq_len == 20 and call.causal and call.cu.tolist() == [0, 2, 3]


@pytest.mark.parametrize("rows", [3, 5])
def test_host_copies_of_the_sequences_that_count(layer, rows):
    """The host's copies name two sequences; the device's tensors go on with a captured batch's idle ones."""
    md = metadata([2, 1] + [0] * (rows - 2), [20, 1] + [0] * (rows - 2), 4)
    md.rq_seq_lens_cpu, md.rq_query_start_loc_cpu = torch.tensor([20, 1], dtype=torch.int32), torch.tensor([0, 2, 3], dtype=torch.int32)
    out = forward(layer, md)
    assert bool(out[:3].any(-1).all()) and not out[3:].any()
    (call,) = layer.calls
    assert call.lens.tolist() == [20, 1] and call.table.tolist() == [[0, 1], [2, 3]] and call.cu.tolist() == [0, 2, 3]


@pytest.mark.parametrize("error", [None, ImportError, RuntimeError, OSError])
def test_without_the_torch_module(monkeypatch, caplog, error):
    """_rq_torch.so missing, or of another torch: the backend says so when it is imported and goes on without the calls that need it."""
    import importlib.util
    import sys

    from rotorquant_vllm import _lib

    there = error is None

    def missing():
        raise error("rotorquant_vllm._rq_torch failed to load: undefined symbol")

    if not there:
        monkeypatch.setattr(_lib, "ops", missing)
    spec = importlib.util.spec_from_file_location("rq_backend_again", B.__file__)
    again = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, "rq_backend_again", again)
    with caplog.at_level("WARNING"):
        spec.loader.exec_module(again)
    assert again._fused_paged_kernel_available and again._compress_store_fn is not None and again._q8_attention_fn is not None
    for name in ("_kv16_attention_fn", "_rope_compress_store_fn", "_rope_q8_store_fn"):
        assert (getattr(again, name) is not None) == there
    assert ("undefined symbol" in caplog.text) == (not there)
    layer = again.RQAttentionImpl(HQ, D, 1.0, num_kv_heads=H)
    assert layer._plain_kernel(SimpleNamespace(is_cuda=True, dtype=torch.bfloat16)) == there
    if not there:  # the matmuls, and a refusal that names what is missing
        x = torch.zeros(1, H, D)
        with pytest.raises(RuntimeError, match="_rq_torch"):
            layer.rope_and_store(x, x, x, torch.zeros(1, dtype=torch.int64), torch.zeros(1, D), True, torch.zeros(1, 16, 512, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64))


@pytest.mark.parametrize("ok,kw", [
    (True, {}), (True, dict(seqs=65535)), (False, dict(seqs=65536)), (True, dict(most=1 << 20)), (False, dict(most=(1 << 20) + 1)),
    (False, dict(most=1 << 20, heads=256)), (True, dict(most=1 << 19, heads=256)), (True, dict(pages=(1 << 26) - 1)), (False, dict(pages=1 << 26)),
    (True, dict(block=65536)), (False, dict(block=65537))])
def test_calls_past_the_kernel(ok, kw):
    """Batches that rq_kv16_attention refuses go to the matmuls, as before there was one."""
    layer = B.RQAttentionImpl(kw.get("heads", HQ), D, 1.0, num_kv_heads=H)
    q = SimpleNamespace(is_cuda=True, dtype=torch.float16, shape=(1, kw.get("heads", HQ), D))
    block = kw.get("block", 4)
    pages = SimpleNamespace(shape=(kw.get("pages", 1), block, H, D))
    assert layer._plain_kernel(q, pages, kw.get("seqs", 1), kw.get("most", 1)) == ok
