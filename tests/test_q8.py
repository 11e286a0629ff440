"""The 8-bit KV cache without a GPU: the format's plain implementation, the page layout, refusals."""
import numpy as np
import pytest
import torch

import q8_testlib as Q
from rotorquant_vllm import _lib
from rotorquant_vllm import kernels as K


def test_slot_bytes():
    lib = _lib.load()
    for H in (1, 2, 3, 5, 8, 64):
        for D in (64, 128):
            assert K.q8_slot_bytes(H, D) == Q.slot_bytes(H, D) == lib.rq_q8_slot_bytes(H, D)
            for block in (16, 48, 64):  # a page holds its codes and scales, in whole 128-byte lines
                page = block * Q.slot_bytes(H, D)
                assert page % 128 == 0 and page >= block // 16 * H * (32 * D + 16)
    assert K.q8_slot_bytes(8, 128) == 2056 and lib.rq_q8_slot_bytes(0, 128) == 0


def test_slot_bytes_past_32_bits():
    assert _lib.load().rq_q8_slot_bytes(1 << 20, 1 << 20) == 0
    assert _lib.load().rq_q8_slot_bytes(1 << 20, 1 << 9) == (1 << 20) * 1025


@pytest.mark.parametrize("D,H,block", [(64, 1, 16), (128, 3, 32)])
def test_page_bytes_are_used_once(D, H, block):
    k, v, s = Q.code_index(block, H, D)
    used = np.concatenate([k.ravel(), v.ravel()])
    assert len(np.unique(used)) == len(used) == 2 * block * H * D
    first_scale = 4 * s.min()
    assert used.max() < first_scale == block // 16 * H * 32 * D
    assert 4 * s.max() + 16 <= block * Q.slot_bytes(H, D)


def test_rounding_of_the_plain_codes():
    """Against torch's e4m3 conversion, and numpy's rint."""
    x = np.concatenate([np.linspace(-448, 448, 100001), np.random.RandomState(0).randn(20000) * 2.0 ** np.random.RandomState(1).randint(-12, 8, 20000)])
    x = x.astype(np.float32).astype(np.float64)
    want = torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(Q.round_code("fp8", x), want)
    assert np.array_equal(Q.round_code("int8", np.array([0.5, 1.5, -0.5, 126.5, 300, np.nan, np.inf])), [0, 2, 0, 126, 127, 0, 127])
    for fmt in ("int8", "fp8"):
        assert Q.exponent(fmt, 0.0) == -40 and Q.exponent(fmt, 1e38) == 60
        assert Q.exponent(fmt, Q.LARGEST[fmt]) == 0 and Q.exponent(fmt, Q.LARGEST[fmt] * 1.001) == 1


ATTN = dict(q=None, dtype=1, total=1, hq=32, qst=4096, qsh=128, cu=None, ns=1, mq=1, causal=1, kv=16, nb=1, bs=16, sb=16 * 2056, h=8, d=128, fmt=0,
            bt=16, mb=1, bts=1, sl=16, msl=16, scale=0.1, out=None, ost=4096, osh=128, ws=None, wsb=0, stream=None)
STORE = dict(k=16, v=16, dtype=1, n=1, kst=1024, ksh=128, vst=1024, vsh=128, h=8, d=128, fmt=0, slots=16, kv=16, nb=1, bs=16, sb=16 * 2056, ws=None,
             wsb=0, stream=None)
READ = dict(kv=16, nb=1, bs=16, sb=16 * 2056, h=8, d=128, fmt=0, bt=16, mb=1, bts=1, sl=16, starts=16, ns=1, total=16, ok=16, ov=16, dtype=1, stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(fmt=2), b"format"), (dict(d=96), b"head_dim"), (dict(d=256), b"head_dim"), (dict(h=0), b"num_kv_heads"), (dict(bs=8), b"block_size"),
    (dict(bs=24), b"block_size"), (dict(sb=16 * 2048), b"pages must be"), (dict(sb=16 * 2056 + 8), b"pages must be"), (dict(kv=24), b"aligned"),
    (dict(kv=None), b"aligned"), (dict(nb=1 << 40), b"num_blocks")])
def test_c_abi_refuses_bad_caches(change, msg):
    """Before any device work, in every entry point; the pointers here are never read."""
    lib = _lib.load()
    for fn, base in ((lib.rq_q8_attention, ATTN), (lib.rq_q8_store, STORE), (lib.rq_q8_read, READ)):
        assert fn(*{**base, **change}.values()) == 1 and msg in lib.rq_last_error(), (fn.__name__, change, lib.rq_last_error())


@pytest.mark.parametrize("change,status,msg", [
    (dict(dtype=2), 1, b"f16 or bf16"), (dict(hq=33), 1, b"multiple"), (dict(total=2), 1, b"one query token"), (dict(mq=2), 1, b"one query token"), (dict(scale=float("nan")), 1, b"finite"),
    (dict(scale=float("inf")), 1, b"finite"), (dict(mq=-1), 1, b"bad sizes"), (dict(ns=65536, total=65536), 1, b"bad sizes"), (dict(nb=0), 1, b"no pages"),
    (dict(), 1, b"null"), (dict(q=8, out=16), 1, b"16-byte"), (dict(q=16, out=16, qst=4100), 1, b"16-byte"), (dict(q=16, out=12), 1, b"8-byte"),
    (dict(q=16, out=16, osh=130), 1, b"8-byte"), (dict(q=16, out=16, mb=1000, msl=16000), 2, b"workspace too small"),
    (dict(q=16, out=16, mb=1000, msl=16000, ws=8, wsb=1 << 30), 1, b"aligned"),
    (dict(q=16, out=16, mb=1000, msl=16000, ws=None, wsb=1 << 30), 1, b"aligned"),
    (dict(ns=0, total=0), 0, None), (dict(total=0, cu=16), 0, None), (dict(mq=0), 0, None)])
def test_c_abi_refuses_bad_attention(change, status, msg):
    lib = _lib.load()
    assert lib.rq_q8_attention(*{**ATTN, **change}.values()) == status
    assert msg is None or msg in lib.rq_last_error(), lib.rq_last_error()


@pytest.mark.parametrize("change,status,msg", [
    (dict(dtype=3), 1, b"dtype"), (dict(n=-1), 1, b"n_tokens"), (dict(n=1 << 30), 1, b"n_tokens"), (dict(n=(1 << 27) + 1), 1, b"n_tokens"), (dict(k=None), 1, b"null"), (dict(slots=None), 1, b"null"),
    (dict(v=18), 1, b"16-byte"), (dict(kst=1028), 1, b"16-byte"), (dict(dtype=2, ksh=130), 1, b"16-byte"), (dict(n=513), 2, b"workspace too small"),
    (dict(n=513, ws=20, wsb=1 << 20), 1, b"aligned"), (dict(n=0), 0, None), (dict(nb=0), 0, None)])
def test_c_abi_refuses_bad_stores(change, status, msg):
    lib = _lib.load()
    assert lib.rq_q8_store(*{**STORE, **change}.values()) == status
    assert msg is None or msg in lib.rq_last_error(), lib.rq_last_error()


@pytest.mark.parametrize("change,status,msg", [
    (dict(dtype=3), 1, b"dtype"), (dict(ns=-1), 1, b"bad sizes"), (dict(total=1 << 40), 1, b"bad sizes"), (dict(ns=1 << 24, h=200, sb=1 << 20), 1, b"too many rows"), (dict(starts=None), 1, b"null"),
    (dict(ok=8), 1, b"16-byte"), (dict(ns=0), 0, None), (dict(total=0), 0, None), (dict(mb=0), 0, None)])
def test_c_abi_refuses_bad_reads(change, status, msg):
    lib = _lib.load()
    assert lib.rq_q8_read(*{**READ, **change}.values()) == status
    assert msg is None or msg in lib.rq_last_error(), lib.rq_last_error()


def test_workspaces():
    lib = _lib.load()
    assert lib.rq_q8_store_workspace_bytes(512, 1 << 20, 16) == 0
    assert lib.rq_q8_store_workspace_bytes(513, 100, 32) >= 4 * (200 + 2 * 513)
    assert lib.rq_q8_attention_workspace_bytes(64, 32, 8, 128, 1, 1000) == 0  # a workgroup per item
    assert 0 < lib.rq_q8_attention_workspace_bytes(1, 32, 8, 128, 1, 8192) <= lib.rq_q8_attention_workspace_bytes(64, 32, 8, 128, 1, 8192)
    assert lib.rq_q8_attention_workspace_bytes(0, 32, 8, 128, 1, 8192) == 0


def test_python_refusals():
    cache = torch.zeros(2, 16, K.q8_slot_bytes(2, 128), dtype=torch.uint8)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: K.q8_store(k, k, cache, torch.zeros(3, dtype=torch.int64)),
                 lambda: K.q8_read(cache, i[None], i, i, 2, 128, torch.float16, total=3),
                 lambda: K.q8_attention(k[:1], cache, i[None], i, 2, 128)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="multiple of 2 heads"):
        K.q8_attention(torch.zeros(1, 3, 128), cache, i[None], i, 2, 128)
    from rotorquant_vllm.kernels import q8
    with pytest.raises(ValueError, match="'int8' or 'fp8'"):
        q8._format("int4")
    with pytest.raises(ValueError, match="uint8 tensor"):
        q8._check_cache(cache.float(), 2, 128)
    with pytest.raises(ValueError, match="cache slots of"):
        q8._check_cache(cache, 3, 128)
    with pytest.raises(ValueError, match="contiguous"):
        q8._check_cache(cache.transpose(0, 1), 2, 128)
    with pytest.raises(RuntimeError, match="no CPU path"):
        q8._device_index(cache)
    with pytest.raises(ValueError, match="block_table must be"):
        q8._index(i.long()[None], "block_table", torch.int32, 2)


# ---- backend ------------------------------------------------------------------


def _impl(monkeypatch, fmt="int8", heads=8, head_size=128, kv_heads=2):
    monkeypatch.setenv("RQ_CACHE_8BIT", fmt)
    monkeypatch.delenv("RQ_DENSE_3BIT", raising=False)
    from rotorquant_vllm.vllm import rq_backend as B
    return B, B.RQAttentionImpl(heads, head_size, 0.1, num_kv_heads=kv_heads)


def test_backend_environment(monkeypatch):
    from rotorquant_vllm.vllm import rq_backend as B
    for off in (None, ""):
        monkeypatch.delenv("RQ_CACHE_8BIT", raising=False) if off is None else monkeypatch.setenv("RQ_CACHE_8BIT", off)
        assert B._parse_cache_8bit() is None
        assert B.RQAttentionBackend.get_kv_cache_shape(7, 16, 4, 128) == (7, 16, 1024)
    monkeypatch.setenv("RQ_CACHE_8BIT", "FP8")
    assert B._parse_cache_8bit() == "fp8"
    assert B.RQAttentionBackend.get_kv_cache_shape(100, 32, 8, 128) == (100, 32, 2056)
    assert B.RQFullAttentionSpec(block_size=32, num_kv_heads=8, head_size=128, dtype=torch.uint8).real_page_size_bytes == 32 * 2056
    with pytest.raises(ValueError, match="multiple of 16"):
        B.RQAttentionBackend.get_kv_cache_shape(100, 8, 8, 128)
    monkeypatch.setenv("RQ_DENSE_3BIT", "1")
    with pytest.raises(ValueError, match="two cache layouts"):
        B._parse_cache_8bit()
    monkeypatch.setenv("RQ_CACHE_8BIT", "int4")
    with pytest.raises(ValueError, match="RQ_CACHE_8BIT must be"):
        B._parse_cache_8bit()


def test_backend_shapes(monkeypatch):
    B, impl = _impl(monkeypatch, "int8", 34, 64, 2)  # any GQA group
    assert impl._q8_format == "int8" and not impl._fused_paged_available
    with pytest.raises(ValueError, match="head_size 64 or 128"):
        _impl(monkeypatch, "int8", 8, 96, 2)
    with pytest.raises(ValueError, match="query heads over"):
        _impl(monkeypatch, "int8", 9, 128, 2)
    support = B.RQMetadataBuilder.get_cudagraph_support
    spec = lambda d: B.RQFullAttentionSpec(block_size=16, num_kv_heads=2, head_size=d, dtype=torch.uint8)  # noqa: E731
    if B._fused_paged_kernel_available:
        assert support(None, spec(64)) == support(None, spec(128)) == B.AttentionCGSupport.UNIFORM_SINGLE_TOKEN_DECODE
    assert support(None, spec(96)) == B.AttentionCGSupport.NEVER


@pytest.mark.parametrize("q_lens,max_query_len,want", [
    ([1, 1, 1], 1, [(0, 3, None, 1)]),
    ([1, 3, 2], 3, [(0, 3, 6, 3)]),
    ([1, 1, 5, 300, 1], 300, [(0, 2, None, 1), (2, 3, 308, 5), (3, 5, 308, 300)]),
    ([300, 1], None, [(0, 2, 301, 300)])])
@pytest.mark.parametrize("host", [True, False])
def test_backend_calls(monkeypatch, q_lens, max_query_len, want, host):
    """Which sequences go to which call, with which bounds."""
    from types import SimpleNamespace
    B, impl = _impl(monkeypatch)
    calls, stored = [], []

    def attend(q, kv_cache, block_table, seq_lens, H, D, fmt, sm_scale, causal, cu_seqlens_q, max_q_len, max_seq_len, out):
        b0 = int(block_table[0, 0])
        calls.append((b0, b0 + seq_lens.numel(), None if cu_seqlens_q is None else q.shape[0], max_q_len))
        assert block_table.shape[0] == seq_lens.numel() and (fmt, H, D, sm_scale, causal) == ("int8", 2, 128, 0.1, True)
        assert out.shape == q.shape and out.data_ptr() == (output if cu_seqlens_q is not None else output[b0:]).data_ptr()
        if cu_seqlens_q is None:
            assert q.shape[0] == seq_lens.numel()
        else:
            assert cu_seqlens_q.tolist() == starts[b0:b0 + seq_lens.numel() + 1]
        # host lengths bound the contexts; without them a batch of one call goes by the table's capacity
        assert max_seq_len == (max(lens[b0:b0 + seq_lens.numel()]) if host or len(want) > 1 or max(q_lens) == 300 else None)

    monkeypatch.setattr(B, "_q8_attention_fn", attend)
    monkeypatch.setattr(B, "_q8_store_fn", lambda k, v, cache, slots, fmt: stored.append((k.shape[0], v.shape[0], slots.numel(), fmt)))
    n, lens = sum(q_lens), [600 + i for i in range(len(q_lens))]
    starts = [0] + list(np.cumsum(q_lens))
    q, output = torch.zeros(n + 2, 8, 128), torch.zeros(n + 2, 8, 128)
    k = torch.zeros(n + 2, 2, 128)
    md = SimpleNamespace(num_actual_tokens=n, block_table=torch.arange(len(q_lens), dtype=torch.int32)[:, None].repeat(1, 3),
                         seq_lens=torch.tensor(lens, dtype=torch.int32), query_start_loc=torch.tensor(starts, dtype=torch.int32),
                         slot_mapping=torch.arange(n), max_query_len=max_query_len)
    if host:
        md.rq_query_start_loc_cpu, md.rq_seq_lens_cpu = md.query_start_loc, md.seq_lens
    cache = torch.zeros(4, 16, 520, dtype=torch.uint8)
    assert impl.forward(None, q, k, k, cache, md, output=output) is output
    assert calls == want and stored == [(n, n, n, "int8")]
    impl.forward(None, q, None, None, cache, md, output=output)  # nothing new to store
    assert len(stored) == 1
    md.use_cascade = True
    with pytest.raises(NotImplementedError):
        impl.forward(None, q, k, k, cache, md, output=output)
