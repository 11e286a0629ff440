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
