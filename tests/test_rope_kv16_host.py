"""Position rotation and 16-bit pages without a GPU: refusals of the C entry points, sizes of scratch, the plain implementations."""
import math

import pytest
import torch

import kv16_testlib as P
from rotorquant_vllm import _lib

A = 1 << 20  # an address that is only looked at


def call(name, args, **kw):
    """(status, message) of an entry point with some of its arguments changed.  No launch: every call here is refused or empty."""
    lib = _lib.load()
    args = dict(args, **kw)
    rc = getattr(lib, name)(*args.values())
    return rc, lib.rq_last_error().decode() if rc else ""


ROPE = dict(query=A, key=A, value=A, dtype=1, n_tokens=4, num_q_heads=8, q_st=1024, q_sh=128, k_st=256, k_sh=128, v_st=256, v_sh=128, H=2, D=128,
            positions=A, cos_sin=A, table_dtype=2, table_rows=100, table_stride=128, rot_dim=128, halves=1, out_q=A, o_st=1024, o_sh=128)
STORES = {
    "rq_rope_kv16_store": dict(ROPE, slots=A, k_cache=A, v_cache=A, num_blocks=4, block_size=16, kc_sb=4096, kc_ss=256, kc_sh=128, vc_sb=4096, vc_ss=256,
                               vc_sh=128, stream=None),
    "rq_rope_q8_store": dict(ROPE, format=0, slots=A, kv_cache=A, num_blocks=4, block_size=16, stride_block=16 * 520, ws=None, ws_bytes=0, stream=None),
    "rq_rope_compress_store": dict(ROPE, index_layout=0, slots=A, kv_cache=A, num_blocks=4, block_size=16, stride_block=16 * 512, stride_token=512,
                                   total_bytes=512, rte=A, rto=A, rot_block=4, kb=A, nkb=7, vb=A, nvb=7, stream=None)}


@pytest.mark.parametrize("name", STORES)
@pytest.mark.parametrize("match,kw", [
    ("dtype|must be f16", dict(dtype=3)), ("table must be fp32", dict(table_dtype=0)), ("table must be fp32", dict(table_dtype=7)),
    ("head_dim", dict(D=136)), ("head_dim", dict(D=0)), ("rot_dim 8 must", dict(rot_dim=8)), ("rot_dim 144 must", dict(rot_dim=144)),
    ("rot_dim 0 must", dict(rot_dim=0)), ("rot_dim 24 must", dict(rot_dim=24)), ("bad sizes", dict(n_tokens=-1)), ("bad sizes", dict(n_tokens=1 << 25)),
    ("bad sizes", dict(num_q_heads=-1)), ("bad sizes", dict(table_rows=0)), ("null pointer", dict(positions=None)), ("null pointer", dict(cos_sin=None)),
    ("null pointer", dict(query=None)), ("null pointer", dict(out_q=None)), ("null pointer", dict(key=None)), ("null pointer", dict(value=None)),
    ("null pointer", dict(slots=None)), ("table rows", dict(cos_sin=A + 8)), ("table rows", dict(table_stride=64)), ("table rows", dict(table_stride=130)),
    ("query rows must", dict(query=A + 8)), ("query rows must", dict(out_q=A + 2)), ("query rows must", dict(q_st=1028)), ("query rows must", dict(o_sh=4)),
    ("16-byte aligned", dict(key=A + 2)), ("16-byte aligned", dict(v_sh=4)), ("too many rows", dict(n_tokens=1 << 24, num_q_heads=65536))])
def test_refusals_of_the_stores(name, match, kw):
    import re
    rc, message = call(name, STORES[name], **kw)
    assert rc == 1 and re.search(match, message), message


def test_refusals_of_each_cache():
    for name, match, kw in [
            ("rq_rope_kv16_store", "must be f16", dict(dtype=2)), ("rq_rope_kv16_store", "num_kv_heads", dict(H=0)), ("rq_rope_kv16_store", "cache sizes", dict(block_size=0)),
            ("rq_rope_kv16_store", "null", dict(k_cache=None)), ("rq_rope_kv16_store", "16-byte", dict(vc_sb=4097)), ("rq_rope_kv16_store", "16-byte", dict(k_cache=A + 8)),
            ("rq_rope_q8_store", "head_dim 96", dict(D=96, rot_dim=96)), ("rq_rope_q8_store", "format", dict(format=2)), ("rq_rope_q8_store", "block_size", dict(block_size=8)),
            ("rq_rope_compress_store", "rot_block", dict(rot_block=3)), ("rq_rope_compress_store", "payload", dict(total_bytes=100)),
            ("rq_rope_compress_store", "too many positions", dict(table_rows=1 << 31)), ("rq_rope_compress_store", "head_dim 512", dict(D=512, rot_dim=16)),
            ("rq_rope_compress_store", "null", dict(rte=None))]:
        rc, message = call(name, STORES[name], **kw)
        assert rc == 1 and match in message, (name, message)
    rc, message = call("rq_rope_q8_store", STORES["rq_rope_q8_store"], n_tokens=600)
    assert rc == 2 and "workspace too small" in message
    for name in STORES:
        assert call(name, STORES[name], n_tokens=0)[0] == 0


ATTENTION = dict(q=A, dtype=1, total_q=2, HQ=8, q_st=1024, q_sh=128, cu=None, num_seqs=2, max_q_len=1, causal=1, k=A, v=A, num_blocks=9, block_size=16,
                 kc_sb=4096, kc_ss=256, kc_sh=128, vc_sb=4096, vc_ss=256, vc_sh=128, H=2, D=128, bt=A, max_blocks=4, bt_ss=4, lens=A, max_seq_len=64,
                 scale=0.1, out=A, o_st=1024, o_sh=128, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("match,kw", [
    ("must be f16 or bf16", dict(dtype=2)), ("head_dim 4 must", dict(D=4)), ("head_dim 132 must", dict(D=132)), ("head_dim 264 must", dict(D=264)),
    ("num_kv_heads 0", dict(H=0)), ("multiple of", dict(HQ=7)), ("cache sizes", dict(block_size=0)), ("bad sizes", dict(num_seqs=65536, total_q=65536)),
    ("bad sizes", dict(max_seq_len=-1)), ("without cu_seqlens_q", dict(total_q=3)), ("without cu_seqlens_q", dict(max_q_len=2)),
    ("sm_scale", dict(scale=math.inf)), ("sm_scale", dict(scale=math.nan)), ("sm_scale", dict(scale=2.0 ** 127.5)), ("no pages", dict(num_blocks=0)),
    ("null", dict(q=None)), ("null", dict(out=None)), ("null", dict(k=None)), ("null", dict(lens=None)), ("null", dict(bt=None)),
    ("q rows", dict(q=A + 8)), ("q rows", dict(q_sh=4)), ("out rows", dict(out=A + 4)), ("out rows", dict(o_st=2)), ("cache rows", dict(v=A + 8)),
    ("cache rows", dict(kc_ss=4)), ("within 64 GiB", dict(kc_sb=1 << 33)), ("within 64 GiB", dict(vc_ss=-256)), ("within 64 GiB", dict(num_blocks=1 << 30)),
    ("within 64 GiB", dict(vc_sb=-4096)), ("max_q_len 1048576 with 256", dict(cu=A, max_q_len=1 << 20, HQ=256))])
def test_refusals_of_attention(match, kw):
    rc, message = call("rq_kv16_attention", ATTENTION, **kw)
    assert rc == 1 and match in message, message


def test_attention_without_work_or_scratch():
    for kw in (dict(num_seqs=0, total_q=0), dict(total_q=0, cu=A), dict(max_q_len=0)):
        assert call("rq_kv16_attention", ATTENTION, **kw)[0] == 0
    size = _lib.load().rq_kv16_attention_workspace_bytes
    assert size(2, 8, 2, 128, 1, 512) == 0 and size(0, 8, 2, 128, 1, 9000) == 0 and size(2, 8, 2, 300, 1, 9000) == 0
    assert size(64, 32, 8, 128, 8, 2048) == 0 and size(64, 32, 8, 128, 8, 2049) > 0 and size(1, 32, 8, 128, 8, 513) > 0
    assert size(64, 32, 8, 128, 1, 768) == 0 and size(64, 32, 8, 128, 1, 769) > 0 and size(64, 32, 8, 128, 4, 769) > 0
    need = size(2, 8, 2, 128, 1, 9000)
    assert need > 0 and size(2, 8, 2, 128, 9, 9000) > need and size(2, 8, 2, 128, 1, 1 << 60) >= need
    rc, message = call("rq_kv16_attention", ATTENTION, max_seq_len=9000, max_blocks=1000)
    assert rc == 2 and f"{need} bytes" in message


def test_cpu_tensors_are_refused():
    from rotorquant_vllm import kernels as K
    x, at, table = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int64), torch.zeros(9, 64)
    pages, q8 = torch.zeros(2, 16, 2, 64, dtype=torch.float16), torch.zeros(2, 16, K.q8_slot_bytes(2, 64), dtype=torch.uint8)
    rot = torch.zeros(64, 32)
    for run in (lambda: K.rope_kv16_store(x, x, x, at, table, pages, pages, at), lambda: K.rope_q8_store(x, x, x, at, table, q8, at),
                lambda: K.rope_compress_store(x, x, x, at, table, q8, at, rot, rot, torch.zeros(7), torch.zeros(7)),
                lambda: K.kv16_attention(x, pages, pages, torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            run()


@pytest.mark.parametrize("neox", [True, False])
def test_the_plain_rotation_turns(neox):
    """It keeps lengths and, between two rows, depends on the distance of their positions alone."""
    g = P.gen(1)
    x, y, table = torch.randn(6, 2, 64, generator=g), torch.randn(6, 2, 64, generator=g), P.table(100, 64, torch.float64)
    at = torch.tensor([0, 3, 10, 40, 41, 60])
    a, b = P.rotate(x, at, table, neox), P.rotate(y, at + 30, table, neox)
    assert torch.allclose(a.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-12)
    far = P.rotate(x, at + 5, table, neox), P.rotate(y, at + 35, table, neox)
    assert torch.allclose((a * b).sum(-1), (far[0] * far[1]).sum(-1), rtol=1e-9, atol=1e-9)
    assert P.rotate(x, torch.tensor([-1] + [100] * 5), table, neox).isnan().all()


def test_the_plain_attention():
    """Against torch's softmax attention."""
    g = P.gen(2)
    q, k, v = torch.randn(5, 4, 16, generator=g), torch.randn(9, 2, 16, generator=g), torch.randn(9, 2, 16, generator=g)
    out, err = P.attention(q, [k], [v], [9], [5])
    want = torch.nn.functional.scaled_dot_product_attention(
        q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(2, 0), v.double().transpose(0, 1).repeat_interleave(2, 0),
        attn_mask=torch.arange(9)[None, :] <= 4 + torch.arange(5)[:, None]).transpose(0, 1)
    assert torch.allclose(out, want, rtol=1e-10, atol=1e-12) and bool((err > 0).all()) and float(err.max()) < 1e-3
