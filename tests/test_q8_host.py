"""Host side of the 8-bit cache without a GPU: sizes of scratch, refusals of the backend, strides."""
import contextlib
import os
import re
import sys
from types import SimpleNamespace

import pytest
import torch

from rotorquant_vllm import _lib
from rotorquant_vllm.kernels import q8


def test_scratch_is_sized_for_the_tensors_device(monkeypatch):
    """Two GPUs of different sizes: each call's scratch by its own, whichever is current, also once the other's is known."""
    current, cus = [0], [64, 256]

    @contextlib.contextmanager
    def device(dev):
        before, current[0] = current[0], dev
        yield
        current[0] = before

    fake = SimpleNamespace(rq_q8_attention_workspace_bytes=lambda *sizes: cus[current[0]] * 1000)
    monkeypatch.setattr(q8._lib, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", device)
    q8._attention_bytes.cache_clear()
    try:
        for dev in (1, 0, 1, 0):
            assert q8._attention_bytes(dev, 4, 32, 8, 128, 1, 9000) == cus[dev] * 1000
        assert current == [0]
    finally:
        q8._attention_bytes.cache_clear()


# ---- backend ------------------------------------------------------------------


def _impl(monkeypatch, **kw):
    monkeypatch.setenv("RQ_CACHE_8BIT", "int8")
    monkeypatch.delenv("RQ_DENSE_3BIT", raising=False)
    from rotorquant_vllm.vllm import rq_backend as B
    return B.RQAttentionImpl(8, 128, 0.1, num_kv_heads=2, **kw)


@pytest.mark.parametrize("kw,name", [
    (dict(sliding_window=256), "sliding_window"), (dict(sliding_window=(255, 0)), "sliding_window"), (dict(sliding_window=(0, 0)), "sliding_window"),
    (dict(logits_soft_cap=30.0), "logits_soft_cap"), (dict(alibi_slopes=[0.5] * 8), "alibi_slopes"), (dict(alibi_slopes=torch.ones(8)), "alibi_slopes")])
def test_backend_refuses_what_the_kernels_do_not_do(monkeypatch, kw, name):
    with pytest.raises(ValueError, match=f"does not support {name}"):
        _impl(monkeypatch, **kw)


def test_backend_refuses_sinks(monkeypatch):
    from rotorquant_vllm.vllm import rq_backend as B
    monkeypatch.setattr(B.RQAttentionImpl, "sinks", torch.zeros(8), raising=False)
    with pytest.raises(ValueError, match="does not support sinks"):
        _impl(monkeypatch)


@pytest.mark.parametrize("kw", [
    {}, dict(sliding_window=None), dict(sliding_window=(-1, -1)), dict(sliding_window=-1), dict(logits_soft_cap=0), dict(logits_soft_cap=0.0),
    dict(alibi_slopes=None)])
def test_backend_takes_what_is_off(monkeypatch, kw):
    assert _impl(monkeypatch, **kw)._q8_format == "int8"


def test_backend_leaves_encoders_to_their_own_attention(monkeypatch):
    """Layers without a cache do not reach these kernels."""
    from rotorquant_vllm.vllm import rq_backend as B
    assert _impl(monkeypatch, sliding_window=(128, 128), attn_type=B.AttentionType.ENCODER_ONLY)._q8_format == "int8"


@pytest.mark.parametrize("dtype,ok", [(torch.float16, True), (torch.bfloat16, True), (torch.float32, False), ("auto", True)])
def test_backend_refuses_models_of_32_bits_when_built(monkeypatch, dtype, ok):
    from rotorquant_vllm.vllm import rq_backend as B
    config = SimpleNamespace(model_config=SimpleNamespace(dtype=dtype))
    monkeypatch.setattr(B, "_HAVE_VLLM", True)
    monkeypatch.setitem(sys.modules, "vllm", SimpleNamespace())
    monkeypatch.setitem(sys.modules, "vllm.config", SimpleNamespace(get_current_vllm_config_or_none=lambda: config))
    if ok:
        assert _impl(monkeypatch)._q8_format == "int8"
    else:
        with pytest.raises(ValueError, match="float16 or bfloat16 model"):
            _impl(monkeypatch)
    config = None  # outside a configuration
    assert _impl(monkeypatch)._q8_format == "int8"


def test_backend_refuses_queries_of_32_bits_while_profiling(monkeypatch):
    """The run without metadata that sizes the cache, not the first request."""
    impl = _impl(monkeypatch)
    q, k = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    out = torch.ones_like(q)
    assert impl.forward(None, q, k, k, None, None, output=out) is out and not out.any()
    with pytest.raises(ValueError, match="float16 or bfloat16 model"):
        impl.forward(None, q.float(), k.float(), k.float(), None, None, output=out.float())


@pytest.mark.parametrize("q_lens", [[1, 0, 1], [0, 1], [0, 0, 1, 1, 0]])
@pytest.mark.parametrize("host", [True, False])
def test_backend_batches_of_decodes_with_idle_sequences(monkeypatch, q_lens, host):
    """A sequence without a token in a batch of decodes: the others' tokens still go to their own contexts."""
    from rotorquant_vllm.vllm import rq_backend as B
    impl, calls = _impl(monkeypatch), []
    monkeypatch.setattr(B, "_q8_store_fn", lambda *a, **k: None)
    monkeypatch.setattr(B, "_q8_attention_fn", lambda q, cache, table, lens, H, D, **kw: calls.append((q, table, lens, kw)))
    n, lens = sum(q_lens), [70 + b for b in range(len(q_lens))]
    starts = [sum(q_lens[:b]) for b in range(len(q_lens) + 1)]
    q = torch.zeros(n, 8, 128, dtype=torch.bfloat16)
    k = torch.zeros(n, 2, 128, dtype=torch.bfloat16)
    md = SimpleNamespace(num_actual_tokens=n, max_query_len=1, block_table=torch.arange(len(q_lens), dtype=torch.int32)[:, None],
                         seq_lens=torch.tensor(lens, dtype=torch.int32), query_start_loc=torch.tensor(starts, dtype=torch.int32),
                         slot_mapping=torch.arange(n))
    if host:
        md.rq_query_start_loc_cpu, md.rq_seq_lens_cpu = md.query_start_loc, md.seq_lens
    impl.forward(None, q, k, k, torch.zeros(4, 16, 520, dtype=torch.uint8), md, output=torch.empty_like(q))
    seen = {}  # query row -> sequence
    for q_, table, lens_, kw in calls:
        cu = kw["cu_seqlens_q"]
        for b in range(lens_.numel()):
            for row in range(*(cu[b:b + 2].tolist() if cu is not None else (b, b + 1))):
                seen[row] = int(table[b, 0])
                assert kw["max_seq_len"] is None or kw["max_seq_len"] >= int(lens_[b])
    assert seen == {starts[b]: b for b, m in enumerate(q_lens) if m}


def test_no_call_needs_more_than_the_bound():
    import random
    lib, rng = _lib.load(), random.Random(3)
    for _ in range(3000):
        D, H, G = rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 32, 128]), rng.choice([1, 4, 7, 8, 17, 200])
        longest = int(2 ** rng.uniform(0, 22))
        bound = lib.rq_q8_attention_workspace_bound(H * G, H, D, longest)
        sizes = (int(2 ** rng.uniform(0, 16)) - 1, H * G, H, D, int(2 ** rng.uniform(0, 15)), rng.choice([longest, rng.randint(0, longest)]))
        need = lib.rq_q8_attention_workspace_bytes(*sizes)
        assert need <= bound, (sizes, need, bound)
        assert bound < max(256 << 20, longest * 800) + (40 << 20)
    assert lib.rq_q8_attention_workspace_bound(0, 0, 128, 100) == lib.rq_q8_attention_workspace_bound(8, 8, 128, -1) == 0


def test_strides_over_one_element_do_not_count():
    assert q8._row_strides((3, 2, 64), (500, 64, 1)) == (500, 64, 1)
    assert q8._row_strides((1, 2, 64), (501, 64, 1)) == (0, 64, 1)
    assert q8._row_strides((3, 1, 64), (64, 5, 1)) == (64, 0, 1)
    assert q8._row_strides((1, 1, 64), (7, 5, 2)) == (0, 0, 2)


def test_the_backend_and_the_library_agree_on_prompts():
    """One number in two languages, and the sizes of scratch change with it: images from there on."""
    from rotorquant_vllm.vllm import rq_backend as B
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rq_abi.h")) as f:
        assert int(re.search(r"#define RQ_Q8_PROMPT_COLUMNS (\d+)", f.read())[1]) == B.RQ_8BIT_PROMPT_COLUMNS
    need, cols = _lib.load().rq_q8_attention_workspace_bytes, B.RQ_8BIT_PROMPT_COLUMNS
    assert need(1, 1, 1, 128, cols - 1, 64) == 0 < need(1, 1, 1, 128, cols, 64)


@pytest.mark.parametrize("scale,status", [(2.0 ** 127, 2), (-2.0 ** 127, 2), (2.0 ** 127 * 1.01, 1), (-3.4e38, 1), (1.4e-45, 2)])
def test_scales_past_the_kernels_range_are_refused(scale, status):
    """In base 2 a scale is 1.44 times as large; 2 (too little scratch) says that it was taken."""
    from test_q8 import ATTN
    assert _lib.load().rq_q8_attention(*{**ATTN, "q": 16, "out": 16, "mb": 1000, "msl": 16000, "scale": scale}.values()) == status, _lib.load().rq_last_error()
