"""Scratch that the caller of the 8-bit cache's kernels keeps: sizes, several calls, graphs that share it."""
import numpy as np
import pytest
import torch

import q8_bounds as X
import q8_testlib as Q
from rotorquant_vllm import _lib
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
H, G, D, BLOCK = 2, 4, 128, 16


def _need(*sizes):
    return _lib.load().rq_q8_attention_workspace_bytes(*sizes)


# (sequences, keys, tokens of each): shares, two column blocks, prompts, prompts in key chunks
CALLS = [(3, 4000, 1), (2, 3000, 7), (2, 700, 60), (1, 4000, 50)]


@pytest.mark.parametrize("seqs,keys,T", CALLS)
def test_a_callers_scratch(seqs, keys, T):
    """Just enough, with anything in it, and more: the results of a call without; too little or another type: refused."""
    lens = [keys - 100 * b for b in range(seqs)]
    cache, ref, table = X.filled(lens, BLOCK, H, D, "fp8", torch.bfloat16, 3)
    q = torch.randn(seqs * T, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(X.DEV)
    args = (q, cache, X.i32(table), X.i32(lens), H, D)
    kw = dict(fmt="fp8", cu_seqlens_q=X.i32(np.arange(seqs + 1) * T), max_q_len=T)
    want = K.q8_attention(*args, **kw)
    need = _need(seqs, H * G, H, D, T, table.shape[1] * BLOCK)
    assert need > 0
    for size, fill in ((need, 0xff), (need, 0), (need + 4096, 0x7f)):
        ws = torch.full((size + 64,), fill, dtype=torch.uint8, device=X.DEV)
        for _ in range(2):
            assert torch.equal(K.q8_attention(*args, workspace=ws[:size], **kw), want)
        assert bool((ws[size:] == fill).all())
    with pytest.raises(RuntimeError, match="workspace too small"):
        K.q8_attention(*args, workspace=ws[:need - 1], **kw)
    with pytest.raises(ValueError, match="contiguous uint8"):
        K.q8_attention(*args, workspace=ws.view(torch.int32), **kw)
    with pytest.raises(ValueError, match="16-byte aligned"):
        K.q8_attention(*args, workspace=ws[8:], **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.q8_attention(*args, workspace=torch.zeros(need, dtype=torch.uint8), **kw)


def test_a_callers_scratch_of_a_long_store():
    n, pages = 1500, 100
    k, v = Q.rows(n, H, D, 3, torch.bfloat16)
    slots = np.random.RandomState(1).permutation(pages * BLOCK)[:n]
    need = _lib.load().rq_q8_store_workspace_bytes(n, pages, BLOCK)
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device=X.DEV)
    for _ in range(2):
        cache, ref = X.new_cache(pages, BLOCK, H, D), Q.Cache(pages, BLOCK, H, D, "int8")
        K.q8_store(k.to(X.DEV), v.to(X.DEV), cache, torch.from_numpy(slots).to(X.DEV), workspace=ws[:need])
        ref.store(k, v, slots)
        assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), "int8")
        assert bool((ws[need:] == 0xff).all())
    with pytest.raises(RuntimeError, match="workspace too small"):
        K.q8_store(k.to(X.DEV), v.to(X.DEV), cache, torch.from_numpy(slots).to(X.DEV), workspace=ws[:need - 1])


def test_two_graphs_that_share_scratch():
    """A decode and a prompt, captured apart with one buffer, replayed in turn with other lengths and eager work between."""
    lens = [4000, 300]
    cache, ref, table = X.filled(lens, BLOCK, H, D, "int8", torch.bfloat16, 3)
    bt, sl = X.i32(table), X.i32(lens)
    calls, need = [], 0
    for T in (1, 60):
        q = torch.randn(2 * T, H * G, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(X.DEV)
        calls.append(dict(q=q, cu_seqlens_q=X.i32([0, T, 2 * T]), max_q_len=T, out=torch.zeros_like(q)))
        need = max(need, _need(2, H * G, H, D, T, table.shape[1] * BLOCK))
    ws = torch.zeros(need, dtype=torch.uint8, device=X.DEV)

    def run(c, **kw):
        c = dict(c, **kw)
        return K.q8_attention(c.pop("q"), cache, bt, sl, H, D, **c)

    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            run(c, workspace=ws)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                run(c, workspace=ws)
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for i, now in enumerate(([4000, 300], [3100, 61], [70, 299], [4000, 0])):
        sl.copy_(torch.tensor(now, dtype=torch.int32))
        for c, g in list(zip(calls, graphs))[::1 if i % 2 else -1]:
            c["out"].fill_(5.0)
            g.replay()
        got = [c["out"].clone() for c in calls]
        for c, x in zip(calls, got):
            assert torch.equal(x, run(c, out=None))
            out, tol = X.attention(c["q"].cpu(), ref, table, now, c["cu_seqlens_q"].tolist())
            X.check(x, out, tol)


def test_long_stores_on_two_streams():
    """Calls that overlap, each to pages of its own, with scratch of their own."""
    n, pages = 3000, 200
    data = [Q.rows(n, H, D, 20 + i, torch.bfloat16) for i in range(2)]
    slots = [np.random.RandomState(i).permutation(pages * BLOCK)[:n] + i * pages * BLOCK for i in range(2)]
    cache, ref = X.new_cache(2 * pages, BLOCK, H, D), Q.Cache(2 * pages, BLOCK, H, D, "fp8")
    on = [[x.to(X.DEV) for x in (*data[i], torch.from_numpy(slots[i]))] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, (k, v, at) in zip(streams, on):
            with torch.cuda.stream(s):
                K.q8_store(k, v, cache, at, fmt="fp8")
    torch.cuda.synchronize()
    for i in range(2):
        ref.store(*data[i], slots[i])
        ref.store(*data[i], slots[i])
    assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), "fp8")
