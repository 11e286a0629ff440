"""The 8-bit cache's attention at the edges of what its calls allow: query lengths past their bound, tiny scales."""
import numpy as np
import pytest
import torch

import q8_bounds as X
import q8_testlib as Q
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,G,D,lens,queries,most", [
    (2, 4, 128, [40, 30], [10, 3], 4),            # one launch
    (1, 8, 64, [2500, 700], [7, 20], 5),          # shares and a merge
    (1, 4, 128, [200, 90, 120], [130, 90, 60], 60),  # prompts
    (1, 1, 64, [2500], [250], 200)])              # prompts in key chunks
def test_queries_longer_than_their_bound(H, G, D, lens, queries, most, causal):
    """The first max_q_len tokens of each sequence stay at their positions; the others' rows are left as they were."""
    cache, ref, table = X.filled(lens, 16, H, D, "int8", torch.bfloat16, 23)
    cu = np.concatenate([[0], np.cumsum(queries)])
    q = torch.randn(int(cu[-1]), H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, tol = X.attention(q, ref, table, lens, cu, causal)
    got = torch.full(q.shape, 7.0, dtype=q.dtype, device=X.DEV)
    K.q8_attention(q.to(X.DEV), cache, X.i32(table), X.i32(lens), H, D, cu_seqlens_q=X.i32(cu), max_q_len=most, causal=causal, out=got)
    keep = np.concatenate([np.arange(n) < most for n in queries])
    X.check(got[torch.from_numpy(keep).to(X.DEV)], out[keep], tol[keep])
    assert bool((got[torch.from_numpy(~keep).to(X.DEV)] == 7.0).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("T,n", [(1, 5), (1, 2100), (3, 21), (40, 70), (40, 2100)])
@pytest.mark.parametrize("sm_scale", [1e-8, 1e-17, -1e-25, 1e-38, 1.5e-45])
def test_tiny_scales(fmt, T, n, sm_scale):
    """Zero queries and zero keys under a scale near fp32's end: the mean of the values that a row sees."""
    H, G, D = 1, 8, 128
    k, v = Q.rows(n, H, D, 2, torch.bfloat16)
    k[:16] = 0
    k[n // 2:] = 0
    table, pages = Q.layout([n], 16, 5)
    ref, cache = Q.Cache(pages, 16, H, D, fmt), X.new_cache(pages, 16, H, D)
    X.store(cache, ref, k, v, Q.slots_of(table, 0, 0, n, 16), fmt)
    q = torch.randn(T, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[:, ::2] = 0
    q[:, 1] *= 1e-30
    out, tol = X.attention(q, ref, table, [n], [0, T], sm_scale=sm_scale)
    got = K.q8_attention(q.to(X.DEV), cache, X.i32(table), X.i32([n]), H, D, fmt=fmt, cu_seqlens_q=X.i32([0, T]), max_q_len=T, sm_scale=sm_scale)
    X.check(got, out, tol)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_a_tiny_scale_times_large_numbers(fmt):
    """The scale alone says nothing about the scores: 2^-60 times queries of 2^30 and keys of 2^30."""
    H, G, D, n = 1, 8, 64, 50
    k, v = Q.rows(n, H, D, 4, torch.bfloat16)
    table, pages = Q.layout([n], 16, 5)
    ref, cache = Q.Cache(pages, 16, H, D, fmt), X.new_cache(pages, 16, H, D)
    X.store(cache, ref, k * 2.0 ** 30, v, Q.slots_of(table, 0, 0, n, 16), fmt)
    for T in (1, 30):
        q = torch.randn(T, H * G, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16) * 2.0 ** 30
        out, tol = X.attention(q, ref, table, [n], [0, T], sm_scale=2.0 ** -62)
        got = K.q8_attention(q.to(X.DEV), cache, X.i32(table), X.i32([n]), H, D, fmt=fmt, cu_seqlens_q=X.i32([0, T]), max_q_len=T, sm_scale=2.0 ** -62)
        X.check(got, out, tol)


def test_one_row_of_any_stride():
    """One token, and one head, as views whose stride over it is odd: stored, and attended to."""
    D, block = 128, 16
    wide = torch.randn(3, 4 * D + 3, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(X.DEV)
    for H, HQ in ((2, 4), (1, 1)):
        cache, ref = X.new_cache(2, block, H, D), Q.Cache(2, block, H, D, "int8")
        k = torch.as_strided(wide, (1, H, D), (4 * D + 3, D if H > 1 else 5, 1))
        slots = torch.tensor([16], device=X.DEV)
        K.q8_store(k, k, cache, slots)
        ref.store(k.cpu(), k.cpu(), [16])
        assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), "int8")
        q = torch.as_strided(wide, (1, HQ, D), (4 * D + 3, D if HQ > 1 else 7, 1))
        out = torch.as_strided(torch.zeros(5 * D, dtype=torch.bfloat16, device=X.DEV), (1, HQ, D), (9, D if HQ > 1 else 11, 1))
        table = np.array([[1]], np.int32)
        want, tol = X.attention(q.cpu(), ref, table, [1], [0, 1])
        X.check(K.q8_attention(q, cache, X.i32(table), X.i32([1]), H, D, out=out), want, tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,keys", [(1, 60), (1, 2500), (5, 60), (5, 2500), (70, 150), (70, 2500)])
def test_lengths_near_the_end_of_an_int(T, keys, causal):
    """Contexts said to be longer than anything: what the table holds is seen, by every query."""
    H, G, D = 1, 4, 64
    cache, ref, table = X.filled([keys], 16, H, D, "int8", torch.bfloat16, 3)
    table = table[:, :keys // 16]
    q = torch.randn(3 * T, H * G, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    lens, table, cu = [2 ** 31 - 1, 2 ** 31 - 40, -2 ** 31], np.repeat(table, 3, axis=0), [0, T, 2 * T, 3 * T]
    out, tol = X.attention(q, ref, table, lens, cu, causal)
    got = K.q8_attention(q.to(X.DEV), cache, X.i32(table), X.i32(lens), H, D, cu_seqlens_q=X.i32(cu), max_q_len=T, causal=causal)
    X.check(got, out, tol)
    assert not got[2 * T:].any()
