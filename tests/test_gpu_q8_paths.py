"""Every form of the 8-bit cache's attention kernels over long contexts: column counts, head sizes, formats, several sequences."""
import functools

import numpy as np
import pytest
import torch

import q8_bounds as X
import q8_testlib as Q
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu


LENGTHS = {"long": (2500, 0, 5, 3100, 1950, 33), "short": (700, 0, 5, 1900, 129, 33)}


@functools.lru_cache(maxsize=2)  # (cases of the same cache follow one another)
def filled(lens, block, H, D, fmt):
    return X.filled(lens, block, H, D, fmt, torch.bfloat16, 29)


# (kv heads, query heads of each, query tokens at most): up to 16 columns, 17 to 32, 33 to 191
COLUMNS = [(2, 4, 1), (2, 4, 3), (2, 4, 8), (2, 4, 20), (4, 7, 2), (4, 7, 4), (4, 7, 11), (1, 17, 1), (1, 17, 11)]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("D,block", [(64, 16), (128, 48)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("H,G,T", COLUMNS)
def test_decodes_and_drafts(H, G, T, fmt, D, block, lengths):
    """Sequences of mixed lengths, one without keys and one of fewer keys than queries: items cut between workgroups under the
    bounds of long contexts, a workgroup each under those of short ones; twice the same bits."""
    lens, queries = LENGTHS[lengths], [T, T, max(1, T - 1), 1, (T + 1) // 2, T]
    cache, ref, table = filled(lens, block, H, D, fmt)
    cu = np.concatenate([[0], np.cumsum(queries)])
    q = torch.randn(int(cu[-1]), H * G, D, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    wide = np.zeros((len(lens), 40000 // block), np.int32)
    wide[:, :table.shape[1]] = table
    for causal in (True, False):
        out, tol = X.attention(q, ref, table, lens, cu, causal)
        for t, bound in ((table, None), (table, max(lens)), (wide, None)):
            args = (q.to(X.DEV), cache, X.i32(t), X.i32(lens), H, D)
            kw = dict(fmt=fmt, causal=causal, cu_seqlens_q=X.i32(cu), max_q_len=T, max_seq_len=bound)
            got = K.q8_attention(*args, **kw)
            X.check(got, out, tol)
            assert torch.equal(got, K.q8_attention(*args, **kw))


@pytest.mark.parametrize("H,G,D,lens,queries", [
    (2, 4, 128, [3000, 90, 0, 2100], [70, 90, 3, 48]), (4, 8, 64, [2300, 2100], [33, 100]), (1, 1, 128, [4100, 700], [193, 260]), (8, 7, 128, [2000], [29])])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_behind_long_prefixes(fmt, causal, H, G, D, lens, queries):
    """The prefill kernels with and without key chunks, by the bound on the lengths."""
    cache, ref, table = X.filled(lens, 16, H, D, fmt, torch.float16, 31)
    cu = np.concatenate([[0], np.cumsum(queries)])
    q = torch.randn(int(cu[-1]), H * G, D, generator=torch.Generator().manual_seed(2)).to(torch.float16)
    out, tol = X.attention(q, ref, table, lens, cu, causal)
    wide = np.zeros((len(lens), 4000), np.int32)
    wide[:, :table.shape[1]] = table
    for t in (table, wide):
        args = (q.to(X.DEV), cache, X.i32(t), X.i32(lens), H, D)
        kw = dict(fmt=fmt, causal=causal, cu_seqlens_q=X.i32(cu), max_q_len=max(queries))
        got = K.q8_attention(*args, **kw)
        X.check(got, out, tol)
        assert torch.equal(got, K.q8_attention(*args, **kw))
