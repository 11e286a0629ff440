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
