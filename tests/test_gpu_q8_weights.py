"""Softmax weights of the 8-bit cache's attention far under the largest one, and scores far from 1."""
import numpy as np
import pytest
import torch

import q8_bounds as X
import q8_testlib as Q
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
FMTS = ["int8", "fp8"]
# (keys, query tokens, head_dim): one launch, shares with a merge, two column blocks of both, prompts, prompts in key chunks
PATHS = [(300, 1, 128), (3000, 1, 64), (300, 2, 64), (3000, 2, 128), (230, 20, 128), (2500, 20, 64)]
GAPS = np.linspace(8.0, 26.0, 12)  # log2 of the sink's weight over the others'


def _case(n, D, fmt, k, v, fix=None):
    table, pages = Q.layout([n], 16, 5)
    ref, cache = Q.Cache(pages, 16, 1, D, fmt), X.new_cache(pages, 16, 1, D)
    slots = Q.slots_of(table, 0, 0, n, 16)
    X.store(cache, ref, k, v, slots, fmt)
    if fix is not None:
        X.store(cache, ref, k[fix], v[fix], slots[fix], fmt)
    return table, ref, cache


def _attend(q, cache, ref, table, n, fmt, sm_scale):
    T = q.shape[0]
    out, tol = X.attention(q, ref, table, [n], [0, T], sm_scale=sm_scale)
    got = K.q8_attention(q.to(X.DEV), cache, X.i32(table), X.i32([n]), 1, q.shape[2], fmt=fmt, sm_scale=sm_scale,
                         cu_seqlens_q=X.i32([0, T]), max_q_len=T)
    return got, out, tol


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,T,D", PATHS)
def test_small_weights_beside_a_sink(fmt, n, T, D):
    """One key takes nearly all of the softmax and has values of 0: the output is that of the others, each of a small weight."""
    g = torch.Generator().manual_seed(n + D)
    k, v = torch.zeros(n, 1, D), torch.rand(n, 1, D, generator=g) * 0.5 + 0.5
    k[0, 0, 0], v[0] = 8.0, 0.0
    table, ref, cache = _case(n, D, fmt, k, v)
    q = torch.zeros(T, len(GAPS), D)
    q[..., 0] = torch.from_numpy(GAPS * np.log(2) / 8)
    got, out, tol = _attend(q.to(torch.float16), cache, ref, table, n, fmt, 1.0)
    assert (np.abs(tol) < 0.05 * np.abs(out)).all()  # the tolerance is under the output's own size
    X.check(got, out, tol)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,T,D", PATHS)
@pytest.mark.parametrize("up", [12, 18, 22])
def test_small_weights_beside_a_scale_held_up(fmt, n, T, D, up):
    """A group whose scale a token raised that was written over since: the groups beside it keep their values."""
    g = torch.Generator().manual_seed(n + D)
    k, v = torch.randn(n, 1, D, generator=g) * 0.1, torch.rand(n, 1, D, generator=g) * 0.5 + 0.5
    v[37] *= 2.0 ** up
    table, pages = Q.layout([n], 16, 5)
    ref, cache = Q.Cache(pages, 16, 1, D, fmt), X.new_cache(pages, 16, 1, D)
    slots = Q.slots_of(table, 0, 0, n, 16)
    X.store(cache, ref, k, v, slots, fmt)
    v[37] *= 2.0 ** -up
    X.store(cache, ref, k[33:40], v[33:40], slots[33:40], fmt)
    q = torch.randn(T, 12, D, generator=g)
    got, out, tol = _attend(q.to(torch.float16), cache, ref, table, n, fmt, None)
    assert (np.abs(tol) < 0.05 * np.abs(out)).all()
    X.check(got, out, tol)


@pytest.mark.parametrize("n,T,D", PATHS)
@pytest.mark.parametrize("sm_scale", [2.0 ** 10, 2.0 ** 17, 2.0 ** 19, 2.0 ** 21])
def test_large_scores(n, T, D, sm_scale):
    """Scores up to 2^26, where their own rounding reaches 8: finite outputs, and the value of a key that stands out."""
    fmt = "int8"
    k, v = Q.rows(n, 1, D, 3, torch.bfloat16, outliers=False)
    table, ref, cache = _case(n, D, fmt, k, v)
    q = torch.randn(T, 12, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    got, out, tol = _attend(q, cache, ref, table, n, fmt, sm_scale)
    assert bool(torch.isfinite(got).all())
    X.check(got, out, tol)
    kv, at = ref.values(), Q.slots_of(table, 0, 0, n, 16)
    plain, alone = got.double().cpu().numpy(), 0
    for i in range(T):
        seen = at[:n - T + i + 1]
        for j in range(12):
            s = kv[0, seen, 0] @ q[i, j].double().numpy() * sm_scale
            # off by this much (fp32 sums of D products, scaled, less the maximum), so that what lies behind has a weight under 2^-40
            ds = (D + 8) * 2.0 ** -24 * float((np.abs(kv[0, seen, 0]) @ np.abs(q[i, j].double().numpy())).max()) * sm_scale
            top = np.sort(s)[-2:]
            if top[1] - top[0] > 2 * ds + 28 + np.log(len(seen)):
                w = kv[1, seen[s.argmax()], 0]
                assert (np.abs(plain[i, j] - w) <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -23) * np.abs(w) + 2.0 ** -30).all()
                alone += 1
    assert alone > 0
