"""What the 8-bit cache costs against K and V that nothing rounded: attention in 64 bits over the format's values, no GPU."""
import math

import numpy as np
import pytest
import torch

import oracle as O
import q8_testlib as Q
from rq_inputs import Params

N, H, G, D, QUERIES = 1024, 2, 4, 128, 4


def _inputs(strong, seed):
    """Keys with strong channels (1 + |N(0, 3)| per head and channel), as the timing cases draw them, or plain N(0, 1)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, N, H, D, generator=g)
    if strong:
        x[0] *= 1 + (torch.randn(H, D, generator=g) * 3).abs()
    return x, torch.randn(QUERIES, H * G, D, generator=g).double().numpy()


def _attend(q, kv):
    out = np.zeros(q.shape)
    for h in range(H * G):
        s = q[:, h] @ kv[0][:, h // G].T / math.sqrt(D)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = p / p.sum(1, keepdims=True) @ kv[1][:, h // G]
    return out


def _q8(x, fmt):
    c = Q.Cache(N // Q.GROUP, Q.GROUP, H, D, fmt)
    c.store(x[0], x[1], np.arange(N))
    return c.values(), np.repeat(2.0 ** c.exps.astype(float), Q.GROUP, axis=1)[..., None]  # values, scales by token and head


def _codebook(x, bits):
    p = Params("iso", bits, bits)
    n = p.np()
    sides = []
    for t, bounds, centroids in ((x[0], n["kb"], p.kc), (x[1], n["vb"], p.vc)):
        packed, norms = O.compress(O.to_bits(t.to(torch.float32))[0], "float32", n["rte"], n["rto"], bounds, p.blk)
        sides.append(O.decompress_f32(packed, norms, centroids.numpy()).astype(np.float64) @ p.R.double().numpy())
    return sides


def _errors(strong, seed):
    x, q = _inputs(strong, seed)
    want = _attend(q, x.double().numpy())
    caches = {"bf16": x.bfloat16().double().numpy(), "int8": _q8(x, "int8")[0], "fp8": _q8(x, "fp8")[0], "4 bits": _codebook(x, 4), "3 bits": _codebook(x, 3)}
    return {name: float(np.linalg.norm(_attend(q, kv) - want) / np.linalg.norm(want)) for name, kv in caches.items()}


@pytest.mark.parametrize("strong", [True, False])
def test_error_against_unquantised_attention(strong):
    """An 8-bit cache lies between a 16-bit one and the codebooks, int8 nearer to the former; with strong key channels, whose scale
    the others share, both lose more."""
    e = [_errors(strong, seed) for seed in (1, 2, 3)]
    mean = {name: sum(x[name] for x in e) / len(e) for name in e[0]}
    print({name: round(v, 4) for name, v in mean.items()})
    assert mean["bf16"] < mean["int8"] < mean["fp8"] < mean["4 bits"] < mean["3 bits"]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("strong", [True, False])
def test_error_is_within_the_formats_bound(fmt, strong):
    """Values are off by half a step at most: 2^(e-1) for int8; for e4m3 2^-4 of the value, 2^(e-10) where it is subnormal.  With scores
    off by at most d, weights are off by a factor of exp(+-2 d) at most: |o' - o| <= (exp(2 d) - 1) sum p |v'| + the values' own."""
    x, q = _inputs(strong, 4)
    x64 = x.double().numpy()
    kv, step = _q8(x, fmt)
    half = step / 2 * np.ones(x64.shape) if fmt == "int8" else np.maximum(np.abs(x64) * 2.0 ** -4, step * 2.0 ** -10)
    assert (np.abs(kv - x64) <= half).all()
    for h in range(H * G):
        k, v, hk, hv = x64[0][:, h // G], x64[1][:, h // G], half[0][:, h // G], half[1][:, h // G]
        s = q[:, h] @ k.T / math.sqrt(D)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        d = (np.abs(q[:, h]) @ hk.T / math.sqrt(D)).max(1, keepdims=True)
        bound = np.expm1(2 * d) * (p @ np.abs(kv[1][:, h // G])) + p @ hv
        off = np.abs(_attend(q, kv)[:, h] - p @ v)
        assert (off <= bound + 1e-12).all()
