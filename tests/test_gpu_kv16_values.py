"""kv16_attention over values at the ends of their type: infinite ones under weights of any size, huge ones, and ones that cancel."""
import math

import pytest
import torch

import kv16_testlib as P
from test_gpu_kv16_forms import assert_a_wave_for_each_head, case, padded, run

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16

# (length, kv heads, table): an item, shares, shares with a wave for each head
FORMS = [(40, 1, False), (1400, 1, False), (1400, 4, True)]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("bits", [20, 45, 100, 135, 300])
@pytest.mark.parametrize("L,H,wide", FORMS)
def test_infinite_values_of_small_weights(L, H, wide, bits, T, dtype):
    """Infinite V under weights of about 2^-bits of the largest, before its key and behind it: the row's sum is infinite in that dim, with its sign, and a
    NaN where two signs meet; other dims are as without them."""
    D, G, peak, before, behind = 64, 2, L - 20, 3, L - 12
    pages, q = case([L], [T], H, G, D, dtype, seed=7)
    k, v = pages.kv[0][0], pages.kv[1][0]
    k.mul_(0.125)
    k[..., 0] = 0
    k[peak, :, 0] = 64.0
    q[..., 0] = bits * math.log(2) / 64 * math.sqrt(D)
    clean = v.clone()
    for at, dim, x in ((before, 5, math.inf), (behind, 9, -math.inf), (before, 20, math.inf), (behind, 20, -math.inf)):
        v[at, :, dim], clean[at, :, dim] = x, 0.0
    table = padded(pages.table) if wide else None
    if wide:
        assert_a_wave_for_each_head(1, H * G, H, D, T)
    got = run(pages, q, [L], [T], table).cpu()
    want, err = P.attention(q, pages.kv[0], [clean], [L], [T])
    assert bool((got[..., 5] == math.inf).all()) and bool((got[..., 9] == -math.inf).all()) and bool(got[..., 20].isnan().all())
    for x in (got, want, err):
        x[..., [5, 9, 20]] = 0
    P.check(got, want, err)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("L,H,wide", FORMS)
def test_values_near_the_largest(L, H, wide, D, T, dtype):
    """Means of values near the end of their type are no larger than those: no sum on the way overflows."""
    if wide and D == 256 and T > 1:
        T = 3  # (one block of columns)
    pages, q = case([L], [T], H, 2, D, dtype, seed=8)
    v, top = pages.kv[1][0], torch.finfo(dtype).max
    v.copy_((0.97 + 0.03 * torch.rand(v.shape, generator=P.gen(2))) * top)
    v[..., ::3] *= -1
    v[::2, :, 1::3] *= -1
    got = run(pages, q, [L], [T], padded(pages.table) if wide else None)
    P.check(got, *P.attention(q, *pages.kv, [L], [T]))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("L,H,wide", FORMS)
def test_weights_that_cancel(L, H, wide, apart, dtype):
    """Beside a key of weight 1 and V = 0, two of weights w = e^-x and w (1 - d) with V and -V, d of 2^-14 to 2^-11, and all others hidden far below: what
    is left is about w d / 2, and shows the weights' bits.

    x is 1 at most, and u = S scale log2(e) three roundings of 1.5 or less: 3.1 x 2^-24 of the weight; the exponential is off by an ulp, 2^-24, its 16-bit parts
    by less than half of that.  Of two weights, then, 9 x 2^-24, and their sum and l round a few times to 2^-24 of 1 and 2: 13 in all, over l >= 1.7: 8."""
    D, G, T = 64, 8, 5
    pages, q = case([L], [T], H, G, D, dtype, seed=9)
    k, v = pages.kv[0][0], pages.kv[1][0]
    k.zero_()
    k[..., 1] = -2048.0
    top, first, second = (700 % L, 1, L - 9) if apart else (5, 4, 6)
    k[[top, first, second], :, 1] = 0
    k[[first, second], :, 0] = -1.0
    k[second, :, 2] = -1.0
    g = P.gen(3)
    q.zero_()
    q[..., 1] = 8.0
    q[..., 0] = ((0.05 + 0.95 * torch.rand(T, H * G, generator=g)) * math.sqrt(D)).to(dtype)
    q[..., 2] = (2.0 ** (-11 - 3 * torch.rand(T, H * G, generator=g)) * math.sqrt(D)).to(dtype)
    v[top], v[second] = 0, -v[first]
    got = run(pages, q, [L], [T], padded(pages.table) if wide else None).cpu()
    want, _ = P.attention(q, *pages.kv, [L], [T])
    P.check(got, want, (8 * 2.0 ** -24) * v[first].double().abs().repeat_interleave(G, 0)[None])
