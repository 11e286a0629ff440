"""Rotating stores: calls that their documentation allows, against the stores of rotated fp32 keys."""
import numpy as np
import pytest
import torch

import kv16_testlib as P
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def inputs(n, HQ, H, D, rot, seed, rows=500, dtype=BF):
    g = P.gen(seed)
    q, k, v = (torch.randn(n, h, D, generator=g).to(dtype) for h in (HQ, H, H))
    return q, k, v, torch.randint(0, rows, (n,), generator=g), P.table(rows, rot, F32)


def on(*tensors):
    return [x.to(DEV) for x in tensors]


def turned(x, positions, cos_sin, neox=True):
    return P.rotate(x, positions, cos_sin, neox, F32)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n,rot", [(40, 128), (40, 64), (700, 128), (700, 32)])
def test_a_slot_twice_in_the_8_bit_cache(n, rot, fmt, neox):
    """The last of a slot's tokens counts, with its own position."""
    H, D, pages = 3, 128, n // 16 + 2
    q, k, v, positions, cos_sin = inputs(n, 2, H, D, rot, n)
    slots = torch.from_numpy(np.random.RandomState(n).randint(-1, pages * 16, n)).to(DEV)
    ours, theirs = (torch.zeros(pages, 16, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV) for _ in range(2))
    out = K.rope_q8_store(*on(q, k, v, positions, cos_sin), ours, slots, fmt=fmt, neox=neox)
    K.q8_store(turned(k, positions, cos_sin, neox).to(DEV), v.float().to(DEV), theirs, slots, fmt=fmt)
    assert torch.equal(ours, theirs) and torch.equal(out.cpu(), turned(q, positions, cos_sin, neox).to(BF))


def block_rotation(D, width, seed):
    """The transpose's even and odd columns of a rotation by blocks of `width`."""
    R = torch.block_diag(*torch.linalg.qr(torch.randn(D // width, width, width, generator=P.gen(seed), dtype=torch.float64)).Q).float().T.contiguous()
    return R[:, 0::2].contiguous(), R[:, 1::2].contiguous()


BOUNDS = {"sorted": [-0.15, -0.09, -0.04, 0.0, 0.04, 0.09, 0.15], "close": [-0.1, 0.0, 1e-6, 2e-6, 3e-6, 0.05, 0.1], "one": [0.01]}


@pytest.mark.parametrize("width", [2, 4, 8])
@pytest.mark.parametrize("bounds", BOUNDS)
@pytest.mark.parametrize("n,D,rot,dtype", [(9, 64, 32, BF), (300, 128, 128, BF), (1500, 128, 64, F32), (70, 256, 256, F32), (50, 80, 48, BF), (2000, 16, 16, BF)])
def test_rotations_by_blocks_of_any_width(n, D, rot, dtype, bounds, width):
    """Blocks of 8 have a kernel of their own, boundaries that lie close a count without a table; groups of 16, 32 and 64 rows."""
    H, pages, total = 2, n // 16 + 3, 1024
    q, k, v, positions, cos_sin = inputs(n, 1, H, D, rot, n + D, dtype=dtype)
    even, odd = on(*block_rotation(D, width, D))
    kb, vb = torch.tensor(BOUNDS[bounds], device=DEV), torch.tensor(BOUNDS["sorted"], device=DEV)
    slots = torch.from_numpy(np.random.RandomState(n).permutation(pages * 16)[:n].astype(np.int64)).to(DEV)
    ours, theirs = (torch.full((pages, 16, total), 5, dtype=torch.uint8, device=DEV) for _ in range(2))
    for neox in (True, False):
        K.rope_compress_store(*on(q, k, v, positions, cos_sin), ours, slots, even, odd, kb, vb, neox=neox, rot_block=width)
        K.compress_store(turned(k, positions, cos_sin, neox).to(DEV), v.float().to(DEV), theirs, slots, even, odd, kb, vb, rot_block=width)
        assert torch.equal(ours, theirs) and bool((ours != 5).any())


def test_no_tokens_no_queries_and_a_table_of_one_row():
    H, D = 2, 64
    pages = torch.zeros(2, 3, 16, H, D, dtype=BF, device=DEV)
    for n, HQ, rows in ((0, 4, 9), (5, 0, 9), (5, 4, 1)):
        q, k, v, positions, cos_sin = inputs(n, HQ, H, D, 32, n, rows)
        pages.zero_()
        out = K.rope_kv16_store(*on(q, k, v, positions, cos_sin), pages[0], pages[1], torch.arange(n, device=DEV) + 7)
        assert out.shape == q.shape and torch.equal(out.cpu(), turned(q, positions, cos_sin).to(BF))
        flat = pages.cpu().view(2, 48, H, D)
        assert torch.equal(flat[0, 7:7 + n], turned(k, positions, cos_sin).to(BF)) and torch.equal(flat[1, 7:7 + n], v)
        assert not flat[:, :7].any() and not flat[:, 7 + n:].any()


def test_attention_of_nothing():
    """No sequences, no tokens, no pages in the table, a bound of 0 on the queries."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q, pages = torch.randn(3, 4, 64, device=DEV).to(BF), torch.randn(2, 2, 16, 2, 64, device=DEV).to(BF)
    assert K.kv16_attention(q[:0], *pages, torch.zeros(0, 2, dtype=torch.int32, device=DEV), i32()).shape == (0, 4, 64)
    out = torch.full_like(q, 3.0)
    assert bool((K.kv16_attention(q, *pages, torch.zeros(0, 2, dtype=torch.int32, device=DEV), i32(), cu_seqlens_q=i32(0), out=out) == 3).all())
    assert bool((K.kv16_attention(q, *pages, torch.zeros(2, 2, dtype=torch.int32, device=DEV), i32(9, 9), cu_seqlens_q=i32(0, 2, 3), max_q_len=0, out=out) == 3).all())
    got = K.kv16_attention(q, *pages, torch.zeros(3, 0, dtype=torch.int32, device=DEV), i32(9, 9, 0), out=out)
    assert got is out and not out.any()
