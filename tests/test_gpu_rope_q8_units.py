"""rope_q8_store in calls so long that a wave takes two or four units of a group, its angles held and the next unit on its way."""
import numpy as np
import pytest
import torch

import kv16_testlib as P
import q8_testlib as Q
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
BLOCK = 32


def tokens_of(units, per_cu):
    """Tokens whose groups have per_cu units or a few more for each CU (a unit: a head, or one of its sides for heads of 128)."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return 16 * (-(-per_cu * cus // units) + 1) + 5


def turns(n, H, D, rot, dtype, table, fmt, neox, padded=True):
    """Two calls' (q, k, v, positions, cos_sin, slots) for one cache: groups begun, and groups gone on with."""
    pages = n // BLOCK + 3
    for turn in range(2):
        g = P.gen(n + turn)
        q, k, v = (torch.randn(n, h, D, generator=g) for h in (2, H, H))
        k = k * (1 + (torch.randn(H, D, generator=g) * 3).abs())
        positions = torch.randint(0, 900, (n,), generator=g)
        slots = np.random.RandomState(n + turn).permutation(pages * BLOCK)[:n].astype(np.int64)
        slots[::7] = -1 if padded else slots[::7]
        if turn == 0:
            slots.sort()  # (whole groups, most of them)
        yield pages, (*(x.to(dtype) for x in (q, k, v)), positions, P.table(900, rot, table), torch.from_numpy(slots))


# (kv heads, D, rotated dims, halves): a unit is a head of 64, or a side of one of 128; 53 units and 54 are no multiples of four, 53 none of two
FORMS = [(27, 128, 128, True), (27, 128, 64, False), (27, 128, 64, True), (27, 128, 48, True), (53, 64, 64, True), (53, 64, 16, False), (53, 64, 32, True)]


@pytest.mark.parametrize("per_cu", [12, 24])
@pytest.mark.parametrize("fmt,dtype,table", [("int8", BF, F32), ("fp8", FP, FP), ("int8", F32, F32)])
@pytest.mark.parametrize("H,D,rot,neox", FORMS)
def test_bytes_of_the_store_of_rotated_keys(H, D, rot, neox, fmt, dtype, table, per_cu):
    n = tokens_of(H * (D // 64), per_cu)
    assert n > 512
    ours = theirs = None
    for pages, (q, k, v, positions, cos_sin, slots) in turns(n, H, D, rot, dtype, table, fmt, neox):
        if ours is None:
            ours, theirs = (torch.zeros(pages, BLOCK, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV) for _ in range(2))
        dev = [x.to(DEV) for x in (q, k, v, positions, cos_sin)]
        turned = P.rotate(dev[1].cpu(), positions, cos_sin, neox, F32).to(DEV)
        out = K.rope_q8_store(*dev, ours, slots.to(DEV), fmt=fmt, neox=neox)
        K.q8_store(turned, v.float().to(DEV), theirs, slots.to(DEV), fmt=fmt)
        assert torch.equal(out.cpu(), P.rotate(q, positions, cos_sin, neox, F32).to(dtype))
        assert torch.equal(ours, theirs) and bool(ours.any())


@pytest.mark.parametrize("H,D,rot,neox,fmt,per_cu", [(53, 64, 32, True, "int8", 24), (27, 128, 128, True, "fp8", 12)])
def test_bytes_of_the_plain_implementation(H, D, rot, neox, fmt, per_cu):
    n, ref = tokens_of(H * (D // 64), per_cu), None
    for pages, (q, k, v, positions, cos_sin, slots) in turns(n, H, D, rot, BF, F32, fmt, neox):
        if ref is None:
            cache, ref = torch.zeros(pages, BLOCK, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV), Q.Cache(pages, BLOCK, H, D, fmt)
        K.rope_q8_store(None, *(x.to(DEV) for x in (k, v, positions, cos_sin)), cache, slots.to(DEV), fmt=fmt, neox=neox)
        ref.store(P.rotate(k, positions, cos_sin, neox, F32), v.float(), slots.numpy())
        assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), fmt)
