"""Position rotation on the way into the caches (rope_compress_store, rope_q8_store, rope_kv16_store) against plain implementations."""
import numpy as np
import pytest
import torch

import kv16_testlib as P
import oracle as O
import q8_testlib as Q
from rotorquant_vllm import kernels as K
from rq_testlib import Params

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
POSITIONS = 5000


def inputs(n, HQ, H, D, rot, dtype, table, seed, far=POSITIONS):
    """(q, k, v, positions, cos_sin) on the host."""
    g = P.gen(seed)
    q, k, v = (torch.randn(n, h, D, generator=g) for h in (HQ, H, H))
    k = k * (1 + (torch.randn(H, D, generator=g) * 3).abs())
    positions = torch.randint(0, far, (n,), generator=g)
    return (*(x.to(dtype) for x in (q, k, v)), positions, P.table(POSITIONS, rot, table))


def on(*tensors):
    return [x.to(DEV) for x in tensors]


def distinct_slots(n, slots, seed, padded=0):
    s = np.random.RandomState(seed).permutation(slots)[:n].astype(np.int64)
    if padded:
        s[np.random.RandomState(seed + 1).permutation(n)[:padded]] = -1
    return s


def same(a, b):
    """Equal values, and NaN in the same places."""
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# (tokens, query heads, kv heads, D, rotated dims)
SHAPES = [(1, 4, 1, 128, 128), (3, 32, 8, 128, 128), (17, 28, 4, 64, 64), (33, 2, 2, 128, 64), (5, 7, 7, 96, 96), (9, 1, 1, 16, 16),
          (70, 16, 1, 256, 256), (21, 4, 2, 80, 16), (600, 8, 2, 128, 32), (2, 5, 5, 512, 512)]


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype,table", [(BF, F32), (BF, BF), (FP, FP), (FP, F32)])
@pytest.mark.parametrize("shape", SHAPES)
def test_pages(shape, dtype, table, neox):
    """Queries and 16-bit pages: the elementary fp32 formula's numbers, and within its roundings of the one in 64 bits."""
    n, HQ, H, D, rot = shape
    q, k, v, positions, cos_sin = inputs(n, HQ, H, D, rot, dtype, table, n + D)
    block, pages = 16, n // 16 + 4
    slots = distinct_slots(n, pages * block, n, padded=n // 5)
    k_cache, v_cache = (torch.full((pages, block, H, D), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    out = K.rope_kv16_store(*on(q, k, v, positions, cos_sin), k_cache, v_cache, torch.from_numpy(slots).to(DEV), neox=neox)
    for got, x in ((out.cpu(), q), (None, k)):
        want = P.rotate(x, positions, cos_sin, neox, F32)
        exact = P.rotate(x, positions, cos_sin, neox)
        assert bool(((want.double() - exact).abs() <= P.rotation_error(x, positions, cos_sin, neox)).all())
        if got is not None:
            assert same(got, want.to(dtype))
    pages_k, pages_v = (torch.full((pages * block, H, D), 7.0, dtype=dtype) for _ in range(2))
    keep = torch.from_numpy(slots) >= 0
    pages_k[slots[slots >= 0]] = want.to(dtype)[keep]
    pages_v[slots[slots >= 0]] = v[keep]
    assert same(k_cache.cpu().view(-1, H, D), pages_k) and same(v_cache.cpu().view(-1, H, D), pages_v)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,table", [(BF, F32), (BF, BF), (FP, FP), (F32, F32)])
@pytest.mark.parametrize("n,HQ,H,D,rot", [(1, 4, 1, 128, 128), (40, 8, 2, 128, 128), (23, 6, 3, 64, 64), (50, 2, 2, 128, 64), (19, 2, 1, 64, 16),
                                          (530, 4, 2, 128, 128), (700, 3, 1, 64, 32), (40, 4, 2, 128, 48), (0, 4, 2, 128, 128)])
def test_8_bit_cache(n, HQ, H, D, rot, dtype, table, fmt, neox):
    """The bytes that the plain implementation stores for the rotated fp32 keys, written twice (groups begun and continued)."""
    pages, block = n // 16 + 6, 32
    cache, ref = torch.zeros(pages, block, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV), Q.Cache(pages, block, H, D, fmt)
    for turn in range(2):
        q, k, v, positions, cos_sin = inputs(n, HQ, H, D, rot, dtype, table, 10 * n + turn)
        slots = distinct_slots(n, pages * block, n + turn, padded=n // 6)
        out = K.rope_q8_store(*on(q, k, v, positions, cos_sin), cache, torch.from_numpy(slots).to(DEV), fmt=fmt, neox=neox)
        assert same(out.cpu(), P.rotate(q, positions, cos_sin, neox, F32).to(dtype))
        ref.store(P.rotate(k, positions, cos_sin, neox, F32), v.float(), slots)
        assert Q.same_numbers(cache.cpu().numpy(), ref.to_bytes(), fmt)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype,table", [(BF, F32), (BF, BF), (FP, FP), (F32, F32)])
@pytest.mark.parametrize("n,HQ,H,D,rot,mode,kb,vb,dense", [
    (1, 4, 1, 128, 128, "iso", 3, 3, False), (37, 8, 2, 128, 128, "iso", 4, 3, False), (64, 6, 3, 128, 64, "planar", 4, 4, False),
    (100, 2, 1, 128, 16, "iso", 3, 3, True), (21, 4, 2, 64, 64, "iso", 4, 4, False), (30, 3, 1, 256, 256, "planar", 3, 3, False),
    (700, 4, 4, 128, 128, "iso", 3, 3, False), (0, 4, 2, 128, 128, "iso", 3, 3, False)])
def test_codebook_cache(n, HQ, H, D, rot, mode, kb, vb, dense, dtype, table, neox):
    """The bytes that the oracle packs for the rotated fp32 keys."""
    from rotorquant_vllm.vllm.rq_backend import _rq_total_bytes
    p = Params(mode, kb, vb, head_dim=D)
    q, k, v, positions, cos_sin = inputs(n, HQ, H, D, rot, dtype, table, n + 3)
    pages, block, total = n // 16 + 4, 16, _rq_total_bytes(D, H, dense)
    slots = distinct_slots(n, pages * block, n, padded=n // 6)
    cache = torch.full((pages, block, total), 9, dtype=torch.uint8, device=DEV)
    want = cache.cpu().numpy()
    out = K.rope_compress_store(*on(q, k, v, positions, cos_sin), cache, torch.from_numpy(slots).to(DEV), *on(p.rte, p.rto, p.kb, p.vb), neox=neox,
                                dense3=dense)
    assert same(out.cpu(), P.rotate(q, positions, cos_sin, neox, F32).to(dtype))
    if n:
        host = p.np()
        turned = P.rotate(k, positions, cos_sin, neox, F32)
        kp, kn = O.compress(O.to_bits(turned)[0], "float32", host["rte"], host["rto"], host["kb"], p.blk)
        vp, vn = O.compress(O.to_bits(v.float())[0], "float32", host["rte"], host["rto"], host["vb"], p.blk)
        O.compress_store(want, slots, kp, kn, vp, vn, dense3=dense)
    assert np.array_equal(cache.cpu().numpy(), want)


def stores(dtype=BF, H=2, D=128, pages=8, block=16):
    """The three stores over caches of one kind each: name -> (call(q, k, v, positions, cos_sin, slots, **kw), the cache's tensors)."""
    p = Params("iso", 3, 3, head_dim=D)
    dev = on(p.rte, p.rto, p.kb, p.vb)
    rq = torch.zeros(pages, block, H * 256, dtype=torch.uint8, device=DEV)
    q8 = torch.zeros(pages, block, K.q8_slot_bytes(H, D), dtype=torch.uint8, device=DEV)
    kv = torch.zeros(2, pages, block, H, D, dtype=dtype, device=DEV)
    return {"rq": (lambda *a, **kw: K.rope_compress_store(*a[:5], rq, a[5], *dev, **kw), rq),
            "q8": (lambda *a, **kw: K.rope_q8_store(*a[:5], q8, a[5], **kw), q8),
            "kv16": (lambda *a, **kw: K.rope_kv16_store(*a[:5], kv[0], kv[1], a[5], **kw), kv)}


KINDS = ["rq", "q8", "kv16"]


@pytest.mark.parametrize("kind", KINDS)
def test_slices_of_one_projection(kind):
    """q, k and v as a fused projection leaves them, queries rotated in place, a table with longer rows."""
    n, HQ, H, D = 30, 8, 2, 128
    q, k, v, positions, cos_sin = inputs(n, HQ, H, D, D, BF, BF, 4)
    slots = torch.from_numpy(distinct_slots(n, 128, 5))
    call, cache = stores()[kind]
    want = call(*on(q, k, v, positions, cos_sin, slots))
    want_cache = cache.clone()
    cache.zero_()
    qkv = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], dim=-1).to(DEV)
    views = [x.view(n, h, D) for x, h in zip(qkv.split([HQ * D, H * D, H * D], dim=-1), (HQ, H, H))]
    wide = torch.cat([cos_sin, torch.full_like(cos_sin, 9.0)], dim=-1).to(DEV)[:, :D]
    got = call(*views, positions.to(DEV), wide, slots.to(DEV), out_q=views[0])
    assert got is views[0] and same(got.cpu(), want.cpu()) and torch.equal(cache, want_cache)
    assert torch.equal(qkv[:, HQ * D:].cpu(), torch.cat([k.flatten(1), v.flatten(1)], dim=-1))
    cache.zero_()
    assert call(None, *views[1:], positions.to(DEV), wide, slots.to(DEV)) is None  # keys alone
    assert torch.equal(cache, want_cache)


@pytest.mark.parametrize("kind", KINDS)
def test_positions_outside_the_table(kind):
    """NaN queries and keys, and nothing else touched: int64 extremes, the table's ends."""
    n, HQ, H, D = 12, 4, 2, 128
    q, k, v, positions, cos_sin = inputs(n, HQ, H, D, 64, BF, F32, 8, far=40)
    positions[:6] = torch.tensor([-1, POSITIONS, 2 ** 31, -2 ** 63, 2 ** 63 - 1, 2 ** 32 + 1])
    positions[6:8] = torch.tensor([POSITIONS - 1, 0])
    slots = torch.arange(n) + 3
    call, cache = stores()[kind]
    out = call(*on(q, k, v, positions, cos_sin, slots)).cpu()
    assert same(out, P.rotate(q, positions, cos_sin, True, F32).to(BF)) and int(out.isnan().any(-1).sum()) == 6 * HQ
    call, cache = stores()[kind]
    call(*on(q[6:], k[6:], v[6:], positions[6:], cos_sin, slots[6:]))
    if kind == "rq":  # (groups of the 8-bit cache share scales)
        first = stores()[kind]
        first[0](*on(q, k, v, positions, cos_sin, slots))
        assert torch.equal(first[1].view(128, -1)[9:15], cache.view(128, -1)[9:15])
    if kind == "kv16":
        both = stores()[kind]
        both[0](*on(q, k, v, positions, cos_sin, slots))
        got = both[1].cpu().view(2, -1, H, D)
        assert same(got[0, 3:15], P.rotate(k, positions, cos_sin, True, F32).to(BF)) and same(got[1, 3:15], v)
        assert not got[:, :3].any() and not got[:, 15:].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [20, 640])
def test_graphs_and_streams(kind, n):
    """A captured call replayed over other data, and calls on a side stream."""
    HQ, H, D = 4, 2, 128
    call, cache = stores(pages=n // 8)[kind]
    data = [inputs(n, HQ, H, D, D, BF, BF, s) for s in range(4)]
    slots = [torch.from_numpy(distinct_slots(n, n // 8 * 16, s, padded=3)) for s in range(4)]
    fixed = on(*data[0], slots[0])
    out = torch.zeros_like(fixed[0])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*fixed, out_q=out)
        with torch.cuda.graph(graph, stream=side):
            call(*fixed, out_q=out)
    torch.cuda.current_stream().wait_stream(side)
    for s in (1, 2, 3, 1):
        for t, x in zip(fixed, (*data[s], slots[s])):
            t.copy_(x)
        cache.zero_()
        out.fill_(3.0)
        graph.replay()
        got, got_cache = out.clone(), cache.clone()
        cache.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = call(*on(*data[s], slots[s]))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert same(got, want) and torch.equal(got_cache, cache)


@pytest.mark.parametrize("H", [1, 3, 8])
def test_codebook_groups_of_all_sizes(H):
    """Rows are the same in a call of thousands of tokens, of hundreds, and of a few: the slots' bytes, rotated and as they are."""
    n, D, p = 6000, 128, Params("iso", 3, 3, head_dim=128)
    dev = on(p.rte, p.rto, p.kb, p.vb)
    _, k, v, positions, cos_sin = on(*inputs(n, 1, H, D, D, BF, BF, H))
    slots = torch.from_numpy(distinct_slots(n, n + 80, H, padded=n // 7)).to(DEV)
    for store in (lambda c, *x: K.rope_compress_store(None, *x[:3], cos_sin, c, x[3], *dev), lambda c, *x: K.compress_store(*x[:2], c, x[3], *dev)):
        whole = torch.full((n // 16 + 5, 16, H * 256), 3, dtype=torch.uint8, device=DEV)
        parts, at = whole.clone(), 0
        store(whole, k, v, positions, slots)
        for i, part in enumerate([1, 2, 1700, 16, 900, 17, 340, 5, 2100, 33, n]):
            to = min(n, at + part)
            store(parts, k[at:to], v[at:to], positions[at:to], slots[at:to])
            at = to
        assert torch.equal(whole, parts) and bool((whole != 3).any())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,HQ", [(25, 32768), (700, 1200)])
def test_many_query_rows(kind, n, HQ):
    """Over 192 MiB of queries: what calls of a part of the heads each give."""
    H, D, part = 2, 128, HQ // 16
    call, cache = stores(pages=n // 8 + 1)[kind]
    q = torch.randn(n, HQ, D, dtype=BF, device=DEV)
    _, k, v, positions, cos_sin = on(*inputs(n, 1, H, D, D, BF, BF, 1))
    slots = torch.from_numpy(distinct_slots(n, n // 8 * 16, 3, padded=3)).to(DEV)
    got = call(q, k, v, positions, cos_sin, slots)
    got_cache = cache.clone()
    for h in range(0, HQ, part):
        cache.zero_()
        assert same(call(q[:, h:h + part], k, v, positions, cos_sin, slots), got[:, h:h + part]) and torch.equal(cache, got_cache)


def test_pages_past_32_bits_of_elements():
    """Slots at the far end of pages of more than 2^32 elements, each side."""
    H, D, block = 8, 128, 64
    pages = (1 << 32) // (H * D * block) + 2
    k_cache, v_cache = (torch.zeros(pages, block, H, D, dtype=FP, device=DEV) for _ in range(2))
    q, k, v, positions, cos_sin = inputs(5, 8, H, D, D, FP, FP, 2)
    slots = torch.tensor([pages * block - 1, 0, pages * block, pages * block - 40, (pages - 1) * block])
    K.rope_kv16_store(*on(q, k, v, positions, cos_sin), k_cache, v_cache, slots.to(DEV))
    want = P.rotate(k, positions, cos_sin, True, F32).to(FP)
    for i in (0, 1, 3, 4):
        assert same(k_cache.view(-1, H, D)[int(slots[i])].cpu(), want[i]) and same(v_cache.view(-1, H, D)[int(slots[i])].cpu(), v[i])
    assert int((k_cache.view(-1, H * D) != 0).any(-1).sum()) == 4


def test_refusals():
    n, HQ, H, D = 4, 4, 2, 128
    data = dict(zip(("query", "key", "value", "positions", "cos_sin"), on(*inputs(n, HQ, H, D, D, BF, BF, 1))))
    slots = torch.arange(n, device=DEV)
    for kind, (call, cache) in stores().items():
        def run(match, error=ValueError, slots=slots, **kw):
            args = dict(data, **{k: x for k, x in kw.items() if k in data})
            more = {k: x for k, x in kw.items() if k not in data}
            with pytest.raises(error, match=match):
                call(*(args[x] for x in ("query", "key", "value", "positions", "cos_sin")), slots, **more)
        run("shape and dtype", value=data["value"].half())
        run("shape and dtype", value=data["value"][:, :1])
        run("query must be", query=data["query"].half())
        run("query must be", query=data["query"][:3])
        run("out_q must", out_q=torch.empty(n, HQ, D, device=DEV))
        run("out_q without", query=None, out_q=data["query"])
        run("positions must", positions=data["positions"].int())
        run("positions must", positions=data["positions"][:3])
        run("positions must", positions=torch.zeros(3, n, dtype=torch.int64, device=DEV))
        run("slot_mapping must", slots=slots.int())
        run("slot_mapping must", slots=slots[:2])
        run("cos_sin must", cos_sin=data["cos_sin"].half())
        run("cos_sin must", cos_sin=data["cos_sin"].t())
        run("rot_dim", cos_sin=data["cos_sin"][:, :24].contiguous())
        run("rot_dim", cos_sin=torch.zeros(9, 256, dtype=BF, device=DEV))
        run("table rows must be 16-byte", cos_sin=torch.zeros(9, 132, dtype=BF, device=DEV)[:, 2:130])
        run("16-byte aligned", query=torch.zeros(n, HQ, D + 4, dtype=BF, device=DEV)[..., :D])
        run("16-byte aligned", key=torch.zeros(n, H, D + 4, dtype=BF, device=DEV)[..., :D])
        run("no CPU path", RuntimeError, positions=data["positions"].cpu())
        run("contiguous over head_dim", key=torch.zeros(n, D, H, dtype=BF, device=DEV).transpose(1, 2))
        assert not cache.any()
    kv = stores()["kv16"][1]
    with pytest.raises(ValueError, match="pages must be of"):
        K.rope_kv16_store(*data.values(), kv[0].half(), kv[1].half(), slots)
    with pytest.raises(ValueError, match="heads of 128"):
        K.rope_kv16_store(*data.values(), kv[0, :, :, :1], kv[1, :, :, :1], slots)
    with pytest.raises(ValueError, match="same"):
        K.rope_kv16_store(*data.values(), kv[0], kv[1, :4], slots)
