"""Attention over plain 16-bit pages (kv16_attention) against a plain implementation in 64 bits."""
import math

import numpy as np
import pytest
import torch

import kv16_testlib as P
from rotorquant_vllm import _lib
from rotorquant_vllm import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def run(lens, q_lens, H, G, D, dtype, block=16, causal=True, scale=None, seed=1, layout="two", bound=None, **kw):
    pages = P.Pages(lens, block, H, D, dtype, seed, layout=layout)
    q = torch.randn(sum(q_lens), H * G, D, generator=P.gen(seed + 1)).to(dtype)
    cu = None if all(n == 1 for n in q_lens) and "cu" not in kw else i32(np.concatenate([[0], np.cumsum(q_lens)]))
    kw.pop("cu", None)
    got = K.kv16_attention(q.to(DEV), *pages.to(DEV), i32(pages.table), i32(lens), sm_scale=scale, causal=causal, cu_seqlens_q=cu, max_q_len=max(q_lens),
                           max_seq_len=bound, **kw)
    P.check(got, *P.attention(q, *pages.kv, lens, q_lens, scale, causal))


# A bound over 512 takes shares of several workgroups, one under it a workgroup for each item.
@pytest.mark.parametrize("bound", [512, None])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 96, 128, 192, 200, 256])
def test_head_dims(D, dtype, bound):
    run([1, 31, 33, 500] + ([1100] if bound is None else []), [1] * (4 if bound else 5), 2, 3, D, dtype, bound=bound)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H,G", [(1, 1), (8, 4), (4, 7), (1, 16), (2, 17), (1, 71)])
def test_groups(H, G, dtype):
    run([700, 15, 64], [1, 1, 1], H, G, 64, dtype)
    run([1300, 2], [1, 1], H, G, 128, dtype)


@pytest.mark.parametrize("block,layout", [(1, "two"), (3, "two"), (16, "paired"), (64, "heads"), (100, "paired"), (2048, "two")])
def test_pages_and_strides(block, layout):
    run([1, 100, 1200, 333], [1, 1, 1, 1], 2, 4, 128, BF, block=block, layout=layout)
    run([50, 700], [3, 1], 2, 4, 64, FP, block=block, layout=layout)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[2, 1, 3], [5, 8, 1], [16, 7, 20], [40, 1, 1]])
def test_drafts(q_lens, D, causal):
    run([700, 41, 64], q_lens, 2, 4, D, BF, causal=causal)


# Two blocks of columns and 32 items or 160: the latter take up to 2048 keys by a workgroup each.
@pytest.mark.parametrize("bound", [512, 513, 2048, 2049])
@pytest.mark.parametrize("H,seqs", [(2, 16), (8, 20)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_drafts_of_many_sequences(D, H, seqs, bound):
    run([bound - 29 * i % bound for i in range(seqs)], [1 + i % 6 for i in range(seqs)], H, 5, D, (BF, FP)[bound % 2], bound=bound)


# 128 items of one block: up to 768 keys by a workgroup each.
@pytest.mark.parametrize("bound", [768, 769])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decodes_of_many_sequences(D, bound):
    run([bound - 31 * i % bound for i in range(32)], [1] * 32, 4, 3, D, (BF, FP)[bound % 2], bound=bound)


def test_longer_queries_than_contexts():
    """Rows before the context's first key are zeros, causal; with no key at all, also otherwise."""
    for causal in (True, False):
        run([3, 0, 1], [9, 4, 2], 2, 4, 128, BF, causal=causal)
        run([3, 0, 1200], [9, 1, 2], 1, 2, 64, FP, causal=causal)


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 255, 256, 257, 1023, 1024, 1025, 2049, 4100])
def test_lengths(length):
    run([length, 1], [1, 1], 1, 4, 128, BF, bound=None if length > 512 else 512)
    run([length], [1], 2, 2, 128, FP, bound=length)
    run([length], [1], 2, 2, 64, FP)


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 200])
def test_many_sequences(seqs):
    lens = [int(x) for x in np.random.RandomState(seqs).randint(0, 90, seqs)]
    lens[-1] = 1500
    run(lens, [1] * seqs, 1, 2, 64, BF)
    run(lens, [1 + b % 3 for b in range(seqs)], 1, 2, 64, FP)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5, 1e-30])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scales(scale, dtype):
    run([300, 1100], [1, 2], 2, 2, 64, dtype, scale=scale)


WIDE = 1 << 24  # a bound on the lengths that gives a wave a kv head of its own, where heads come in fours


@pytest.mark.parametrize("D", [40, 64, 96, 128, 200, 256])
@pytest.mark.parametrize("H,G,q_lens", [(4, 1, [1, 1, 1, 1]), (8, 5, [1, 1, 1, 1]), (4, 3, [4, 1, 7, 5]), (4, 17, [1, 3, 1, 2])])
def test_a_wave_for_each_head(H, G, q_lens, D):
    for dtype in (BF, FP):
        run([1, 260, 0, 1300], q_lens, H, G, D, dtype, bound=WIDE)


@pytest.mark.parametrize("bound", [None, WIDE])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_an_infinite_value(dtype, D, T, bound):
    """One dim of one key's V is infinite in one head of four: that dim is where the key is seen, and all else is as without it."""
    H, G, L, at = 4, 2, 1100, 1095
    pages = P.Pages([L, L], 16, H, D, dtype, 3)
    kc, vc = pages.to(DEV)
    q = torch.randn(2 * T, H * G, D, generator=P.gen(5)).to(dtype)
    want, err = P.attention(q, *pages.kv, [L, L], [T, T])
    vc[int(pages.table[1, at // 16]), at % 16, 2, D - 3] = -math.inf
    got = K.kv16_attention(q.to(DEV), kc, vc, i32(pages.table), i32([L, L]), cu_seqlens_q=i32([0, T, 2 * T]), max_q_len=T, max_seq_len=bound).cpu()
    seen = torch.zeros_like(got, dtype=torch.bool)
    for i in range(T):
        seen[T + i, 2 * G:3 * G, D - 3] = at < L - T + i + 1
    assert bool((got[seen] == -math.inf).all()) and bool(seen.any())
    P.check(got.masked_fill(seen, 0.0), want.masked_fill(seen, 0.0), err)


def plain(q, k, v, end, scale):
    """Softmax attention of one row in 64 bits, infinities and NaN as they come."""
    s = (k[:end].double() @ q.double()) * scale
    return torch.softmax(s, dim=0) @ v[:end].double()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("L", [40, 1400])
def test_infinities_in_masked_places(side, bad, dtype, L):
    """Key L - 2 (of 5 new tokens, L - 5 ...) is infinite: rows before it are as without it, and the others as the formula gives them."""
    D, T = 64, 5
    pages = P.Pages([L], 16, 1, D, dtype, 3)
    k, v = pages.kv[0][0], pages.kv[1][0]
    x = k if side == "k" else v
    x[L - 2, 0, 7] = bad
    cache = pages.view(pages.both)[0 if side == "k" else 1]
    at = torch.arange(L)
    cache[torch.from_numpy(pages.table[0].astype(np.int64))[at // 16], at % 16] = x
    q = torch.randn(T, 2, D, generator=P.gen(5)).to(dtype)
    q[..., 7] = 1.0  # (a score of the infinity's sign)
    got = K.kv16_attention(q.to(DEV), *pages.to(DEV), i32(pages.table), i32([L]), cu_seqlens_q=i32([0, T])).cpu()
    out, err = P.attention(q[:3], [k[:L - 2]], [v[:L - 2]], [L - 2], [3])
    P.check(got[:3], out, err)
    for i in (3, 4):
        for j in range(2):
            want = plain(q[i, j], k[:, 0], v[:, 0], L - T + i + 1, 1 / math.sqrt(D))
            if side == "v":
                keep = torch.arange(D) != 7
                assert bool(torch.isfinite(got[i, j][keep]).all()) and bool(torch.isfinite(want[keep]).all())
                assert math.isnan(got[i, j, 7]) if math.isnan(bad) else float(got[i, j, 7]) == bad
            else:
                assert bool((got[i, j].isnan() == want.isnan()).all())
                if not bool(want.isnan().any()):  # a score of -infinity: the key does not count
                    seen = [n for n in range(L - T + i + 1) if n != L - 2]
                    P.check(got[i:i + 1, j:j + 1], *P.attention(q[i:i + 1, j:j + 1], [k[seen]], [v[seen]], [len(seen)], [1]))


def test_rows_whose_keys_all_score_minus_infinity():
    """0 / 0, as the formula says, and no zeros."""
    pages = P.Pages([40, 40], 16, 1, 64, BF, 3)
    kc, vc = pages.to(DEV)
    kc[torch.from_numpy(pages.table[0].astype(np.int64)).to(DEV)] = -math.inf
    q = torch.ones(2, 1, 64, dtype=BF, device=DEV)
    got = K.kv16_attention(q, kc, vc, i32(pages.table), i32([40, 40]))
    assert bool(got[0].isnan().all()) and bool(torch.isfinite(got[1]).all())


def test_large_and_small_values():
    """Keys that put all weight on one token, V of the largest values, weights far under the largest."""
    D, L = 128, 1500
    for dtype, big in ((BF, 3e38), (FP, 65504.0)):
        pages = P.Pages([L], 16, 1, D, dtype, 6)
        k, v = pages.kv[0][0], pages.kv[1][0]
        q = torch.randn(1, 2, D, generator=P.gen(7)).to(dtype)
        k[700, 0] = q[0, 0] * 4
        v[5, 0, :4] = torch.tensor([big, -big, big, 1e-7]).to(dtype)
        v[700, 0] = v[700, 0] * 2.0 ** -10
        for side, x in enumerate((k, v)):
            at = torch.arange(L)
            pages.view(pages.both)[side][torch.from_numpy(pages.table[0].astype(np.int64))[at // 16], at % 16] = x
        got = K.kv16_attention(q.to(DEV), *pages.to(DEV), i32(pages.table), i32([L]))
        P.check(got, *P.attention(q, [k], [v], [L], [1]))


def test_rows_of_no_sequence_and_past_the_bounds():
    """out keeps rows behind the last sequence and tokens past max_q_len; keys past max_seq_len and the table are not read."""
    lens, H, G, D = [200, 300], 1, 2, 64
    pages = P.Pages(lens, 16, H, D, BF, 4)
    q = torch.randn(9, H * G, D, generator=P.gen(4)).to(BF)
    out = torch.full((9, H * G, D), 5.0, dtype=BF, device=DEV)
    args = (*pages.to(DEV), i32(pages.table), i32(lens))
    got = K.kv16_attention(q.to(DEV), *args, cu_seqlens_q=i32([0, 4, 6]), max_q_len=3, out=out)
    assert got is out and bool((out[6:] == 5).all()) and bool((out[3] == 5).all())
    want, err = P.attention(q[:6], *pages.kv, lens, [4, 2])
    for rows in (slice(0, 3), slice(4, 6)):
        P.check(got[rows], want[rows], err[rows])
    # bounds on the keys: positions go by the whole length
    got = K.kv16_attention(q[:2].to(DEV), *args, max_seq_len=150)
    P.check(got, *P.attention(q[:2], [x[:150] for x in pages.kv[0]], [x[:150] for x in pages.kv[1]], [150, 150], [1, 1]))
    got = K.kv16_attention(q[:2].to(DEV), *args[:2], i32(pages.table[:, :5]), args[3])
    P.check(got, *P.attention(q[:2], [x[:80] for x in pages.kv[0]], [x[:80] for x in pages.kv[1]], [80, 80], [1, 1]))


def test_strided_rows():
    """Queries as a slice of a projection and outputs with gaps; one token and one head with any strides."""
    lens, H, G, D = [70, 1200], 2, 2, 64
    pages = P.Pages(lens, 16, H, D, FP, 4)
    q = torch.randn(2, H * G, D, generator=P.gen(4)).to(FP)
    wide = torch.zeros(2, 3 * H * G, D, dtype=FP, device=DEV)
    wide[:, ::3] = q.to(DEV)
    out = torch.zeros(2, H * G, 2 * D, dtype=FP, device=DEV)
    got = K.kv16_attention(wide[:, ::3], *pages.to(DEV), i32(pages.table), i32(lens), out=out[..., :D])
    P.check(got, *P.attention(q, *pages.kv, lens, [1, 1]))
    assert not out[..., D:].any()


def test_graph_replays_with_other_lengths():
    H, G, D = 2, 4, 128
    pages = P.Pages([3000, 500], 16, H, D, BF, 4)
    q = torch.randn(2, H * G, D, generator=P.gen(4)).to(BF)
    kc, vc = pages.to(DEV)
    q_dev, bt, sl = q.to(DEV), i32(pages.table), i32([3000, 500])
    out, side, graph = torch.zeros_like(q_dev), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.kv16_attention(q_dev, kc, vc, bt, sl, out=out)
        with torch.cuda.graph(graph, stream=side):
            K.kv16_attention(q_dev, kc, vc, bt, sl, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for lens in ([3000, 500], [1, 1], [0, 300], [2999, 17], [1025, 499]):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(3.0)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, K.kv16_attention(q_dev, kc, vc, bt, sl))
        P.check(got, *P.attention(q, [x[:n] for x, n in zip(pages.kv[0], lens)], [x[:n] for x, n in zip(pages.kv[1], lens)], lens, [1, 1]))


def test_scratch_that_the_caller_keeps():
    lens, H, G, D = [3000, 1300], 2, 4, 128
    pages = P.Pages(lens, 16, H, D, BF, 4)
    q = torch.randn(2, H * G, D, generator=P.gen(4)).to(BF).to(DEV)
    args = (q, *pages.to(DEV), i32(pages.table), i32(lens))
    want = K.kv16_attention(*args)
    need = _lib.load().rq_kv16_attention_workspace_bytes(2, H * G, H, D, 1, pages.table.shape[1] * 16)
    assert need > 0
    for size, fill in ((need, 0xff), (need + 4096, 0x7f)):
        ws = torch.full((size + 64,), fill, dtype=torch.uint8, device=DEV)
        for _ in range(2):
            assert torch.equal(K.kv16_attention(*args, workspace=ws[:size]), want)
        assert bool((ws[size:] == fill).all())
    with pytest.raises(RuntimeError, match="workspace too small"):
        K.kv16_attention(*args, workspace=ws[:need - 1])
    with pytest.raises(ValueError, match="contiguous uint8"):
        K.kv16_attention(*args, workspace=ws.view(torch.int32))


def test_graphs_that_share_scratch():
    """Two captured calls of different shapes over one workspace, replayed in turn."""
    calls, graphs, side = [], [], torch.cuda.Stream()
    for b, (H, G, D) in enumerate(((2, 4, 128), (4, 3, 64))):
        pages = P.Pages([2600, 900], 16, H, D, BF, 4 + b)
        q = torch.randn(2, H * G, D, generator=P.gen(b)).to(BF).to(DEV)
        calls.append((q, *pages.to(DEV), i32(pages.table), i32([2600, 900])))
    want = [K.kv16_attention(*c) for c in calls]
    ws, outs = torch.full((64 << 20,), 0xff, dtype=torch.uint8, device=DEV), [torch.empty_like(c[0]) for c in calls]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, out in zip(calls, outs):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                K.kv16_attention(*c, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
        assert torch.equal(K.kv16_attention(*calls[0], workspace=ws), want[0])


def test_two_streams():
    """Calls that overlap, each with scratch of its own."""
    H, G, D = 2, 4, 128
    calls = []
    for b in range(2):
        lens = [2500 - 900 * b, 100]
        pages = P.Pages(lens, 16, H, D, BF, 4 + b)
        calls.append((torch.randn(2, H * G, D, generator=P.gen(b)).to(BF).to(DEV), *pages.to(DEV), i32(pages.table), i32(lens)))
    want = [K.kv16_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for b in range(2):
            with torch.cuda.stream(streams[b]):
                got[b].append(K.kv16_attention(*calls[b]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[b]) for b in range(2) for x in got[b])


def test_pages_past_32_bits_of_elements():
    H, D, block = 8, 128, 64
    pages = (1 << 32) // (H * D * block) + 2
    kc, vc = (torch.zeros(pages, block, H, D, dtype=FP, device=DEV) for _ in range(2))
    ids = [pages - 1, 0, pages - 2]
    lens = [3 * block - 5]
    k, v = (torch.randn(lens[0], H, D, generator=P.gen(s)).to(FP) for s in (1, 2))
    at = torch.arange(lens[0])
    for cache, x in ((kc, k), (vc, v)):
        cache[torch.tensor(ids)[at // block].to(DEV), (at % block).to(DEV)] = x.to(DEV)
    q = torch.randn(1, 2 * H, D, generator=P.gen(3)).to(FP)
    got = K.kv16_attention(q.to(DEV), kc, vc, i32([ids]), i32(lens))
    P.check(got, *P.attention(q, [k], [v], lens, [1]))


def test_append_rotated_and_attend():
    """A server's steps: a prompt, then tokens, each rotated, appended and attended to in turn."""
    H, G, D, block, seqs, prompt = 2, 4, 128, 16, 3, 37
    cos_sin = P.table(200, D, torch.float32)
    table = torch.arange(seqs * 8).reshape(seqs, 8)[:, torch.randperm(8, generator=P.gen(1))]
    kc, vc = (torch.zeros(seqs * 8, block, H, D, dtype=BF, device=DEV) for _ in range(2))
    ks, vs = [torch.zeros(0, H, D, dtype=BF)] * seqs, [torch.zeros(0, H, D, dtype=BF)] * seqs
    g, held = P.gen(9), 0
    for new in [prompt] + [1] * 14 + [4]:
        q, k, v = (torch.randn(seqs * new, h, D, generator=g).to(BF) for h in (H * G, H, H))
        at = torch.arange(held, held + new)
        positions, slots = at.repeat(seqs), (table[:, at // block] * block + at % block).reshape(-1)
        q_dev = K.rope_kv16_store(*(x.to(DEV) for x in (q, k, v, positions, cos_sin)), kc, vc, slots.to(DEV))
        held += new
        turned = P.rotate(k, positions, cos_sin, True, torch.float32).to(BF)
        ks = [torch.cat([a, b]) for a, b in zip(ks, turned.split(new))]
        vs = [torch.cat([a, b]) for a, b in zip(vs, v.split(new))]
        got = K.kv16_attention(q_dev, kc, vc, i32(table), i32([held] * seqs), cu_seqlens_q=i32(np.arange(seqs + 1) * new), max_q_len=new)
        q_host = P.rotate(q, positions, cos_sin, True, torch.float32).to(BF)
        assert torch.equal(q_dev.cpu(), q_host)
        P.check(got, *P.attention(q_host, ks, vs, [held] * seqs, [new] * seqs))


def test_refusals():
    pages = P.Pages([40, 50], 16, 2, 64, BF, 3)
    kc, vc = pages.to(DEV)
    q, bt, sl = torch.zeros(2, 4, 64, dtype=BF, device=DEV), i32(pages.table), i32([40, 50])
    for match, args, kw in [
            ("of the pages' dtype", (q.half(), kc, vc, bt, sl), {}), ("a multiple of the pages' heads", (q[:, :3], kc, vc, bt, sl), {}),
            ("same", (q, kc, vc.half(), bt, sl), {}), ("heads of 64", (q, kc[..., :32], vc[..., :32], bt, sl), {}),
            ("block_table must", (q, kc, vc, bt.long(), sl), {}), ("seq_lens must", (q, kc, vc, bt, sl.long()), {}),
            ("number of sequences", (q, kc, vc, bt[:1], sl), {}), ("cu_seqlens_q is needed", (q[:1], kc, vc, bt, sl), {}),
            ("3 entries", (q, kc, vc, bt, sl), dict(cu_seqlens_q=sl)), ("out must", (q, kc, vc, bt, sl), dict(out=q[:1])),
            ("sm_scale", (q, kc, vc, bt, sl), dict(sm_scale=math.inf)), ("sm_scale", (q, kc, vc, bt, sl), dict(sm_scale=math.nan)),
            ("sm_scale", (q, kc, vc, bt, sl), dict(sm_scale=3e38)),
            ("no pages", (q, kc[:0], vc[:0], bt, sl), {}), ("head_dim 512", (torch.zeros(1, 1, 512, dtype=BF, device=DEV),) + tuple(torch.zeros(2, 1, 16, 1, 512, dtype=BF, device=DEV)) + (bt[:1], sl[:1]), {}),
            ("q rows must be 16-byte", (torch.zeros(2, 4, 68, dtype=BF, device=DEV)[..., :64], kc, vc, bt, sl), {}),
            ("cache rows must be 16-byte", (q, *(torch.zeros(2, 3, 16, 2, 68, dtype=BF, device=DEV)[..., :64]), bt, sl), {})]:
        with pytest.raises(ValueError, match=match):
            K.kv16_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.kv16_attention(q, kc, vc, bt.cpu(), sl)
