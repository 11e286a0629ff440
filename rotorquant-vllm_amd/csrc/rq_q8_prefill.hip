// Attention of prompts and prompt chunks over the 8-bit KV cache (part of rq_q8_attention, whose
// arithmetic rq_q8_attention.hip describes; format in rq_q8.h), bound by the matrix cores.
//
// Two launches (three with key chunks):
//   pack:      every 64-key tile of a (sequence, kv head) becomes a tile image in the workspace: its codes in
//              fp16 (exact), in the order of the MFMA operands, and its groups' scales;
//   attention: a workgroup's four waves take 32 query positions of one head each and stream the
//              images through LDS.  Per tile S^T = K Q^T and O^T += C_v^T w on v_mfma_f32_32x32x16_f16.
// An operand of the image is the 1 KB that a wave reads at 16 bytes a lane, so LDS is read in a row,
// free of bank conflicts, at one address and constant offsets.
//
// Tile step (lane: half hh = lane / 32, column = position = lane % 32):
//   S: element 4 j + i of 32-key block b is key 32 b + 8 j + 4 hh + i;  its group 2 b + j / 2;
//   P V step t is group t: its 8 weights of a lane are elements 8 (t & 1) .. + 7 of block t / 2, keys
//   16 t + {4 hh + i, 8 + 4 hh + i}, i < 4 -- no transposition.
#include <algorithm>
#include <type_traits>

#include "rq_q8_attn.h"

namespace rq {

constexpr int kQ8KT = 64;      // keys of a tile: four groups
constexpr int kQ8PW = 32;      // query positions of a wave
constexpr int kQ8PWaves = 4;   // waves of a workgroup

template <int D>
struct Q8Image {
    static constexpr int kK = D / 8, kV = D / 8;          // operands: K (16-dim step, 32-key block), V (group, 32 dims)
    static constexpr int kKMeta = kK * 1024;              // float 2^e_k of the four groups, then float e_v
    static constexpr int kVAt = kKMeta + 1024;
    static constexpr int kVMeta = kVAt + kV * 1024;       // float 2^-e_v of the four groups
    static constexpr int kBytes = kVMeta + 1024;
    static constexpr int kLdsK = kKMeta + 1024, kLdsV = kV * 1024 + 1024;
    static constexpr int kPart = kQ8PW * D + kQ8PW * 2;   // floats of a wave's partial
};

struct Q8PrefillArgs {
    Q8AttnArgs a;
    int b0, h0, nh;     // first sequence and kv head of this pass, its kv heads
    int64_t max_tiles;  // images of a (sequence, kv head)
    uint8_t *images;
    int nx, split;      // query blocks; workgroups of a query block (key chunks)
};

// ---- pack -------------------------------------------------------------------------
// Bound by memory: 8 x 4096 tokens of 8 heads, 67 MB of codes to 143 MB of images, in 34 us.
template <int FMT, int D>
__global__ __launch_bounds__(256) void q8_pack_kernel(Q8PrefillArgs p) {
    using Im = Q8Image<D>;
    const Q8AttnArgs &a = p.a;
    const int tile = blockIdx.x, h = p.h0 + blockIdx.y;
    const int64_t b = p.b0 + blockIdx.z;
    const Q8Seq s = q8_seq(a, b);
    const int k0 = tile * kQ8KT;
    if (k0 >= s.vis || s.T == 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t *const img = p.images + (((int64_t)blockIdx.z * p.nh + blockIdx.y) * p.max_tiles + tile) * Im::kBytes;
    const Q8Layout lay(a.H, D, a.block_size);
    auto page_of = [&](int gr, int &gi) -> const uint8_t * {  // group gr of the tile: its page, its place there
        const int g = k0 / kQ8Group + gr, lp = g / a.groups;
        gi = g - lp * a.groups;
        int64_t page = a.bt[b * a.bt_ss + lp];
        page = page < 0 || page >= a.num_blocks ? 0 : page;
        return a.cache + page * a.stride_block;
    };
    // K: 16-byte piece (group, chunk, 16-dim part, token); V: (group, chunk, half, dim % 16), two pieces
    constexpr int kPieces = D, kRounds = kPieces * 4 / 256, kItems = D / 2;
    u32x4 kw[kRounds], vw[2];
    bool kin[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int gr = (wave * 64 + 256 * r) / kPieces;
        kin[r] = k0 + kQ8Group * gr < s.vis;
        int gi = 0;
        if (kin[r]) kw[r] = *reinterpret_cast<const u32x4 *>(page_of(gr, gi) + lay.codes_at(gi, h) + 16 * ((tid + 256 * r) % kPieces));
    }
    const int vg = kItems == 64 ? wave : tid / kItems, item = tid % kItems;
    const int hh = (item >> 4) & 1, c = item & 15, chunk = item >> 5;
    const bool vin = vg < 4 && k0 + kQ8Group * vg < s.vis;
    if (vin) {
        int gi;
        const uint8_t *page = page_of(vg, gi), *from = page + lay.codes_at(gi, h) + kQ8Group * D + 1024 * chunk + 256 * hh + 16 * c;
        vw[0] = *reinterpret_cast<const u32x4 *>(from);
        vw[1] = *reinterpret_cast<const u32x4 *>(from + 512);
    }
    if (tid < 4) {
        float2 sc = make_float2(0.f, 0.f);
        int gi;
        if (k0 + kQ8Group * tid < s.vis) {
            const uint8_t *page = page_of(tid, gi);
            sc = *reinterpret_cast<const float2 *>(page + lay.scale_at(gi, h));
        }
        const int ev = q8_scale_exp(sc.y);
        reinterpret_cast<float *>(img + Im::kKMeta)[tid] = exp2i(q8_scale_exp(sc.x));
        reinterpret_cast<float *>(img + Im::kKMeta)[4 + tid] = (float)ev;
        reinterpret_cast<float *>(img + Im::kVMeta)[tid] = exp2i(-ev);
    }
    auto halves = [](uint32_t w0, uint32_t w1) {
        u32x4 o;
        uint32_t x[4];
        q8_to_f16<FMT>(w0, x[0], x[1]);
        q8_to_f16<FMT>(w1, x[2], x[3]);
        o = u32x4{x[0], x[1], x[2], x[3]};
        return o;
    };
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int idx = tid + 256 * r, gr = idx / kPieces, l = idx & 63, j = (idx % kPieces) >> 6;
        // dims 16 ks .. + 15 of key 16 gr + t: both halves of operand (ks, gr / 2)
        const int ks = 4 * j + (l >> 4), row = 16 * (gr & 1) + (l & 15);
        uint8_t *const to = img + (2 * ks + (gr >> 1)) * 1024 + 16 * row;
        *reinterpret_cast<u32x4 *>(to) = kin[r] ? halves(kw[r][0], kw[r][1]) : zero;
        *reinterpret_cast<u32x4 *>(to + 512) = kin[r] ? halves(kw[r][2], kw[r][3]) : zero;
    }
    if (vg < 4) {
        // tokens at or past the context's end: zeros, whatever their codes (0 * NaN is NaN)
        const int left = s.vis - (k0 + kQ8Group * vg + 4 * hh);
        auto keep = [](int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; };
        const uint32_t keep0 = keep(left), keep1 = keep(left - 8);
        constexpr uint32_t kZero = FMT == RQ_Q8_INT8 ? 0x80808080u : 0u;  // the code of 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = 2 * chunk + (i >> 1), col = 16 * (i & 1) + c;
            u32x4 o = zero;
            if (vin) o = halves((vw[0][i] & keep0) | (kZero & ~keep0), (vw[1][i] & keep1) | (kZero & ~keep1));
            *reinterpret_cast<u32x4 *>(img + Im::kVAt + (vg * (D / 32) + m) * 1024 + 512 * hh + 16 * col) = o;
        }
    }
}

// ---- attention ----------------------------------------------------------------------
// N consecutive KB: the immediate offset moves both the source and the place in LDS.
template <int N>
__device__ __forceinline__ void copy16n(const uint8_t *src, uint32_t voff, uint32_t dst) {
    if constexpr (N == 4)
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n\tglobal_load_lds_dwordx4 %0, %1 offset:1024\n\t"
                     "global_load_lds_dwordx4 %0, %1 offset:2048\n\tglobal_load_lds_dwordx4 %0, %1 offset:3*1024" ::"v"(voff), "s"(src), "{m0}"(dst) : "memory");
    else
        asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n\tglobal_load_lds_dwordx4 %0, %1 offset:1024" ::"v"(voff), "s"(src), "{m0}"(dst) : "memory");
}

constexpr int kQ8MinTiles = 4;  // tiles of a key chunk, at least
struct Q8Block {
    Q8Seq s;
    int units, f0, kv_end, n_tiles;
};
// Query block -> its first unit (32-position group, query head), the sequence's units, and the tiles that any of its positions sees.
__device__ __forceinline__ Q8Block q8_block(const Q8AttnArgs &a, int64_t b, int qblk) {
    Q8Block q;
    q.s = q8_seq(a, b);
    q.units = (q.s.T + kQ8PW - 1) / kQ8PW * a.G;
    q.f0 = qblk * kQ8PWaves;
    const int last_i = min(q.s.T, (min(q.f0 + kQ8PWaves, q.units) - 1) / a.G * kQ8PW + kQ8PW) - 1;
    q.kv_end = a.causal ? min(q.s.vis, q.s.pos + last_i + 1) : q.s.vis;
    q.n_tiles = q.kv_end > 0 ? (q.kv_end + kQ8KT - 1) / kQ8KT : 0;
    return q;
}
__device__ __forceinline__ int q8_chunk_tiles(int n_tiles, int split) { return max(kQ8MinTiles, (n_tiles + split - 1) / split); }

// What bounds it: the matrix cores and vector issue together, under the card's power limit.  8 prompts of 2222 to 4096 tokens, 32 / 8
// heads (0.84 TFLOP): 820 to 880 us by card, 955 to 1020 TFLOP/s (the library's 8192^3 product: 1240 to 1340 of random numbers,
// 1800 of zeros).  The matrix cores are busy half of the cycles, at 1.8 GHz (the memory-bound kernels run at 2.1).  A wave's tile
// is 32 MFMAs, 32 exponentials and 117 other vector instructions (the listing: 50 in the first phase, 67 in the second), a tile on the
// diagonal 69 more, a raised maximum 73; with those, the first and the last tile and the prologue the counters give 148 a tile.
// Measured by itself, an MFMA with a pair of exponentials and its packing takes 21.4 ns of a SIMD, without 13.8, so the first phase is
// bound by issue.  Without the tile copies 9 % less time, without exponentials 6 %.
// Tried without gain: two units a wave at one wave a SIMD (half the LDS reads; 226 registers spilled), eight waves on one tile
// (926 -> 931 us, one prompt of 700 tokens 24 -> 32), one wait for two operand reads, other depths of reading ahead.
// A gain that is not taken: two sets of four waves on alternate tiles, one prompt of 1000 tokens 35 -> 30 us, of 700 and less 1 us slower; it
// would be a second form of this kernel, for calls of few workgroups and many tiles.
template <int DT, int D>
__global__ __launch_bounds__(64 * kQ8PWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void q8_prefill_kernel(Q8PrefillArgs p) {
    using Im = Q8Image<D>;
    constexpr int kSteps = D / 16, kM = D / 32, kF = D / 8;  // k steps of Q K^T, 32-dim blocks of O, MFMAs of a phase
    const Q8AttnArgs &a = p.a;
    int qblk, hl;
    int64_t bl;
    attn_work_item(qblk, hl, bl);
    const int h = p.h0 + hl;
    const int64_t b = p.b0 + bl;
    int chunk = 0;
    if (p.split > 1) {
        chunk = qblk % p.split;
        qblk /= p.split;
    }
    const Q8Block qb = q8_block(a, b, qblk);
    const Q8Seq &s = qb.s;
    if (qb.f0 >= qb.units) return;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hh = lane >> 5, col = lane & 31;
    const int f = qb.f0 + wave;
    const int i0 = f < qb.units ? f / a.G * kQ8PW : s.T;  // first position of this wave's unit (past the end: inactive)
    const int hq = h * a.G + f % a.G;
    const bool wave_active = i0 < s.T;
    const int my_i = i0 + col, pos_base = s.pos, my_pos = pos_base + my_i;
    const int kv_end = qb.kv_end;
    int t0 = 0, n_tiles = qb.n_tiles;
    if (p.split > 1) {
        const int per = q8_chunk_tiles(n_tiles, p.split);
        t0 = chunk * per;
        n_tiles = min(per, n_tiles - t0);
        if (n_tiles <= 0 && (chunk > 0 || qb.n_tiles > 0)) return;  // (the merge does not look at this chunk)
    }
    const int wv_end = a.causal ? min(kv_end, pos_base + i0 + kQ8PW) : kv_end;
    const int nw = wave_active ? max(0, min(n_tiles, (max(wv_end, 0) + kQ8KT - 1) / kQ8KT - t0)) : 0;

    // LDS: two K buffers (operands, then 2^e_k and e_v) and two V buffers (operands, then 2^-e_v)
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const kbuf[2] = {lds, lds + Im::kLdsK};
    uint8_t *const vbuf[2] = {lds + 2 * Im::kLdsK, lds + 2 * Im::kLdsK + Im::kLdsV};
    const uint8_t *const img0 = p.images + (((int64_t)bl * p.nh + hl) * p.max_tiles + t0) * Im::kBytes;
    const uint32_t lds0 = lds_addr(lds);
    constexpr int kChunksW = kF / kQ8PWaves;  // 1 KB chunks of a wave: consecutive, one address and immediate offsets for all
    auto copy = [&](int t, int from, uint32_t dst_) {
        const uint64_t src64 = reinterpret_cast<uint64_t>(img0 + (int64_t)t * Im::kBytes + from + wave * (kChunksW * 1024));
        const uint32_t slo = __builtin_amdgcn_readfirstlane((uint32_t)src64), shi = __builtin_amdgcn_readfirstlane((uint32_t)(src64 >> 32));
        const uint8_t *src = reinterpret_cast<const uint8_t *>(((uint64_t)shi << 32) | slo);
        const uint32_t dst = __builtin_amdgcn_readfirstlane(dst_);
        copy16n<kChunksW>(src, 16 * lane, dst + wave * (kChunksW * 1024));
        if (wave == 0) copy16(src + kF * 1024, 16 * lane, dst + kF * 1024);  // the groups' scales
    };
    auto copy_k = [&](int t) { if (t < n_tiles) copy(t, 0, lds0 + (t & 1) * Im::kLdsK); };
    auto copy_v = [&](int t) { if (t < n_tiles) copy(t, Im::kVAt, lds0 + 2 * Im::kLdsK + (t & 1) * Im::kLdsV); };

    // Q^T operand, loaded before the first copies go out (a wait for a load also waits for copies issued before it)
    u32x4 qop[kSteps];
    const bool qvalid = wave_active && my_i < s.T;
    {
        const uint16_t *qrow = static_cast<const uint16_t *>(a.q) + (int64_t)(s.q0 + (qvalid ? my_i : 0)) * a.q_st + (int64_t)(qvalid ? hq : h * a.G) * a.q_sh;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) qop[k] = qvalid ? *reinterpret_cast<const u32x4 *>(qrow + 16 * k + 8 * hh) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) asm volatile("" : "+v"(qop[k]));  // (arrived)
    copy_k(0);
    copy_v(0);
    copy_k(1);
    copy_v(1);
    float colf;
    {
        uint32_t big = 0;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) big = q8_max_bits(qop[k], big);
        big = max(big, (uint32_t)__shfl_xor((int)big, 32));
        const int up = q8_query_exp<DT>(a, big);
        const float fq = exp2i(up) * a.q_sign;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) qop[k] = q8_query_f16<DT>(qop[k], fq);
        colf = a.score_scale * exp2i(-up);
    }

    f32x16 acc[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) acc[m] = f32x16{};
    float l_run = 0.f, B = kQ8NoBias;
    f32x16 sa[2], sb[2];  // scores of an even and of an odd tile
    float fg[4], add[4];  // of the tile whose exponentials come next: a weight is 2^(S fg + add)
    auto mask = [&](int t, f32x16 (&sc)[2]) {
        const int k0 = (t0 + t) * kQ8KT, nk = min(kQ8KT, kv_end - k0);
        if (!(nk == kQ8KT && (!a.causal || k0 + kQ8KT - 1 <= pos_base + i0)))
            wide_mask(sc, (a.causal ? min(k0 + nk, my_pos + 1) : k0 + nk) - (k0 + 4 * hh));
    };
    // From the largest raw scores of a tile's groups: the running maximum, and fg, add.
    auto raise = [&](const float (&gm)[4], const float4 ks, const float4 ev) {
        fg[0] = colf * ks.x, fg[1] = colf * ks.y, fg[2] = colf * ks.z, fg[3] = colf * ks.w;
        const float e[4] = {ev.x, ev.y, ev.z, ev.w};
        float tm = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) tm = fmaxf(tm, __builtin_fmaf(gm[g], fg[g], e[g]));
        if (__any(q8_passes(tm, B))) {
            auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(tm), __float_as_uint(tm), false, false);
            const float b_new = fminf(B, kQ8Peak - fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
            const float alpha = __builtin_amdgcn_exp2f(b_new - B);
#pragma unroll
            for (int m = 0; m < kM; ++m) acc[m] *= alpha;
            l_run *= alpha;
            B = b_new;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) add[g] = e[g] + B;
    };
    auto k_op = [&](const uint8_t *kt, int fi) { return *reinterpret_cast<const u32x4 *>(kt + 16 * lane + 1024 * fi); };
    auto meta4 = [](const uint8_t *at) { return *reinterpret_cast<const float4 *>(at); };
    // pair i of weights: its place in the operand, and its group's sum, of the weights before their rounding: fp16 loses those of
    // groups whose V is 2^31 times smaller than others' (or zero), which the softmax's sum still has to hold
    auto exp_pair = [&](const f32x16 (&sc)[2], int i, uint32_t (&pop)[16], float (&l)[4]) {
        const int t = i >> 2, e = 8 * (t & 1) + 2 * (i & 3);
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e], fg[t], add[t]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e + 1], fg[t], add[t]));
        pop[i] = pack_f16(p0, p1);
        l[t] += p0 + p1;
    };
    auto add_sums = [&](const float (&l)[4], const float4 iv) {
        l_run = __builtin_fmaf(l[0], iv.x, __builtin_fmaf(l[1], iv.y, __builtin_fmaf(l[2], iv.z, __builtin_fmaf(l[3], iv.w, l_run))));
    };

    wait_copies<0>();
    __syncthreads();
    if (nw > 0) {
        sa[0] = sa[1] = f32x16{};
#pragma unroll
        for (int fi = 0; fi < kF; ++fi) sa[fi & 1] = mfma32<RQ_DTYPE_F16>(k_op(kbuf[0], fi), qop[fi >> 1], sa[fi & 1]);
        mask(0, sa);
        float gm[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            gm[g] = sa[g >> 1][8 * (g & 1)];
#pragma unroll
            for (int e = 1; e < 8; ++e) gm[g] = fmaxf(gm[g], sa[g >> 1][8 * (g & 1) + e]);
        }
        raise(gm, meta4(kbuf[0] + kF * 1024), meta4(kbuf[0] + kF * 1024 + 16));
    }
    // Before tile t: its V and tile t+1's K have landed for every wave, and every wave is done with tile t's K and tile
    // t-1's V, whose buffers are refilled.
    auto turn = [&](int t) {
        wait_copies<0>();
        __syncthreads();
        copy_k(t + 2);
        if (t > 0) copy_v(t + 1);
    };
    // Tile t (t % 2 == par): its exponentials and P V from sc, and tile t+1's scores into sn.  The scores run on the
    // matrix cores under the exponentials, and P V under the search for the next maximum; each slot is fenced, since the
    // compiler neither interleaves them by itself nor reads operands far enough ahead.
    auto step = [&](auto par, int t, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
        constexpr int P = decltype(par)::value;
        turn(t);
        const uint8_t *kt = kbuf[P ^ 1], *vt = vbuf[P];
        uint32_t pop[16];
        float l[4] = {0.f, 0.f, 0.f, 0.f};
        constexpr int kAhead = 5;    // operand reads in flight
        constexpr int kPairsA = 10;  // pairs of weights in the first phase; the others in the second, before they are needed
        u32x4 kf[kF], vf[kF];
        const float4 ks = meta4(kt + kF * 1024), ev = meta4(kt + kF * 1024 + 16), iv = meta4(vt + kF * 1024);
#pragma unroll
        for (int fi = 0; fi < kAhead; ++fi) kf[fi] = k_op(kt, fi);
        sn[0] = sn[1] = f32x16{};
#pragma unroll
        for (int fi = 0; fi < kF; ++fi) {
            if (fi + kAhead < kF) kf[fi + kAhead] = k_op(kt, fi + kAhead);
            else vf[fi + kAhead - kF] = k_op(vt, fi + kAhead - kF);
            sn[fi & 1] = mfma32<RQ_DTYPE_F16>(kf[fi], qop[fi >> 1], sn[fi & 1]);
#pragma unroll
            for (int i = kPairsA * fi / kF; i < kPairsA * (fi + 1) / kF; ++i) {
                exp_pair(sc, i, pop, l);
                asm volatile("" : "+v"(l[i >> 2]), "+v"(pop[i]));  // (values used only after the mask's branch would be computed there)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        mask(t + 1, sn);
        float gm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        __builtin_amdgcn_sched_barrier(0);
        constexpr int kPer = 32 / kF;           // scores of a slot of the second phase
        constexpr int kEvery = kF / 8;          // slots to a pair of weights there
#pragma unroll
        for (int fi = 0; fi < kF; ++fi) {
            if (fi + kAhead < kF) vf[fi + kAhead] = k_op(vt, fi + kAhead);
            const int g = fi / kM;
            acc[fi % kM] = mfma32<RQ_DTYPE_F16>(vf[fi], u32x4{pop[4 * g], pop[4 * g + 1], pop[4 * g + 2], pop[4 * g + 3]}, acc[fi % kM]);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const int x = kPer * fi + e;  // score x of 32
                gm[x >> 3] = fmaxf(gm[x >> 3], sn[x >> 4][x & 15]);
            }
            if (fi % kEvery == 0 && kPairsA + fi / kEvery < 16) exp_pair(sc, kPairsA + fi / kEvery, pop, l);
            __builtin_amdgcn_sched_barrier(0);
        }
        add_sums(l, iv);
        raise(gm, ks, ev);
    };
    // This wave's last tile.
    auto last = [&](const uint8_t *vt, const f32x16 (&sc)[2]) {
        uint32_t pop[16];
        float l[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) exp_pair(sc, i, pop, l);
        add_sums(l, meta4(vt + kF * 1024));
#pragma unroll
        for (int fi = 0; fi < kF; ++fi) {
            const int g = fi / kM;
            acc[fi % kM] = mfma32<RQ_DTYPE_F16>(k_op(vt, fi), u32x4{pop[4 * g], pop[4 * g + 1], pop[4 * g + 2], pop[4 * g + 3]}, acc[fi % kM]);
        }
    };
    int t = 0;
    while (t + 1 < nw) {
        step(std::integral_constant<int, 0>{}, t++, sa, sb);
        if (t + 1 >= nw) break;
        step(std::integral_constant<int, 1>{}, t++, sb, sa);
    }
    if (nw > 0) {
        turn(t);
        if (t & 1) last(vbuf[1], sb);
        else last(vbuf[0], sa);
        ++t;
    }
    for (; t < n_tiles; ++t) turn(t);  // tiles above this wave's diagonal: only their copies and barriers
    if (!wave_active) return;

    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
    const float l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    if (p.split > 1) {
        float *pt = a.part + ((((bl * p.nh + hl) * p.nx + qblk) * p.split + chunk) * kQ8PWaves + wave) * (int64_t)Im::kPart;
        if (hh == 0) *reinterpret_cast<float2 *>(pt + kQ8PW * D + 2 * col) = make_float2(q8_max_of(B), l);
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4 *>(pt + col * D + 32 * m + 8 * j + 4 * hh) =
                    make_float4(acc[m][4 * j], acc[m][4 * j + 1], acc[m][4 * j + 2], acc[m][4 * j + 3]);
        return;
    }
    if (my_i >= s.T) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a position that sees no key: zeros
    uint16_t *orow = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + my_i) * a.o_st + (int64_t)hq * a.o_sh;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint2 *>(orow + 32 * m + 8 * j + 4 * hh) = make_uint2(pack_pair<DT>(acc[m][4 * j] * inv, acc[m][4 * j + 1] * inv),
                                                                                    pack_pair<DT>(acc[m][4 * j + 2] * inv, acc[m][4 * j + 3] * inv));
}

// One workgroup per unit of a split call: thread (position tid / 8, part tid % 8) adds up D / 8 dims of the chunks.
template <int DT, int D>
__global__ __launch_bounds__(256) void q8_prefill_merge_kernel(Q8PrefillArgs p) {
    using Im = Q8Image<D>;
    constexpr int kDims = D / 8;
    const Q8AttnArgs &a = p.a;
    const int f = blockIdx.x, hl = blockIdx.y, h = p.h0 + hl, qblk = f / kQ8PWaves;
    const int64_t bl = blockIdx.z, b = p.b0 + bl;
    const Q8Block qb = q8_block(a, b, qblk);
    if (f >= qb.units) return;
    const int pos = threadIdx.x >> 3, part = threadIdx.x & 7;
    const int qi = f / a.G * kQ8PW + pos;
    if (qi >= qb.s.T) return;
    const int per = q8_chunk_tiles(qb.n_tiles, p.split), nch = (qb.n_tiles + per - 1) / per;
    const float *pt = a.part + ((((bl * p.nh + hl) * p.nx + qblk) * p.split) * kQ8PWaves + f % kQ8PWaves) * (int64_t)Im::kPart;
    float M = -INFINITY, l = 0.f, acc[kDims] = {};
    for (int c = 0; c < nch; ++c) {
        const float *pc = pt + c * (int64_t)kQ8PWaves * Im::kPart;
        const float2 ml = *reinterpret_cast<const float2 *>(pc + kQ8PW * D + 2 * pos);
        float4 x[kDims / 4];
#pragma unroll
        for (int k = 0; k < kDims / 4; ++k) x[k] = *reinterpret_cast<const float4 *>(pc + pos * D + kDims * part + 4 * k);
        const float Mn = fmaxf(M, ml.x);
        const float keep = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - Mn);
        const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - Mn);
        M = Mn;
        l = l * keep + w * ml.y;
#pragma unroll
        for (int k = 0; k < kDims / 4; ++k) {
            const float xs[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[4 * k + i] = acc[4 * k + i] * keep + w * xs[i];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *orow = static_cast<uint16_t *>(a.out) + (int64_t)(qb.s.q0 + qi) * a.o_st + (int64_t)(h * a.G + f % a.G) * a.o_sh + kDims * part;
#pragma unroll
    for (int k = 0; k < kDims; k += 4)
        *reinterpret_cast<uint2 *>(orow + k) = make_uint2(pack_pair<DT>(acc[k] * inv, acc[k + 1] * inv), pack_pair<DT>(acc[k + 2] * inv, acc[k + 3] * inv));
}

// ---- host ---------------------------------------------------------------------------
// A pass takes as many sequences as its images fit kQ8ImageBytes (the Infinity Cache's size: the attention
// then reads them from there), or as many kv heads of one sequence.
constexpr int64_t kQ8ImageBytes = 256LL << 20;
constexpr int kQ8SplitTiles = 8;  // tiles of a key chunk by the call's bound on the lengths, at least
// Key chunks where the workgroups fill at most half of the places (two a CU).  Chunks elsewhere, us for none / 2 / 3: one prompt of 700
// 24 / 33 / 33, of 2500 74 / 92 / 107; 500 tokens behind 3500 keys 55 / 57 / 58; two of about 1480 behind 4100 at head_dim 64 174 / 165 / 173 (1.47 rounds of
// workgroups there: two chunks gain, and no rule that takes them there and not elsewhere was looked for).
struct Q8PrefillShape {
    int64_t tiles, nb, nh, nx, split, image, images, part;
};
static Q8PrefillShape q8_prefill_shape(int64_t num_seqs, int G, int H, int D, int64_t max_q_len, int64_t max_keys) {
    Q8PrefillShape s;
    s.tiles = std::max<int64_t>(1, (max_keys + kQ8KT - 1) / kQ8KT);
    s.image = D == 128 ? Q8Image<128>::kBytes : Q8Image<64>::kBytes;
    const int64_t fit = std::max<int64_t>(1, kQ8ImageBytes / (s.tiles * s.image));  // (sequence, kv head) pairs of a pass
    s.nh = std::min<int64_t>(H, fit);
    s.nb = s.nh == H ? std::min<int64_t>(num_seqs, std::max<int64_t>(1, fit / H)) : 1;
    s.nx = ((max_q_len + kQ8PW - 1) / kQ8PW * G + kQ8PWaves - 1) / kQ8PWaves;
    const int64_t wgs = s.nx * s.nh * s.nb, slots = 2 * (int64_t)device_cus();
    s.split = 2 * wgs <= slots ? std::max<int64_t>(1, std::min<int64_t>(slots / wgs, s.tiles / kQ8SplitTiles)) : 1;
    s.images = s.nb * s.nh * s.tiles * s.image;
    const int64_t part = D == 128 ? Q8Image<128>::kPart : Q8Image<64>::kPart;
    s.part = s.split > 1 ? wgs * s.split * kQ8PWaves * part * 4 : 0;
    return s;
}

int64_t q8_prefill_workspace(int64_t num_seqs, int G, int H, int D, int64_t max_q_len, int64_t max_keys) {
    const Q8PrefillShape s = q8_prefill_shape(num_seqs, G, H, D, max_q_len, max_keys);
    return s.images + s.part;
}

// The images of a pass fit kQ8ImageBytes unless one pair's do not; split calls have a workgroup for each place at most.
int64_t q8_prefill_workspace_bound(int D, int64_t max_keys) {
    const int64_t tiles = std::max<int64_t>(1, (max_keys + kQ8KT - 1) / kQ8KT);
    const int64_t image = D == 128 ? Q8Image<128>::kBytes : Q8Image<64>::kBytes, part = D == 128 ? Q8Image<128>::kPart : Q8Image<64>::kPart;
    return std::max(kQ8ImageBytes, tiles * image) + 2 * (int64_t)device_cus() * kQ8PWaves * part * 4;
}

template <int DT, int FMT, int D>
static void q8_prefill_pass(const Q8PrefillArgs &p, int64_t nb, hipStream_t st) {
    using Im = Q8Image<D>;
    hipLaunchKernelGGL((q8_pack_kernel<FMT, D>), dim3((unsigned)p.max_tiles, (unsigned)p.nh, (unsigned)nb), dim3(256), 0, st, p);
    hipLaunchKernelGGL((q8_prefill_kernel<DT, D>), dim3((unsigned)(p.nx * p.split), (unsigned)p.nh, (unsigned)nb), dim3(64 * kQ8PWaves),
                       2 * (size_t)(Im::kLdsK + Im::kLdsV), st, p);
    if (p.split > 1)
        hipLaunchKernelGGL((q8_prefill_merge_kernel<DT, D>), dim3((unsigned)(p.nx * kQ8PWaves), (unsigned)p.nh, (unsigned)nb), dim3(256), 0, st, p);
}

int q8_prefill(const Q8AttnArgs &a, int dtype, int format, int D, void *workspace, hipStream_t st) {
    const Q8PrefillShape s = q8_prefill_shape(a.num_seqs, a.G, a.H, D, a.max_q, a.bound);
    Q8PrefillArgs p{};
    p.a = a;
    p.max_tiles = s.tiles;
    p.images = static_cast<uint8_t *>(workspace);
    p.a.part = reinterpret_cast<float *>(p.images + s.images);
    p.nx = (int)s.nx;
    p.split = (int)s.split;
    for (int64_t b = 0; b < a.num_seqs; b += s.nb)
        for (int64_t h = 0; h < a.H; h += s.nh) {
            p.b0 = (int)b;
            p.h0 = (int)h;
            p.nh = (int)std::min<int64_t>(s.nh, a.H - h);
            const int64_t nb = std::min<int64_t>(s.nb, a.num_seqs - b);
            const bool bf = dtype == RQ_DTYPE_BF16, i8 = format == RQ_Q8_INT8;
            if (D == 128) {
                if (bf) i8 ? q8_prefill_pass<RQ_DTYPE_BF16, RQ_Q8_INT8, 128>(p, nb, st) : q8_prefill_pass<RQ_DTYPE_BF16, RQ_Q8_E4M3, 128>(p, nb, st);
                else i8 ? q8_prefill_pass<RQ_DTYPE_F16, RQ_Q8_INT8, 128>(p, nb, st) : q8_prefill_pass<RQ_DTYPE_F16, RQ_Q8_E4M3, 128>(p, nb, st);
            } else {
                if (bf) i8 ? q8_prefill_pass<RQ_DTYPE_BF16, RQ_Q8_INT8, 64>(p, nb, st) : q8_prefill_pass<RQ_DTYPE_BF16, RQ_Q8_E4M3, 64>(p, nb, st);
                else i8 ? q8_prefill_pass<RQ_DTYPE_F16, RQ_Q8_INT8, 64>(p, nb, st) : q8_prefill_pass<RQ_DTYPE_F16, RQ_Q8_E4M3, 64>(p, nb, st);
            }
        }
    return check_launch("q8_prefill_kernel");
}

}  // namespace rq
