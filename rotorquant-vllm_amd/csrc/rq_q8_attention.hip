// Attention over the 8-bit KV cache (rq_q8_attention; format in rq_q8.h): queries of one or a few
// tokens, bound by the stream of codes from HBM.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(sm_scale q_i . k_j) over the keys j that i may see.
//
// Columns are the (token, query head) pairs that share a kv head, 16 to an MFMA.  Per group of 16 keys:
//   S^T = K Q^T   on v_mfma_f32_16x16x32_f16: codes c_k (exact in fp16) times q 2^s (s per column, the row's
//                 largest magnitude near 2^14: fp16 holds what bf16 does), fp32 sums;
//   u = S f + e_v, f = |sm_scale| log2(e) 2^(e_k - s): the score in base 2 plus the V exponent;
//   w = 2^(u + B) in fp16, B 7 to 15 less a column's running maximum of u (rq_q8_attn.h);
//   O^T += C_v^T w  (codes again exact), l += 2^-e_v sum w.
// So a group's two scales cost one multiplication per column and an addend that the exponent takes anyway, the
// weights are relative to the largest p 2^e_v whatever the groups' scales are, and out = O / l.
// l stays in fp32 whatever the scales: a token whose w underflows has under 2^-33 of the sum of p of the
// one that sets M (e_v is in -40 .. 60).
//
// Operands need neither LDS nor shuffles: a lane's 16 bytes of K and V are its operands' elements (rq_q8.h), and
// the weights come out of S^T in the order that P V takes.
//
// What bounds it: the stream of codes.  64 sequences of 1024 to 8192 keys, 8 kv heads x 4 (609 MB): the stream kernel
// 99 to 102 us, 6.0 TB/s, which is what a plain read reaches on this card; whole call 106, the merge 4.8.  A wave holds
// the next tile (8 KB at head_dim 128) in registers while it computes one; two workgroups of four waves a CU (175
// registers) keep 64 KB a CU on their way.  Three workgroups a CU (168 registers, 10 spilled, or one tile of registers
// refilled as it is used) 127 to 130 us against 127 before the loads became non-temporal; two tiles ahead 109 against 107;
// twice or four times the workgroups, which balance themselves, 130 and 139 (more partials, more prologues).  Small calls: at
// q8_item_kernel.
#include <algorithm>
#include <cmath>

#include "rq_q8_attn.h"

namespace rq {

// ---- one segment ----------------------------------------------------------------
__device__ __forceinline__ uint32_t rows_umax(uint32_t x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(r[0], r[1]);
    auto t = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max(t[0], t[1]);
}
// One column's operands: q 2^s in fp16 in K's dim order, and f without the group's 2^e_k.
template <int DT, int D>
__device__ __forceinline__ float q8_query(const Q8AttnArgs &a, u32x4 (&qop)[D / 32]) {
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) big = q8_max_bits(qop[k], big);
    const int up = q8_query_exp<DT>(a, rows_umax(big));
    const float f = exp2i(up) * a.q_sign;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) qop[k] = q8_query_f16<DT>(qop[k], f);
    return a.score_scale * exp2i(-up);
}

// Codes of one tile: two groups.
template <int D>
struct Q8Tile {
    u32x4 k[2][D / 64], v[2][D / 64];
};
// Tiles [t0, t1) of the item (sequence, kv head h, columns from c0) by the workgroup's W waves, tile t0 + i by wave i % W.  The result is
// the output rows (part == NULL) or partials.
// ONCE: no other workgroup reads these codes.
template <int DT, int FMT, int D, int NB, int W, bool ONCE>
__device__ __forceinline__ void q8_segment(const Q8AttnArgs &a, int64_t seq, const AttnSeq &s, int h, int c0, int t0, int t1, float *part,
                                           AttnSums<D, W> &lds) {
    constexpr int kSteps = D / 32, kChunks = D / 64, kBlocks = D / 16;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const Q8Layout lay(a.H, D, a.block_size);
    // Lane l looks up group l % 2 of the (l / 2)-th of this wave's next 32 tiles.
    const int last_group = max(0, (s.vis + kQ8Group - 1) / kQ8Group - 1);
    int64_t at = 0;
    float2 sc = make_float2(0.f, 0.f);
    auto look_up = [&](int first) {
        const uint32_t gi = (uint32_t)min(2 * (first + W * (lane >> 1)) + (lane & 1), last_group);
        const uint32_t p = gi / (uint32_t)a.groups;
        int64_t page = s.vis > 0 ? a.bt[seq * a.bt_ss + p] : 0;
        page = page < 0 || page >= a.num_blocks ? 0 : page;
        at = page * a.stride_block + lay.codes_at(gi - p * a.groups, h);
        sc = *reinterpret_cast<const float2 *>(a.cache + page * a.stride_block + lay.scale_at(gi - p * a.groups, h));
    };
    auto slot = [&](int t) { return (t - t0) / W & 31; };
    // Codes read once come by non-temporal loads (64 sequences of 4600 keys on average, 8 kv heads: 126 us -> 114; 32
    // sequences of 4000, 8 tokens x 4: 65.8 -> 60.1), codes that several column blocks read by ordinary ones (the latter with 16
    // tokens: 82.1 -> 76.0, with 48: 265 -> 245).
    Q8Tile<D> next;
    auto code16 = [](const uint8_t *p) {
        const u32x4 *const q = reinterpret_cast<const u32x4 *>(p);
        return ONCE ? __builtin_nontemporal_load(q) : *q;
    };
    auto fetch = [&](int t) {
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
            const uint8_t *p = a.cache + lane64(at, 2 * slot(t) + gr);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                next.k[gr][j] = code16(p + 1024 * j + 16 * lane);
                next.v[gr][j] = code16(p + kQ8Group * D + 1024 * j + 16 * lane);
            }
        }
    };
    int t = t0 + wave;
    // (the look-up's loads depend on one another; the query's are issued between them)
    if (t < t1) look_up(t);
    u32x4 qop[NB][kSteps];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const uint32_t c = c0 + kShareCols * nb + col, i = c / (uint32_t)a.G;
        const bool valid = (int)i < s.T;
        const uint16_t *row = static_cast<const uint16_t *>(a.q) + (int64_t)(s.q0 + (valid ? (int)i : 0)) * a.q_st +
                              (int64_t)(h * a.G + (valid ? (int)(c - i * a.G) : 0)) * a.q_sh + 16 * g;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
            qop[nb][k] = valid ? *reinterpret_cast<const u32x4 *>(row + 64 * (k >> 1) + 8 * (k & 1)) : u32x4{0u, 0u, 0u, 0u};
    }
    if (t < t1) fetch(t);
    float colf[NB], B[NB], l_run[NB];
    int lim[NB];  // keys that this lane's column sees
    f32x4 acc[NB][kBlocks];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        colf[nb] = q8_query<DT, D>(a, qop[nb]);
        lim[nb] = a.causal ? min(s.vis, s.pos + (c0 + kShareCols * nb + col) / a.G + 1) : s.vis;
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) acc[nb][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        B[nb] = kQ8NoBias, l_run[nb] = 0.f;
    }
    const int lim_first = a.causal ? min(s.vis, s.pos + c0 / a.G + 1) : s.vis;  // the fewest that any column sees

    for (; t < t1; t += W) {
        int ev[2];
        float ks[2];
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
            ks[gr] = exp2i(q8_scale_exp(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.x), 2 * slot(t) + gr))));
            ev[gr] = q8_scale_exp(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.y), 2 * slot(t) + gr)));
        }
        Q8Tile<D> cur = next;
        const int tn = t + W;
        if (tn < t1) {
            if (slot(tn) == 0) look_up(tn);
            fetch(tn);
        }
        const int k0 = t * kShareTile;
        f32x4 S[NB][2];
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) S[nb][gr] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const u32x4 w = cur.k[gr][k >> 1];
                uint32_t x[4];
                q8_to_f16<FMT>(w[2 * (k & 1)], x[0], x[1]);
                q8_to_f16<FMT>(w[2 * (k & 1) + 1], x[2], x[3]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) S[nb][gr] = mfma_f16(u32x4{x[0], x[1], x[2], x[3]}, qop[nb][k], S[nb][gr]);
            }
        }
        if (k0 + kShareTile > lim_first) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[nb][gr][i] = k0 + 16 * gr + 4 * g + i < lim[nb] ? S[nb][gr][i] : -INFINITY;
            if (FMT == RQ_Q8_E4M3 && k0 + kShareTile > s.vis) {
                // what lies behind the context may be a NaN's code, and 0 * NaN is one
#pragma unroll
                for (int gr = 0; gr < 2; ++gr) {
                    const int left = min(4, max(0, s.vis - (k0 + 16 * gr + 4 * g)));
                    const uint32_t keep = left == 4 ? ~0u : (1u << (8 * left)) - 1u;
#pragma unroll
                    for (int j = 0; j < kChunks; ++j) cur.v[gr][j] &= u32x4{keep, keep, keep, keep};
                }
            }
        }
        u32x4 pw[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float f[2] = {colf[nb] * ks[0], colf[nb] * ks[1]};
            float tmax = -INFINITY;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const f32x4 x = S[nb][gr];
                tmax = fmaxf(tmax, __builtin_fmaf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), f[gr], (float)ev[gr]));
            }
            if (__any(q8_passes(tmax, B[nb]))) {
                const float b_new = fminf(B[nb], kQ8Peak - rows_max(tmax));
                const float alpha = __builtin_amdgcn_exp2f(b_new - B[nb]);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) acc[nb][m] *= alpha;
                l_run[nb] *= alpha;
                B[nb] = b_new;
            }
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const float add = B[nb] + (float)ev[gr];
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[nb][gr][i], f[gr], add));
                pw[nb][2 * gr] = pack_f16(w[0], w[1]);
                pw[nb][2 * gr + 1] = pack_f16(w[2], w[3]);
                // the sum of the weights before their rounding to fp16 (which has no bias)
                l_run[nb] = __builtin_fmaf((w[0] + w[1]) + (w[2] + w[3]), exp2i(-ev[gr]), l_run[nb]);
            }
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x[4];
                q8_to_f16<FMT>(cur.v[0][j][i], x[0], x[1]);
                q8_to_f16<FMT>(cur.v[1][j][i], x[2], x[3]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) acc[nb][4 * j + i] = mfma_f16(u32x4{x[0], x[1], x[2], x[3]}, pw[nb], acc[nb][4 * j + i]);
            }
    }

    // the waves' sums
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float l_col = rows_sum(l_run[nb]);
        __syncthreads();  // (the sums before these are read)
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) *reinterpret_cast<f32x4 *>(&lds.acc[wave][col][16 * m + 4 * g]) = acc[nb][m];
        if (g == 0) lds.ml[wave][col] = make_float2(q8_max_of(B[nb]), l_col);
        __syncthreads();
        attn_join<DT, D, W, false>(a, s, h, c0 + kShareCols * nb, D, part == nullptr ? nullptr : part + nb * AttnPartial<D>::kFloats, lds);
    }
}

// Workgroups of a CU at once (by registers, 4 waves each).
template <int D, int NB>
constexpr int kQ8Resident = D == 64 ? (NB == 1 ? 4 : 3) : 2;

// The tiles of all items, in the order sequence, block of columns, kv head, in a row and cut into equal shares.
template <int DT, int FMT, int D, int NB, bool ONCE>
__global__ __launch_bounds__(256, (kQ8Resident<D, NB>)) void q8_stream_kernel(Q8AttnArgs a) {
    __shared__ AttnSums<D, 4> lds;
    const int lane = threadIdx.x & 63;
    int64_t block = 0, block_base = 0;  // 64 sequences: their tiles, and the row's up to each
    int64_t mine = attn_seq_tiles<NB>(a, lane), upto = wave_scan64(mine);
    int64_t total = lane64(upto, 63);
    for (int64_t b = 64; b < a.num_seqs; b += 64) total += lane64(wave_scan64(attn_seq_tiles<NB>(a, b + lane)), 63);
    const int64_t share = attn_share(total, gridDim.x);
    int64_t pos = blockIdx.x * share;
    const int64_t end = min(total, pos + share);
    while (pos < end) {
        uint64_t hit = __ballot(block_base + upto > pos);
        while (hit == 0) {
            block_base += lane64(upto, 63);
            block += 64;
            mine = attn_seq_tiles<NB>(a, block + lane);
            upto = wave_scan64(mine);
            hit = __ballot(block_base + upto > pos);
        }
        const int of = __builtin_ctzll(hit);
        const int64_t seq = block + of, in_seq = pos - (block_base + lane64(upto, of) - lane64(mine, of));
        const AttnSeq s = attn_seq(a, seq);
        const int n = attn_tiles(s);
        const int64_t item = div64(in_seq, n), block_of = div64(item, a.H);
        const int t0 = (int)(in_seq - item * n), t1 = (int)min((int64_t)n, t0 + (end - pos));
        // an item cut in two or more: the share that begins it ends with it, the others begin with it
        float *part = t0 == 0 && t1 == n ? nullptr : a.part + (2 * (int64_t)blockIdx.x + (t0 == 0 ? 1 : 0)) * NB * AttnPartial<D>::kFloats;
        q8_segment<DT, FMT, D, NB, 4, ONCE>(a, seq, s, (int)(item - block_of * a.H), (int)block_of * (NB * kShareCols), t0, t1, part, lds);
        pos += t1 - t0;
    }
}

// Adds up the partials of the items that were cut: one workgroup per item and block of 16 columns.  A wave takes four
// columns (lane: column % 4, part of D / 16 dims); with few columns, as decodes have, several waves share them
// and take every second or fourth partial.  Two partials are in flight per wave.
template <int DT, int D, int NB>
__global__ __launch_bounds__(256) void q8_merge_kernel(Q8AttnArgs a, int workgroups) {
    __shared__ AttnSums<D, 4> lds;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int64_t b = blockIdx.y;
    const int item = blockIdx.x / NB, nb = blockIdx.x % NB;
    const AttnSeq s = attn_seq(a, b);
    const int h = item % a.H, c0 = (item / a.H) * (NB * kShareCols) + nb * kShareCols;
    const int cols = min(kShareCols, s.T * a.G - c0);
    if (cols <= 0) return;
    const int n = attn_tiles(s);
    int64_t total = 0, before = 0;
    for (int64_t b0 = 0; b0 < a.num_seqs; b0 += 64) {
        const int64_t mine = attn_seq_tiles<NB>(a, b0 + lane), upto = wave_scan64(mine);
        if (b >= b0 && b < b0 + 64) before = total + lane64(upto, (int)(b - b0)) - lane64(mine, (int)(b - b0));
        total += lane64(upto, 63);
    }
    const int64_t share = attn_share(total, workgroups);
    const int64_t first = before + (int64_t)item * n;
    const int w0 = (int)div64(first, share), w1 = (int)div64(first + n - 1, share);
    if (w0 == w1) return;
    constexpr int kDims = D / 16;
    const int quads = cols > 8 ? 4 : cols > 4 ? 2 : 1, ways = 4 / quads;  // column quads, waves of each
    const int way = wave / quads, d0 = (lane & 15) * kDims;
    {
        const int c = 4 * (wave % quads) + (lane >> 4), cv = min(c, cols - 1);
        float M = -INFINITY, l = 0.f, o[kDims] = {};
        for (int w = w0 + way; w <= w1; w += 2 * ways) {
            float2 ml[2];
            float4 x[2][kDims / 4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int wu = min(w + ways * u, w1);
                const float *pt = a.part + ((2 * (int64_t)wu + (wu == w0 ? 1 : 0)) * NB + nb) * AttnPartial<D>::kFloats;
                ml[u] = *reinterpret_cast<const float2 *>(pt + kShareCols * D + 2 * cv);
#pragma unroll
                for (int k = 0; k < kDims / 4; ++k) x[u][k] = *reinterpret_cast<const float4 *>(pt + cv * D + d0 + 4 * k);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (w + ways * u > w1) continue;
                const float Mn = fmaxf(M, ml[u].x);
                const float keep = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - Mn);
                const float r = ml[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[u].x - Mn);
                M = Mn;
                l = l * keep + r * ml[u].y;
#pragma unroll
                for (int k = 0; k < kDims / 4; ++k) {
                    o[4 * k] = o[4 * k] * keep + r * x[u][k].x, o[4 * k + 1] = o[4 * k + 1] * keep + r * x[u][k].y;
                    o[4 * k + 2] = o[4 * k + 2] * keep + r * x[u][k].z, o[4 * k + 3] = o[4 * k + 3] * keep + r * x[u][k].w;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kDims; k += 4) *reinterpret_cast<float4 *>(&lds.acc[way][c][d0 + k]) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        if ((lane & 15) == 0) lds.ml[way][c] = make_float2(M, l);
    }
    __syncthreads();
    const int c = tid >> 4;
    if (c >= cols) return;
    float Mt = -INFINITY, l = 0.f, o[kDims] = {};
    for (int w = 0; w < ways; ++w) Mt = fmaxf(Mt, lds.ml[w][c].x);
    for (int w = 0; w < ways; ++w) {
        const float2 ml = lds.ml[w][c];
        const float r = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - Mt);
        l += r * ml.y;
#pragma unroll
        for (int k = 0; k < kDims; ++k) o[k] += r * lds.acc[w][c][(tid & 15) * kDims + k];
    }
    const int i = (c0 + c) / a.G;
    uint16_t *row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + i) * a.o_st + (int64_t)(h * a.G + (c0 + c) % a.G) * a.o_sh + (tid & 15) * kDims;
    attn_put<DT, kDims>(row, o, attn_inv<false>(a, s, i, l), kDims);
}

// One workgroup of 8 waves per item: one launch, no partials.  What bounds it is two things in a row.  A chain of dependent loads and its
// launch -- lengths, block table, codes, then the sums of the waves: 5.2 us (one sequence of 16 keys, 8 kv heads x 4).  Then
// what one CU loads, since an item is one workgroup's: 4.7 us for each 1000 keys beyond the first 100 (a tile a wave per 1.07 us, 54 to
// 61 GB/s; 777 to 800 keys 8.6 to 9.3 us, 1600 12.4).  Two, three or four tiles ahead instead of one: 8.7, 9.0 and 9.0 us against 8.6
// (777 keys), so it is the rate and not the latency; more CUs to an item would need a merge between workgroups.
template <int DT, int FMT, int D, int NB, bool ONCE>
__global__ __launch_bounds__(512, 2) void q8_item_kernel(Q8AttnArgs a) {
    __shared__ AttnSums<D, 8> lds;
    const int64_t seq = blockIdx.y;
    const AttnSeq s = attn_seq(a, seq);
    const int block = blockIdx.x / (uint32_t)a.H, h = blockIdx.x - block * a.H;
    if (block >= attn_col_blocks<NB>(a, s.T)) return;
    q8_segment<DT, FMT, D, NB, 8, ONCE>(a, seq, s, h, block * (NB * kShareCols), 0, attn_tiles(s), nullptr, lds);
}

// Blocks of 16 columns that a workgroup takes (two share a stream of codes and its conversions: 32 drafts of up to 8 tokens x 4 heads
// 85 -> 77 us), and the workgroups: what the GPU holds at once, or fewer where the bound on the lengths gives less work.
static int q8_blocks(int G, int64_t max_q_len) { return max_q_len * G > kShareCols ? 2 : 1; }
static int64_t q8_workgroups(int64_t num_seqs, int G, int H, int D, int64_t max_q_len, int64_t max_keys) {
    const int nb = q8_blocks(G, max_q_len);
    const int resident = D == 128 ? (nb == 1 ? kQ8Resident<128, 1> : kQ8Resident<128, 2>) : (nb == 1 ? kQ8Resident<64, 1> : kQ8Resident<64, 2>);
    return attn_workgroups(num_seqs, G, H, max_q_len, max_keys, nb, resident);
}

// Calls of short contexts, by the bound on their lengths, take a workgroup per item.  One launch without partials saves 4 to 7 us; a long item
// by itself is slower, as one workgroup walks it.  8 kv heads x 4, equal lengths, graph replays, items / shares:
//   1 sequence of 800 keys 8.6 / 13.7 us, 1600: 12.4 / 14.3, 3200: 19.3 / 14.3;  8: 9.5 / 14.5, 13.6 / 17.2, 22.1 / 20.3;
//   64: 24.6 / 25.0, 40.8 / 42.4, 73.5 / 78.0.
constexpr int64_t kQ8ItemTiles = 60;
static bool q8_is_short(int64_t max_keys) {
    return max_keys <= kQ8ItemTiles * kShareTile;
}

template <int DT, int FMT, int D, int NB, bool ONCE>
static void launch_stream(const Q8AttnArgs &a, int64_t workgroups, hipStream_t st) {
    if (q8_is_short(a.bound)) {
        const int64_t items = ((int64_t)a.max_q * a.G + NB * kShareCols - 1) / (NB * kShareCols) * a.H;
        hipLaunchKernelGGL((q8_item_kernel<DT, FMT, D, NB, ONCE>), dim3((unsigned)items, (unsigned)a.num_seqs), dim3(512), 0, st, a);
        return;
    }
    hipLaunchKernelGGL((q8_stream_kernel<DT, FMT, D, NB, ONCE>), dim3((unsigned)workgroups), dim3(256), 0, st, a);
    const int64_t items = ((int64_t)a.max_q * a.G + NB * kShareCols - 1) / (NB * kShareCols) * a.H;
    hipLaunchKernelGGL((q8_merge_kernel<DT, D, NB>), dim3((unsigned)(items * NB), (unsigned)a.num_seqs), dim3(256), 0, st, a, (int)workgroups);
}
template <int DT, int FMT, int D>
static void launch_stream_b(const Q8AttnArgs &a, int64_t wgs, hipStream_t st) {
    if (q8_blocks(a.G, a.max_q) == 1) launch_stream<DT, FMT, D, 1, true>(a, wgs, st);
    else if ((int64_t)a.max_q * a.G <= 2 * kShareCols) launch_stream<DT, FMT, D, 2, true>(a, wgs, st);
    else launch_stream<DT, FMT, D, 2, false>(a, wgs, st);
}
template <int DT, int FMT>
static void launch_stream_d(const Q8AttnArgs &a, int D, int64_t wgs, hipStream_t st) {
    D == 128 ? launch_stream_b<DT, FMT, 128>(a, wgs, st) : launch_stream_b<DT, FMT, 64>(a, wgs, st);
}
template <int DT>
static void launch_stream_f(const Q8AttnArgs &a, int fmt, int D, int64_t wgs, hipStream_t st) {
    fmt == RQ_Q8_INT8 ? launch_stream_d<DT, RQ_Q8_INT8>(a, D, wgs, st) : launch_stream_d<DT, RQ_Q8_E4M3>(a, D, wgs, st);
}

// Calls of RQ_Q8_PROMPT_COLUMNS per kv head or more go to the prefill kernels.  8 kv heads x 4, queries of 1 to n tokens, these / those:
// 8 sequences of 8000 keys, n = 20: 58 / 156 us, 32: 95 / 160, 47: 128, 64: 164 / 196;  32 of 1000, 32: 58 / 77, 64: 109 / 81;  1 of
// 8000, 64: 40 / 40;  head_dim 64, 8 of 4000, 32: 38 / 44, 64: 52 / 51.
static bool q8_is_prompt(int64_t max_q_len, int G) { return max_q_len > 1 && max_q_len * G >= RQ_Q8_PROMPT_COLUMNS; }

}  // namespace rq

using namespace rq;

extern "C" int64_t rq_q8_attention_workspace_bytes(int64_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                                   int32_t head_dim, int64_t max_q_len, int64_t max_seq_len) {
    if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0 || max_q_len <= 0 || max_seq_len < 0) return 0;
    const int G = num_q_heads / num_kv_heads;
    max_seq_len = attn_bound(max_seq_len);
    if (q8_is_prompt(max_q_len, G)) return q8_prefill_workspace(num_seqs, G, num_kv_heads, head_dim, max_q_len, max_seq_len);
    if (q8_is_short(max_seq_len)) return 0;
    const int64_t wgs = q8_workgroups(num_seqs, G, num_kv_heads, head_dim, max_q_len, max_seq_len);
    return 2 * wgs * q8_blocks(G, max_q_len) * kShareCols * (head_dim + 2) * 4;
}

// (The stream's partials, two of up to 2 x 16 columns for each of up to four workgroups a CU, are smaller than the prefill's.)
extern "C" int64_t rq_q8_attention_workspace_bound(int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t max_seq_len) {
    if (num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0 || max_seq_len < 0) return 0;
    return q8_prefill_workspace_bound(head_dim, attn_bound(max_seq_len));
}

extern "C" int rq_q8_attention(const void *q, int32_t dtype, int64_t total_q, int32_t num_q_heads,
                               int64_t q_stride_tok, int64_t q_stride_head, const int32_t *cu_seqlens_q, int64_t num_seqs,
                               int64_t max_q_len, int32_t causal, const uint8_t *kv_cache, int64_t num_blocks,
                               int32_t block_size, int64_t stride_block, int32_t num_kv_heads, int32_t head_dim,
                               int32_t format, const int32_t *block_table, int64_t max_blocks, int64_t bt_stride_seq,
                               const int32_t *seq_lens, int64_t max_seq_len, float sm_scale, void *out,
                               int64_t out_stride_tok, int64_t out_stride_head, void *workspace, int64_t workspace_bytes,
                               void *stream) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_BF16 || dtype == RQ_DTYPE_F16, "q must be f16 or bf16");
    const int rc = check_q8_cache(head_dim, num_kv_heads, block_size, num_blocks, kv_cache, stride_block, format);
    if (rc) return rc;
    RQ_CHECK_ARG(num_q_heads >= 1 && num_q_heads <= 65536 && num_q_heads % num_kv_heads == 0,
                 "num_q_heads %d must be a multiple of num_kv_heads %d", num_q_heads, num_kv_heads);
    RQ_CHECK_ARG(num_seqs >= 0 && num_seqs <= 65535 && total_q >= 0 && total_q <= INT32_MAX && max_q_len >= 0 && max_q_len <= (1 << 20) &&
                     max_blocks >= 0 && max_seq_len >= 0, "bad sizes");
    RQ_CHECK_ARG(cu_seqlens_q != nullptr || (total_q == num_seqs && max_q_len <= 1),
                 "without cu_seqlens_q there is one query token per sequence");
    uint32_t scale_bits;  // (by its bits: this file is compiled for arithmetic without NaN)
    __builtin_memcpy(&scale_bits, &sm_scale, 4);
    RQ_CHECK_ARG((scale_bits & 0x7f800000u) != 0x7f800000u, "sm_scale must be finite");
    RQ_CHECK_ARG(__builtin_fabsf(sm_scale) <= 0x1p127f, "sm_scale %g is past 2^127", (double)sm_scale);  // (times log2(e) it is finite)
    if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return RQ_OK;
    RQ_CHECK_ARG(num_blocks > 0, "the cache has no pages");
    RQ_CHECK_ARG(q && out && seq_lens && (block_table || max_blocks == 0), "null pointer");
    RQ_CHECK_ARG((uintptr_t)q % 16 == 0 && q_stride_tok % 8 == 0 && q_stride_head % 8 == 0, "q rows must be 16-byte aligned");
    RQ_CHECK_ARG((uintptr_t)out % 8 == 0 && out_stride_tok % 4 == 0 && out_stride_head % 4 == 0, "out rows must be 8-byte aligned");
    Q8AttnArgs a{};
    a.q = q, a.q_st = q_stride_tok, a.q_sh = q_stride_head;
    a.cu_q = cu_seqlens_q;
    a.total_q = total_q, a.num_seqs = num_seqs;
    a.causal = causal != 0;
    a.cache = kv_cache, a.num_blocks = num_blocks, a.stride_block = stride_block;
    a.H = num_kv_heads, a.G = num_q_heads / num_kv_heads, a.groups = block_size / kQ8Group, a.block_size = block_size;
    a.bt = block_table, a.max_blocks = max_blocks, a.bt_ss = bt_stride_seq;
    a.seq_lens = seq_lens;
    a.bound = attn_bound(max_seq_len);
    a.cap = std::min<int64_t>(a.bound, max_blocks > a.bound / block_size ? a.bound : max_blocks * block_size);
    a.max_q = (int)max_q_len;
    a.score_scale = sm_scale == 0.f ? 1.f : __builtin_fabsf(sm_scale) * kAttnLog2e;
    a.q_sign = sm_scale > 0.f ? 1.f : sm_scale < 0.f ? -1.f : 0.f;
    a.max_up = std::min(60, 86 + std::ilogb(a.score_scale));  // (of numbers under 2^-126, too)
    a.out = out, a.o_st = out_stride_tok, a.o_sh = out_stride_head;
    const int64_t need = rq_q8_attention_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, max_seq_len);
    RQ_CHECK_SPACE(workspace_bytes >= need, "workspace too small: the call needs %lld bytes (got %lld)", (long long)need, (long long)workspace_bytes);
    RQ_CHECK_ARG(need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "workspace must be 16-byte aligned");
    a.part = static_cast<float *>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if (q8_is_prompt(a.max_q, a.G)) return q8_prefill(a, dtype, format, head_dim, workspace, st);
    const int64_t wgs = q8_workgroups(num_seqs, a.G, a.H, head_dim, a.max_q, a.bound);
    if (dtype == RQ_DTYPE_BF16) launch_stream_f<RQ_DTYPE_BF16>(a, format, head_dim, wgs, st);
    else launch_stream_f<RQ_DTYPE_F16>(a, format, head_dim, wgs, st);
    return check_launch("q8_stream_kernel");
}
