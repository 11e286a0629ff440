// What the attention kernels over the 8-bit cache (rq_q8_attention.hip) and over plain 16-bit pages (rq_kv16_attention.hip) share for
// queries of one or a few tokens: the batch, its work in equal shares, and the sums that several waves or workgroups join.
//
// Columns are the (token, query head) pairs that share a kv head, 16 to an MFMA; items are (sequence, block of 16 NB columns,
// kv head), in that order, and the tiles of all items in a row are cut into equal shares, one per workgroup.
#pragma once

#include "rq_attn_tile.h"

namespace rq {

constexpr int kShareCols = 16;     // columns of an MFMA; a workgroup takes NB blocks of them
constexpr int kShareTile = 32;     // keys of a tile
constexpr int kShareMinChunk = 8;  // tiles of a workgroup, at least

struct AttnBatch {
    const int32_t *cu_q;  // NULL: one token per sequence
    int64_t total_q, num_seqs;
    int causal;
    int H, G, block_size;
    const int32_t *bt;
    int64_t max_blocks, bt_ss;
    const int32_t *seq_lens;
    int64_t bound;  // max_seq_len: sizes launches and workspace
    int64_t cap;    // keys of a sequence that may be read: bound, its table's capacity
    int max_q;      // tokens of a query that count
    void *out;
    int64_t o_st, o_sh;
    float *part;  // partial sums of items that several workgroups share
};

// A sequence's query tokens that count (q0 .. q0 + T), the position of the first, and the keys that may be seen.
struct AttnSeq {
    int q0, T, pos, vis;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnBatch &a, int64_t b) {
    AttnSeq s;
    s.q0 = a.cu_q ? a.cu_q[b] : (int)b;
    const int end = a.cu_q ? a.cu_q[b + 1] : (int)b + 1;
    s.T = min(max(min((int64_t)end, a.total_q) - max(s.q0, 0), (int64_t)0), (int64_t)a.max_q);
    if (s.q0 < 0) s.T = 0;
    const int L = a.seq_lens[b];
    s.vis = (int)max((int64_t)0, min((int64_t)L, a.cap));
    // (by the query's whole length, also where max_q cuts it; far below 0, where no key is seen, or far above, where all are, the
    // exact place is of no account, and sums with a query's tokens stay ints)
    s.pos = (int)min(max((int64_t)L - ((int64_t)end - s.q0), (int64_t)-(1 << 30)), (int64_t)INT32_MAX - (1 << 21));
    return s;
}
__device__ __forceinline__ int attn_tiles(const AttnSeq &s) { return max(1, (s.vis + kShareTile - 1) / kShareTile); }
template <int NB>
__device__ __forceinline__ int attn_col_blocks(const AttnBatch &a, int T) { return (T * a.G + NB * kShareCols - 1) / (NB * kShareCols); }

// ---- shares -------------------------------------------------------------------
// Each workgroup sums over the sequences itself, 64 at a time.
template <int NB>
__device__ __forceinline__ int64_t attn_seq_tiles(const AttnBatch &a, int64_t b) {
    if (b >= a.num_seqs) return 0;
    const AttnSeq s = attn_seq(a, b);
    return (int64_t)attn_tiles(s) * attn_col_blocks<NB>(a, s.T) * a.H;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {  // inclusive
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
    return x;
}
// Of values under 2^41: the low 16 bits and the rest are summed apart.
__device__ __forceinline__ int64_t wave_scan64(int64_t x) {
    return (int64_t)wave_scan((uint32_t)x & 0xffffu) + ((int64_t)wave_scan((uint32_t)((uint64_t)x >> 16)) << 16);
}
__device__ __forceinline__ int64_t lane64(int64_t x, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)x >> 32), lane);
    return (int64_t)((uint64_t)hi << 32 | lo);
}
// a / b; in 32 bits (a tenth of the instructions) where both fit.
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int64_t attn_share(int64_t tiles, int workgroups) {
    return max((int64_t)kShareMinChunk, div64(tiles + workgroups - 1, workgroups));
}

template <int D>
struct AttnPartial {
    static constexpr int kFloats = kShareCols * (D + 2);  // of a block: accumulators by column, then (M, l) by column
};
template <int D, int W>
struct AttnSums {  // of a workgroup's W waves
    float acc[W][kShareCols][D + 4];
    float2 ml[W][kShareCols];
};

// Stores the first `left` of N values of a row (N = 2 or a multiple of 4; left a multiple of 4 unless N is 2).
template <int DT, int N>
__device__ __forceinline__ void attn_put(uint16_t *row, const float (&o)[N], float f, int left) {
    if constexpr (N == 2) {
        if (left > 0) *reinterpret_cast<uint32_t *>(row) = pack_pair<DT>(o[0] * f, o[1] * f);
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4)
            if (k < left) *reinterpret_cast<uint2 *>(row + k) = make_uint2(pack_pair<DT>(o[k] * f, o[k + 1] * f), pack_pair<DT>(o[k + 2] * f, o[k + 3] * f));
    }
}

// What a row of accumulators is multiplied by: 1 / l; rows that see no key are zeros.  NANS: weights may all be 0 where every
// score is -infinity, which is a NaN and no row without keys.
template <bool NANS>
__device__ __forceinline__ float attn_inv(const AttnBatch &a, const AttnSeq &s, int token, float l) {
    if constexpr (NANS) return s.vis > 0 && (!a.causal || s.pos + token >= 0) ? 1.f / l : 0.f;
    else return l == 0.f ? 0.f : 1.f / l;
}

// The sums of a workgroup's waves, which lie in lds (a barrier behind their writes), joined and put out: the output rows
// of block nb's columns from c0 (part == nullptr), or partials.
template <int DT, int D, int W, bool NANS>
__device__ __forceinline__ void attn_join(const AttnBatch &a, const AttnSeq &s, int h, int c0, int dims, float *part, const AttnSums<D, W> &lds) {
    constexpr int kPer = 4 * W, kDims = D / kPer;  // threads of a column, dims of a thread
    const int tid = threadIdx.x, c = tid / kPer, d0 = tid % kPer * kDims;
    const uint32_t cc = c0 + c, i = cc / (uint32_t)a.G;
    if ((int)i >= s.T) return;
    float Mt = -INFINITY, l = 0.f, o[kDims] = {};
#pragma unroll
    for (int w = 0; w < W; ++w) Mt = fmaxf(Mt, lds.ml[w][c].x);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 ml = lds.ml[w][c];
        const float r = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - Mt);
        l += r * ml.y;
#pragma unroll
        for (int k = 0; k < kDims; ++k) o[k] += r * lds.acc[w][c][d0 + k];
    }
    if (part == nullptr) {
        uint16_t *row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + (int)i) * a.o_st + (int64_t)(h * a.G + (int)(cc - i * a.G)) * a.o_sh + d0;
        attn_put<DT, kDims>(row, o, attn_inv<NANS>(a, s, (int)i, l), dims - d0);
    } else {
#pragma unroll
        for (int k = 0; k < kDims; k += 2) *reinterpret_cast<float2 *>(part + c * D + d0 + k) = make_float2(o[k], o[k + 1]);
        if (tid % kPer == 0) *reinterpret_cast<float2 *>(part + kShareCols * D + 2 * c) = make_float2(Mt, l);
    }
}

// Adds up the partials of the items that were cut: one workgroup of 256 threads per item and block of 16 columns.  A wave takes four
// columns (lane: column % 4, part of D / 16 dims); with few columns, as decodes have, several waves share them
// and take every second or fourth partial.  Two partials are in flight per wave.
template <int DT, int D, int NB, bool NANS>
__device__ __forceinline__ void attn_merge(const AttnBatch &a, int workgroups, int dims, AttnSums<D, 4> &lds) {
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
    attn_put<DT, kDims>(row, o, attn_inv<NANS>(a, s, i, l), dims - (tid & 15) * kDims);
}

// Walks a workgroup's equal share of all items' tiles: segment(sequence, its AttnSeq, kv head, first column, t0, t1, part) for
// each stretch of one item; part is nullptr where the item is the workgroup's alone.
template <int D, int NB, typename Segment>
__device__ __forceinline__ void attn_walk(const AttnBatch &a, Segment segment) {
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
        segment(seq, s, (int)(item - block_of * a.H), (int)block_of * (NB * kShareCols), t0, t1, part);
        pos += t1 - t0;
    }
}

// Workgroups of a call: what the GPU holds at once, or fewer where the bound on the lengths gives less work.
inline int64_t attn_workgroups(int64_t num_seqs, int G, int H, int64_t max_q_len, int64_t max_keys, int nb, int resident) {
    const int cols = nb * kShareCols;
    const int64_t tiles = max_keys / kShareTile + (max_keys % kShareTile != 0 || max_keys == 0);
    const int64_t work = num_seqs * ((max_q_len * G + cols - 1) / cols) * H * tiles, most = resident * (int64_t)device_cus();
    const int64_t wanted = (work + kShareMinChunk - 1) / kShareMinChunk;
    return wanted < 1 ? 1 : wanted < most ? wanted : most;
}

// Lengths are ints in the kernels.
inline int64_t attn_bound(int64_t max_seq_len) { return max_seq_len < INT32_MAX - 64 ? max_seq_len : INT32_MAX - 64; }

}  // namespace rq
