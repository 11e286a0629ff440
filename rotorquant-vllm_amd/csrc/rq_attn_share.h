// What the attention kernels over the 8-bit cache (rq_q8_attention.hip) and over plain 16-bit pages (rq_kv16_attention.hip) share for
// queries of one or a few tokens: the batch, its work in equal shares, and the sums that several waves or workgroups join.
//
// Columns are the (token, query head) pairs that share a kv head, 16 to an MFMA; an item is a (sequence, block of 16 NB columns, kv head).
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

// 2^d, d <= 0, for sums that may be infinite, which 0 would turn into NaN: at least the smallest number there is.  (A sum is at most its keys
// times the weight 1's scale times the largest value, so that this adds less than keys x 2^-149 of that to a row.)
__device__ __forceinline__ float attn_shrink(float d) { return fmaxf(__builtin_amdgcn_exp2f(d), 0x1p-149f); }

// What a row of accumulators is multiplied by: 1 / l; rows that see no key are zeros.  NANS: weights may all be 0 where every
// score is -infinity, which is a NaN and no row without keys.
template <bool NANS>
__device__ __forceinline__ float attn_inv(const AttnBatch &a, const AttnSeq &s, int token, float l) {
    if constexpr (NANS) return s.vis > 0 && (!a.causal || s.pos + token >= 0) ? 1.f / l : 0.f;
    else return l == 0.f ? 0.f : 1.f / l;
}

// The sums of a workgroup's waves, which lie in lds (a barrier behind their writes), joined and put out: the output rows
// of block nb's columns from c0 (part == nullptr), or partials.  NANS: sums may be infinite.
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
        const float r = ml.x == -INFINITY ? 0.f : NANS ? attn_shrink(ml.x - Mt) : __builtin_amdgcn_exp2f(ml.x - Mt);
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
