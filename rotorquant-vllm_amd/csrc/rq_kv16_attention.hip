// Attention over plain 16-bit pages (rq_kv16_attention): queries of one or a few tokens, bound by the stream of K and V from HBM.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(sm_scale q_i . k_j) over the keys j that i may see.
//
// Columns are the (token, query head) pairs that share a kv head, 16 to an MFMA.  Per tile of 32 keys of a wave:
//   S^T = K Q^T  on v_mfma_f32_16x16x32 of the pages' type (products exact, sums fp32), two 16-key halves;
//   w = 2^(u - m) 2^peak, u = S sm_scale log2(e), m a column's running maximum; l += w in fp32;
//   O^T += V^T w, w as 16-bit numbers (its rounding, the rounding of what that leaves, ...): two of fp16 or three of bf16 have
//                 the bits of an fp32 weight.  The third costs 1 % (one sequence of 777 keys 10.23 / 10.38 us, 32 drafts 133.2 / 134.3, 24 sequences
//                 over one head of 256 31.3 / 31.6), and nothing in long decodes.
// peak is 14 for fp16, whose small numbers end at 2^-24, and -24 for bf16, whose largest end where fp32's do: sums of 2^24 of them do not overflow.
// out = O / l.
//
// Rows may lie anywhere (any page size and strides): lane l looks up where key l % 32 of a tile is, a tile ahead, and lanes ask it
// by bpermute.  K needs no more: a lane's 16 bytes are operand elements.  V is loaded by rows, 16 lanes to a row, and its operand
// (two tokens of a dim in a dword) made by one byte permute a dword: dim 8 c + m of lane c is row c of product m.
#include <algorithm>
#include <type_traits>

#include "rq_attn_share.h"

namespace rq {

struct Kv16Args : AttnBatch {
    const void *q;
    int64_t q_st, q_sh;
    const uint16_t *k, *v;
    int64_t num_blocks;
    uint32_t k_sb, k_ss, v_sb, v_ss;  // 8 elements between pages, slots
    int64_t k_sh, v_sh;               // elements between heads
    int D;
    float scale;  // sm_scale log2(e)
};

template <typename T>
__device__ __forceinline__ T kv16_load(const uint16_t *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
}

// Infinities and NaN are the 16-bit numbers whose magnitude, as an integer, is kHuge or more.
template <int DT>
constexpr uint32_t kHuge = DT == RQ_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
__device__ __forceinline__ uint32_t larger16(uint32_t big, uint32_t w) {  // of magnitudes, by halves
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, big), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
template <int DT>
__device__ __forceinline__ uint32_t huge_halves(uint32_t w) {  // all ones where a half is an infinity or NaN
    return ((w & 0x7fffu) >= kHuge<DT> ? 0xffffu : 0u) | ((w >> 16 & 0x7fffu) >= kHuge<DT> ? 0xffff0000u : 0u);
}

// Tiles [t0, t1) of the item (sequence, kv head h, columns from c0) by the workgroup's W waves, tile t0 + i by wave i % W.  The result is
// the output rows (part == nullptr) or partials.  DP: D rounded up to 64, 128 or 256 (FULL: D is that).
//
// Keys past the context are loaded as its last one, with a weight of 0.  0 * infinity is a NaN, there and where an infinite V is hidden
// from some columns, and a weight's further parts may be 0 or negative: so a segment that met an infinity or NaN in V is done again, as FAR,
// which adds one token's columns at a time, with the rows that token sees, and the infinities apart, by weights of 1 wherever the score is finite
// (its weight may round to 0, and 0 * infinity is a NaN).  Sums that are infinite stay so when they are scaled and joined.
// HEADS: each wave has a head of its own and all the tiles (W is 1); otherwise the waves share a head.
template <int DT, int DP, bool FULL, int NB, int W, bool HEADS, bool FAR = false>
__device__ __forceinline__ void kv16_segment(const Kv16Args &a, int64_t seq, const AttnSeq &s, int h, int c0, int t0, int t1, float *part,
                                             AttnSums<DP, W> &lds) {
    constexpr int kSteps = DP / 32, kBlocks = DP / 16;
    constexpr int kVDims = DP == 64 ? 4 : 8, kVParts = DP == 256 ? 2 : 1;  // dims of a lane's V load, loads of a row
    constexpr int kParts = DT == RQ_DTYPE_F16 ? 2 : 3;  // 16-bit numbers of a weight
    constexpr float kPeak = DT == RQ_DTYPE_F16 ? 0x1p14f : 0x1p-24f;
    using VRow = std::conditional_t<DP == 64, u32x2, u32x4>;
    const int lane = threadIdx.x & 63, wave = HEADS ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, D = FULL ? DP : a.D;

    // Where the rows of a tile are: lane l has key l % 32.  Past the last key that counts here, that one again.
    const int last = max(0, min(s.vis, t1 * kShareTile) - 1);
    int page = 0, slot = 0;         // of the tile that comes next
    uint32_t k_row = 0, v_row = 0;  // of the present one: 16-byte units from the head's first row (under 2^32, the host checks)
    auto look_up = [&](int j) {
        const uint32_t key = min((uint32_t)(t0 + wave + W * j) * kShareTile + (lane & 31), (uint32_t)last), p = key / (uint32_t)a.block_size;
        slot = (int)(key - p * a.block_size);
        page = s.vis > 0 ? a.bt[seq * a.bt_ss + p] : 0;
    };
    auto resolve = [&]() {
        const uint32_t p = (uint32_t)page < (uint64_t)a.num_blocks ? page : 0;
        k_row = p * a.k_sb + (uint32_t)slot * a.k_ss;
        v_row = p * a.v_sb + (uint32_t)slot * a.v_ss;
    };
    auto row_of = [&](const uint16_t *base, uint32_t row, int at) {  // at: four times the lane that has the row
        return base + 8 * (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)row);
    };
    u32x4 kr[2][kSteps];
    VRow vr[2][4][kVParts];
    const uint16_t *const k_base = a.k + h * a.k_sh, *const v_base = a.v + h * a.v_sh;
    auto fetch_k = [&]() {
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
            const uint16_t *row = row_of(k_base, k_row, 4 * col + 64 * gr) + 8 * g;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) kr[gr][k] = kv16_load<u32x4>(row + (FULL || 32 * k + 8 * g < D ? 32 * k : -8 * g));
        }
    };
    auto fetch_v = [&]() {  // (dims past D: any, not used)
        const int d = FULL || kVDims * col < D ? kVDims * col : 0;
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t *row = row_of(v_base, v_row, 16 * g + 64 * gr + 4 * i) + d;
                vr[gr][i][0] = kv16_load<VRow>(row);
                if constexpr (kVParts == 2) vr[gr][i][1] = kv16_load<VRow>(row + (FULL || 128 + 8 * col < D ? 128 : 0));
            }
    };
    const int n = (t1 - t0 - wave + W - 1) / W;  // tiles of this wave (0 or less: none)
    if (n > 0) {
        look_up(0);
        resolve();
        look_up(1);
    }
    u32x4 qop[NB][kSteps];
    float m_run[NB], l_run[NB];
    int lim[NB], token[NB];  // keys that this lane's column sees, its token
    f32x4 acc[NB][kBlocks];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const uint32_t c = c0 + kShareCols * nb + col, i = c / (uint32_t)a.G;
        const bool valid = (int)i < s.T;
        const uint16_t *row = static_cast<const uint16_t *>(a.q) + (int64_t)(s.q0 + (valid ? (int)i : 0)) * a.q_st +
                              (int64_t)(h * a.G + (valid ? (int)(c - i * a.G) : 0)) * a.q_sh + 8 * g;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
            qop[nb][k] = valid && (FULL || 32 * k + 8 * g < D) ? *reinterpret_cast<const u32x4 *>(row + 32 * k) : u32x4{0u, 0u, 0u, 0u};
        token[nb] = (int)i;
        lim[nb] = a.causal ? min(s.vis, s.pos + (int)i + 1) : s.vis;
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) acc[nb][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        m_run[nb] = -INFINITY, l_run[nb] = 0.f;
    }
    uint32_t big = 0;  // the largest magnitude in V, as integers by halves
    const int lim_first = a.causal ? min(s.vis, s.pos + c0 / a.G + 1) : s.vis;  // the fewest that any column sees
    if (n > 0) {
        fetch_k();
        fetch_v();
    }
    // Product m's operand from V's rows.
    auto v_op = [&](int m) {
        u32x4 o;
        const int p = kVParts == 2 ? m >> 3 : 0, d = m % kVDims;
        const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = perm(vr[x >> 1][2 * (x & 1) + 1][p][d >> 1], vr[x >> 1][2 * (x & 1)][p][d >> 1], sel);
        return o;
    };

#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        const int k0 = (t0 + wave + W * j) * kShareTile;
        f32x4 S[NB][2];
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) S[nb][gr] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                // (what was loaded in the place of dims past D may be infinite, and 0 * infinity is a NaN)
                const u32x4 x = FULL || 32 * k + 8 * g < D ? kr[gr][k] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) S[nb][gr] = mfma_qk<DT>(x, qop[nb][k], S[nb][gr]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (the next rows go where these are)
        resolve();
        look_up(j + 2);
        fetch_k();
        const bool masked = k0 + kShareTile > lim_first;
        uint32_t part_of[NB][kParts][4], one[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float tmax = -INFINITY;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                S[nb][gr] *= a.scale;
                if (masked) {
                    const int left = lim[nb] - k0 - 4 * g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[nb][gr][i] = 16 * gr + i < left ? S[nb][gr][i] : -INFINITY;
                }
                tmax = fmaxf(tmax, fmaxf(fmaxf(S[nb][gr][0], S[nb][gr][1]), fmaxf(S[nb][gr][2], S[nb][gr][3])));
            }
            if (__any(tmax > m_run[nb])) {
                const float m_new = fmaxf(m_run[nb], rows_max(tmax));
                const float alpha = m_new == -INFINITY ? 1.f : FAR ? attn_shrink(m_run[nb] - m_new) : __builtin_amdgcn_exp2f(m_run[nb] - m_new);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) acc[nb][m] *= alpha;
                l_run[nb] *= alpha;
                m_run[nb] = m_new;
            }
            const float top = m_run[nb] == -INFINITY ? 0.f : m_run[nb];
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(S[nb][gr][i] - top) * kPeak;
                l_run[nb] += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w0 = w[2 * x], w1 = w[2 * x + 1];
#pragma unroll
                    for (int n = 0; n < kParts; ++n) {
                        const uint32_t p = part_of[nb][n][2 * gr + x] = pack_pair<DT>(w0, w1);
                        w0 -= Elem<DT>::to_f32(p & 0xffffu), w1 -= Elem<DT>::to_f32(p >> 16);
                    }
                    if constexpr (FAR) {
                        constexpr uint32_t kOne = DT == RQ_DTYPE_BF16 ? 0x3f80u : 0x3c00u;
                        one[nb][2 * gr + x] = (S[nb][gr][2 * x] == -INFINITY ? 0u : kOne) | (S[nb][gr][2 * x + 1] == -INFINITY ? 0u : kOne << 16);
                    }
                }
            }
        }
        auto operand = [](const uint32_t (&w)[4]) { return u32x4{w[0], w[1], w[2], w[3]}; };
        if constexpr (!FAR) {
#pragma unroll
            for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int p = 0; p < kVParts; ++p)
#pragma unroll
                        for (int x = 0; x < (DP == 64 ? 2 : 4); ++x) big = larger16(big, vr[gr][i][p][x]);
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const u32x4 x = v_op(m);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int n = 0; n < kParts; ++n) acc[nb][m] = mfma_qk<DT>(x, operand(part_of[nb][n]), acc[nb][m]);
            }
        } else {
            const int i1 = min(s.T - 1, (c0 + NB * kShareCols - 1) / a.G);
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                const u32x4 v = v_op(m);
#pragma unroll 1
                for (int i = c0 / a.G; i <= i1; ++i) {
                    const int end = (a.causal ? min(s.vis, s.pos + i + 1) : s.vis) - k0 - 4 * g;
                    u32x4 x, y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int left = end - (16 * (e >> 1) + 2 * (e & 1));
                        const uint32_t seen = v[e] & (left >= 2 ? ~0u : left == 1 ? 0xffffu : 0u), far = huge_halves<DT>(seen);
                        x[e] = seen & ~far, y[e] = seen & far;
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        f32x4 o = mfma_qk<DT>(y, operand(one[nb]), acc[nb][m]);
#pragma unroll
                        for (int n = 0; n < kParts; ++n) o = mfma_qk<DT>(x, operand(part_of[nb][n]), o);
                        if (token[nb] == i) acc[nb][m] = o;
                    }
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        fetch_v();
    }

    if constexpr (!FAR) {
        const bool far = (big & 0xffffu) >= kHuge<DT> || big >> 16 >= kHuge<DT>;
        if (HEADS ? __any(far) : __syncthreads_or(far)) {
            kv16_segment<DT, DP, FULL, NB, W, HEADS, true>(a, seq, s, h, c0, t0, t1, part, lds);
            return;
        }
    }
    if constexpr (HEADS) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float l = rows_sum(l_run[nb]);
            if (token[nb] >= s.T) continue;
            const uint32_t cc = c0 + kShareCols * nb + col;
            const float f = part == nullptr ? attn_inv<true>(a, s, token[nb], l) : 1.f;
            uint16_t *const row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + token[nb]) * a.o_st + (int64_t)(h * a.G + (int)(cc - token[nb] * a.G)) * a.o_sh;
            float *const pt = part + nb * AttnPartial<DP>::kFloats;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int p = 0; p < kVParts; ++p) {
                    const int d0 = 128 * p + kVDims * (4 * g + i);
                    float o[kVDims];
#pragma unroll
                    for (int d = 0; d < kVDims; ++d) o[d] = acc[nb][8 * p + d][i];
                    if (part == nullptr) {
                        attn_put<DT, kVDims>(row + d0, o, f, D - d0);
                    } else {
#pragma unroll
                        for (int d = 0; d < kVDims; d += 4) *reinterpret_cast<float4 *>(pt + col * DP + d0 + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
                    }
                }
            if (part != nullptr && g == 0) *reinterpret_cast<float2 *>(pt + kShareCols * DP + 2 * col) = make_float2(m_run[nb], l);
        }
        return;
    }
    // the waves' sums
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float l_col = rows_sum(l_run[nb]);
        __syncthreads();  // (the sums before these are read)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < kVParts; ++p)
#pragma unroll
                for (int d = 0; d < kVDims; d += 4)
                    *reinterpret_cast<f32x4 *>(&lds.acc[wave][col][128 * p + kVDims * (4 * g + i) + d]) =
                        f32x4{acc[nb][8 * p + d][i], acc[nb][8 * p + d + 1][i], acc[nb][8 * p + d + 2][i], acc[nb][8 * p + d + 3][i]};
        if (g == 0) lds.ml[wave][col] = make_float2(m_run[nb], l_col);
        __syncthreads();
        attn_join<DT, DP, W, true>(a, s, h, c0 + kShareCols * nb, D, part == nullptr ? nullptr : part + nb * AttnPartial<DP>::kFloats, lds);
    }
}

// ---- shares -------------------------------------------------------------------
// The tiles of all (sequence, block of columns) pairs in a row are cut into equal shares, and a share is taken by one workgroup for each kv
// head: the heads of a token lie together in memory, and are read at about the same time.
template <int NB>
__device__ __forceinline__ int64_t kv16_seq_tiles(const Kv16Args &a, int64_t b, AttnSeq &s) {
    if (b >= a.num_seqs) return 0;
    s = attn_seq(a, b);
    return (int64_t)attn_tiles(s) * attn_col_blocks<NB>(a, s.T);
}
__device__ __forceinline__ AttnSeq seq_of_lane(const AttnSeq &s, int lane) {  // (in SGPRs)
    return {__builtin_amdgcn_readlane(s.q0, lane), __builtin_amdgcn_readlane(s.T, lane), __builtin_amdgcn_readlane(s.pos, lane),
            __builtin_amdgcn_readlane(s.vis, lane)};
}
// Place of share w's part of an item in the workspace: an item cut in two or more is the last of the share that begins it and the first of the others.
template <int DP, int NB>
__device__ __forceinline__ float *kv16_part(const Kv16Args &a, int64_t w, bool begins, int h) {
    return a.part + ((2 * w + (begins ? 1 : 0)) * a.H + h) * (NB * AttnPartial<DP>::kFloats);
}

// Tiles of a share, at least: a wave of the four has one.  One sequence of 2000 keys with 2 / 4 / 8: 11.0 / 10.6 / 12.0 us, of 4000 13.7 / 11.9 / 12.8.
constexpr int kKv16MinChunk = 4;
__device__ __forceinline__ int64_t kv16_share(int64_t tiles, int shares) {
    return max((int64_t)kKv16MinChunk, div64(tiles + shares - 1, shares));
}

// Workgroups of a CU at once (4 waves each): as many as their registers allow.  Heads of 64 would fit three where they have one block of columns,
// and are slower: 64 sequences of 1024 to 8192 keys 107 us for 105, 16 of 1024 17.2 for 14.3.
template <int DP, int NB>
constexpr int kKv16Resident = DP == 256 ? 1 : 2;

// Bound by memory in long calls: 64 sequences of 1024 to 8192 keys, 8 heads x 4 of 128, 1.2 GB in 187 to 191 us, 6.3 TB/s (HEADS).
template <int DT, int DP, bool FULL, int NB, bool HEADS>
__global__ __launch_bounds__(256, (kKv16Resident<DP, NB>)) void kv16_stream_kernel(Kv16Args a) {
    constexpr int kHeads = HEADS ? 4 : 1;  // of a workgroup
    __shared__ AttnSums<DP, HEADS ? 1 : 4> lds;
    auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };  // (what is the workgroup's, into SGPRs)
    const int lane = threadIdx.x & 63, hs = a.H / kHeads, shares = gridDim.x / (uint32_t)hs, w = blockIdx.x / (uint32_t)hs,
              h = (blockIdx.x - w * hs) * kHeads + (HEADS ? scalar(threadIdx.x >> 6) : 0);
    int64_t block = 0, block_base = 0;  // 64 sequences: a lane's, its tiles, and the row's up to it
    AttnSeq own{}, other{};
    int64_t mine = kv16_seq_tiles<NB>(a, lane, own), upto = wave_scan64(mine);
    int64_t total = lane64(upto, 63);
    for (int64_t b = 64; b < a.num_seqs; b += 64) total += lane64(wave_scan64(kv16_seq_tiles<NB>(a, b + lane, other)), 63);
    const int64_t share = kv16_share(total, shares);
    int64_t pos = w * share;
    const int64_t end = min(total, pos + share);
    while (pos < end) {
        uint64_t hit = __ballot(block_base + upto > pos);
        while (hit == 0) {
            block_base += lane64(upto, 63);
            block += 64;
            mine = kv16_seq_tiles<NB>(a, block + lane, own);
            upto = wave_scan64(mine);
            hit = __ballot(block_base + upto > pos);
        }
        const int of = __builtin_ctzll(hit);
        const int64_t seq = block + of, in_seq = pos - (block_base + lane64(upto, of) - lane64(mine, of));
        const AttnSeq s = seq_of_lane(own, of);
        const int n = attn_tiles(s), cols = scalar((int)div64(in_seq, n));
        const int t0 = scalar((int)(in_seq - (int64_t)cols * n)), t1 = scalar((int)min((int64_t)n, t0 + (end - pos)));
        float *part = t0 == 0 && t1 == n ? nullptr : kv16_part<DP, NB>(a, w, t0 == 0, h);
        kv16_segment<DT, DP, FULL, NB, HEADS ? 1 : 4, HEADS>(a, scalar((int)seq), s, h, cols * (NB * kShareCols), t0, t1, part, lds);
        pos += t1 - t0;
    }
}

// Adds up the parts of the items that were cut: `per` workgroups for a sequence and head.  A wave takes a column at a time; lane: D / 16 dims, and every
// fourth part, four of them on their way.  4 to 6 us, mostly its launch; 11 for 32 drafts of 8 tokens (38 MB of parts).
template <int DT, int DP, int NB>
__global__ __launch_bounds__(256) void kv16_merge_kernel(Kv16Args a, int shares, int per) {
    constexpr int kDims = DP / 16, kAhead = DP == 256 ? 2 : 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, way = lane >> 4, d0 = (lane & 15) * kDims;
    const int64_t b = blockIdx.y;
    const int h = blockIdx.x % (uint32_t)a.H;
    int64_t total = 0, before = 0;
    AttnSeq s{}, own{};
    for (int64_t b0 = 0; b0 < a.num_seqs; b0 += 64) {
        const int64_t mine = kv16_seq_tiles<NB>(a, b0 + lane, own), upto = wave_scan64(mine);
        if (b >= b0 && b < b0 + 64) {
            before = total + lane64(upto, (int)(b - b0)) - lane64(mine, (int)(b - b0));
            s = seq_of_lane(own, (int)(b - b0));
        }
        total += lane64(upto, 63);
    }
    const int n = attn_tiles(s);
    const int64_t share = kv16_share(total, shares);
    for (int cc = blockIdx.x / (uint32_t)a.H * 4 + wave; cc < s.T * a.G; cc += 4 * per) {  // (the column, of all blocks')
        const int nb = cc / kShareCols % NB, c = cc % kShareCols;
        const int64_t first = before + (int64_t)(cc / (NB * kShareCols)) * n;
        const int w0 = (int)div64(first, share), w1 = (int)div64(first + n - 1, share);
        if (w0 == w1) continue;
        float M = -INFINITY, l = 0.f, o[kDims] = {};
        for (int w = w0 + way; w <= w1; w += 4 * kAhead) {
            float2 ml[kAhead];
            float4 x[kAhead][kDims / 4];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int wu = min(w + 4 * u, w1);
                const float *pt = kv16_part<DP, NB>(a, wu, wu == w0, h) + nb * AttnPartial<DP>::kFloats;
                ml[u] = *reinterpret_cast<const float2 *>(pt + kShareCols * DP + 2 * c);
#pragma unroll
                for (int k = 0; k < kDims / 4; ++k) x[u][k] = *reinterpret_cast<const float4 *>(pt + c * DP + d0 + 4 * k);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (w + 4 * u > w1) continue;
                const float Mn = fmaxf(M, ml[u].x);
                const float keep = M == -INFINITY ? (Mn == -INFINITY ? 1.f : 0.f) : attn_shrink(M - Mn);
                const float r = ml[u].x == -INFINITY ? (Mn == -INFINITY ? 1.f : 0.f) : attn_shrink(ml[u].x - Mn);
                M = Mn;
                l = l * keep + r * ml[u].y;
#pragma unroll
                for (int k = 0; k < kDims / 4; ++k) {
                    o[4 * k] = o[4 * k] * keep + r * x[u][k].x, o[4 * k + 1] = o[4 * k + 1] * keep + r * x[u][k].y;
                    o[4 * k + 2] = o[4 * k + 2] * keep + r * x[u][k].z, o[4 * k + 3] = o[4 * k + 3] * keep + r * x[u][k].w;
                }
            }
        }
        const float Mt = rows_max(M), r = M == -INFINITY ? (Mt == -INFINITY ? 1.f : 0.f) : attn_shrink(M - Mt);
        l = rows_sum(l * r);
#pragma unroll
        for (int k = 0; k < kDims; ++k) o[k] = rows_sum(o[k] * r);
        if (way != 0) continue;
        const int i = cc / a.G;
        uint16_t *row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + i) * a.o_st + (int64_t)(h * a.G + cc % a.G) * a.o_sh + d0;
        attn_put<DT, kDims>(row, o, attn_inv<true>(a, s, i, l), a.D - d0);
    }
}

// One workgroup per item: one launch, no partials.  Four waves: with eight, which join twice the sums, 64 sequences of 256 keys take 20.1 us for
// 16.1, one of 256 7.5 for 7.0; with two 16.6 and 7.9.
constexpr int kKv16ItemWaves = 4;
template <int DT, int DP, bool FULL, int NB>
__global__ __launch_bounds__(64 * kKv16ItemWaves, DP == 256 ? 1 : 2) void kv16_item_kernel(Kv16Args a) {
    __shared__ AttnSums<DP, kKv16ItemWaves> lds;
    const int64_t seq = blockIdx.y;
    const AttnSeq s = attn_seq(a, seq);
    const int block = blockIdx.x / (uint32_t)a.H, h = blockIdx.x - block * a.H;
    if (block >= attn_col_blocks<NB>(a, s.T)) return;
    kv16_segment<DT, DP, FULL, NB, kKv16ItemWaves, false>(a, seq, s, h, block * (NB * kShareCols), 0, attn_tiles(s), nullptr, lds);
}

// Whether a head's rows span less than 2^32 units of 8 elements.
static bool kv16_span(int64_t num_blocks, int64_t block_size, int64_t stride_block, int64_t stride_slot) {
    return ((double)(num_blocks - 1) * (double)stride_block + (double)(block_size - 1) * (double)stride_slot) / 8 < 4294967295.0;
}

static int kv16_blocks(int G, int64_t max_q_len) { return max_q_len * G > kShareCols ? 2 : 1; }
static int kv16_width(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
// How a call is cut, by its bounds.
// Short contexts: a workgroup per item (shares 0), one launch and no parts.  One CU loads 55 to 60 GB/s, and lengths differ, so long ones are slower:
// up to 16 tiles; where half the CUs or more get an item, which costs shares their parts and cuts, 24, or 64 with two blocks of columns (whose
// parts are twice as large).  8 heads x 4 of 128, items / shares, us:
//   single tokens, 1 sequence of 256 keys 7.0 / 9.9, 512: 9.5 / 9.9, 777: 12.6 / 10.0; 32 of 600: 18.1 / 24.8, of 50 to 600 15.8 / 19.0, of 1024
//   27.4 / 31.0, of 50 to 1400 30.5 / 28.7; 128 of 50 to 600 44 / 48, of 50 to 777 55 / 50; heads of 64, 64 of 600 21 / 23; 4 heads x 8 of 256, 64 of
//   50 to 777 32 / 37, to 1400 50 / 48;
//   8 tokens each, 1 of 1024 21 / 14, 16 of 1400 32 / 39, 64 of 2000 102 / 134, of 50 to 2000 79 / 94; 4 heads x 8 of 256, 4 tokens, 64 of 50 to 2000
//   77 / 114.
// Longer ones: shares of tiles, each taken by H / heads workgroups.  heads 4 (a wave each) where that leaves a wave 12 tiles or more, else 1 (the
// waves share the tiles, and their sums): the former reads 1 KB of a token at about the same time, but its parts are four times as many.  8 heads x
// 4 of 128, us by waves / by tiles: 64 sequences of 1024 to 8192 keys 196 / 221, of 2000 93.5 / 97.4, 16 of 2000 (4 tiles a wave) 32.9 / 33.1, 1 of
// 4000 16.9 / 12.9; 4 heads x 7, 4 sequences of 20000 to 32768 (8 tiles a wave) 59.7 / 54.5.  8 tokens, 32 of 600 to 8000: 134 / 146.  Two blocks of
// columns of 256 fill the registers, and a wave's with a head of its own do not hold them: 4 heads x 8, 4 tokens, 64 of 4000 keys 293 / 222.
constexpr bool kv16_by_heads(int width, int blocks) { return width < 256 || blocks == 1; }
struct Kv16Cut {
    int heads;
    int64_t shares;
};
static Kv16Cut kv16_cut(int64_t num_seqs, int G, int H, int D, int64_t max_q_len, int64_t max_keys) {
    const int w = kv16_width(D), blocks = kv16_blocks(G, max_q_len), cols = blocks * kShareCols;
    const int64_t cus = device_cus(), resident = (w == 64 ? kKv16Resident<64, 1> : w == 128 ? kKv16Resident<128, 1> : kKv16Resident<256, 1>) * cus;
    const int64_t tiles = max_keys / kShareTile + (max_keys % kShareTile != 0 || max_keys == 0);
    const int64_t rows = num_seqs * ((max_q_len * G + cols - 1) / cols), work = rows * tiles;
    if (tiles <= (2 * rows * H < cus ? 16 : blocks == 1 ? 24 : 64)) return {1, 0};
    const int heads = kv16_by_heads(w, blocks) && H % 4 == 0 && work * (H / 4) >= 12 * resident ? 4 : 1;
    return {heads, std::max<int64_t>(1, std::min<int64_t>(resident * heads / H, (work + kKv16MinChunk - 1) / kKv16MinChunk))};
}

template <int DT, int DP, bool FULL, int NB>
static void launch_kv16(const Kv16Args &a, const Kv16Cut &cut, hipStream_t st) {
    const int64_t items = ((int64_t)a.max_q * a.G + NB * kShareCols - 1) / (NB * kShareCols) * a.H;
    if (cut.shares == 0) {
        hipLaunchKernelGGL((kv16_item_kernel<DT, DP, FULL, NB>), dim3((unsigned)items, (unsigned)a.num_seqs), dim3(64 * kKv16ItemWaves), 0, st, a);
        return;
    }
    // (enough workgroups for the parts of few items, and no more than one each where there are many)
    const int64_t quads = ((int64_t)a.max_q * a.G + 3) / 4, per = std::max<int64_t>(1, std::min<int64_t>(quads, 512 / std::max<int64_t>(1, a.num_seqs * a.H)));
    const dim3 grid((unsigned)(cut.shares * (a.H / cut.heads)));
    constexpr bool kHeads = kv16_by_heads(DP, NB);
    if (kHeads && cut.heads == 4) hipLaunchKernelGGL((kv16_stream_kernel<DT, DP, FULL, NB, kHeads>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv16_stream_kernel<DT, DP, FULL, NB, false>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((kv16_merge_kernel<DT, DP, NB>), dim3((unsigned)(per * a.H), (unsigned)a.num_seqs), dim3(256), 0, st, a, (int)cut.shares, (int)per);
}
template <int DT, int DP, bool FULL>
static void launch_kv16_b(const Kv16Args &a, const Kv16Cut &cut, hipStream_t st) {
    kv16_blocks(a.G, a.max_q) == 1 ? launch_kv16<DT, DP, FULL, 1>(a, cut, st) : launch_kv16<DT, DP, FULL, 2>(a, cut, st);
}
template <int DT, int DP>
static void launch_kv16_f(const Kv16Args &a, const Kv16Cut &cut, hipStream_t st) {
    a.D == DP ? launch_kv16_b<DT, DP, true>(a, cut, st) : launch_kv16_b<DT, DP, false>(a, cut, st);
}
template <int DT>
static void launch_kv16_d(const Kv16Args &a, const Kv16Cut &cut, hipStream_t st) {
    const int w = kv16_width(a.D);
    w == 64 ? launch_kv16_f<DT, 64>(a, cut, st) : w == 128 ? launch_kv16_f<DT, 128>(a, cut, st) : launch_kv16_f<DT, 256>(a, cut, st);
}

}  // namespace rq

using namespace rq;

extern "C" int64_t rq_kv16_attention_workspace_bytes(int64_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                                     int64_t max_q_len, int64_t max_seq_len) {
    if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0 || head_dim > 256 || max_q_len <= 0 || max_seq_len < 0)
        return 0;
    const int G = num_q_heads / num_kv_heads;
    return 2 * kv16_cut(num_seqs, G, num_kv_heads, head_dim, max_q_len, attn_bound(max_seq_len)).shares * num_kv_heads * kv16_blocks(G, max_q_len) * kShareCols * (kv16_width(head_dim) + 2) * 4;
}

extern "C" int rq_kv16_attention(const void *q, int32_t dtype, int64_t total_q, int32_t num_q_heads, int64_t q_stride_tok, int64_t q_stride_head,
                                 const int32_t *cu_seqlens_q, int64_t num_seqs, int64_t max_q_len, int32_t causal, const void *k_cache,
                                 const void *v_cache, int64_t num_blocks, int32_t block_size, int64_t kc_stride_block, int64_t kc_stride_slot,
                                 int64_t kc_stride_head, int64_t vc_stride_block, int64_t vc_stride_slot, int64_t vc_stride_head,
                                 int32_t num_kv_heads, int32_t head_dim, const int32_t *block_table, int64_t max_blocks, int64_t bt_stride_seq,
                                 const int32_t *seq_lens, int64_t max_seq_len, float sm_scale, void *out, int64_t out_stride_tok,
                                 int64_t out_stride_head, void *workspace, int64_t workspace_bytes, void *stream) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_BF16 || dtype == RQ_DTYPE_F16, "q and the pages must be f16 or bf16");
    RQ_CHECK_ARG(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, "head_dim %d must be a multiple of 8 up to 256", head_dim);
    RQ_CHECK_ARG(num_kv_heads >= 1 && num_kv_heads <= 4096, "num_kv_heads %d unsupported", num_kv_heads);
    RQ_CHECK_ARG(num_q_heads >= 1 && num_q_heads <= 65536 && num_q_heads % num_kv_heads == 0,
                 "num_q_heads %d must be a multiple of num_kv_heads %d", num_q_heads, num_kv_heads);
    RQ_CHECK_ARG(block_size >= 1 && block_size <= 65536 && num_blocks >= 0 && num_blocks <= INT32_MAX, "bad cache sizes");
    RQ_CHECK_ARG(num_seqs >= 0 && num_seqs <= 65535 && total_q >= 0 && total_q <= INT32_MAX && max_q_len >= 0 && max_q_len <= (1 << 20) &&
                     max_blocks >= 0 && max_seq_len >= 0, "bad sizes");
    RQ_CHECK_ARG(max_q_len * num_q_heads <= (1 << 27), "max_q_len %lld with %d query heads: more rows of a sequence than a launch takes",
                 (long long)max_q_len, num_q_heads);
    RQ_CHECK_ARG(cu_seqlens_q != nullptr || (total_q == num_seqs && max_q_len <= 1),
                 "without cu_seqlens_q there is one query token per sequence");
    RQ_CHECK_ARG(__builtin_fabsf(sm_scale) <= 0x1p127f, "sm_scale must be finite, 2^127 at most");  // (times log2(e) it is finite)
    if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return RQ_OK;
    RQ_CHECK_ARG(num_blocks > 0, "the cache has no pages");
    RQ_CHECK_ARG(q && out && k_cache && v_cache && seq_lens && (block_table || max_blocks == 0), "null pointer");
    RQ_CHECK_ARG((uintptr_t)q % 16 == 0 && q_stride_tok % 8 == 0 && q_stride_head % 8 == 0, "q rows must be 16-byte aligned");
    RQ_CHECK_ARG((uintptr_t)out % 8 == 0 && out_stride_tok % 4 == 0 && out_stride_head % 4 == 0, "out rows must be 8-byte aligned");
    RQ_CHECK_ARG(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && kc_stride_block % 8 == 0 && kc_stride_slot % 8 == 0 && kc_stride_head % 8 == 0 &&
                     vc_stride_block % 8 == 0 && vc_stride_slot % 8 == 0 && vc_stride_head % 8 == 0, "cache rows must be 16-byte aligned");
    RQ_CHECK_ARG(kc_stride_block >= 0 && kc_stride_slot >= 0 && vc_stride_block >= 0 && vc_stride_slot >= 0 &&
                     kv16_span(num_blocks, block_size, kc_stride_block, kc_stride_slot) && kv16_span(num_blocks, block_size, vc_stride_block, vc_stride_slot),
                 "a head's rows must lie within 64 GiB, each side, in ascending order");
    Kv16Args a{};
    a.q = q, a.q_st = q_stride_tok, a.q_sh = q_stride_head;
    a.cu_q = cu_seqlens_q;
    a.total_q = total_q, a.num_seqs = num_seqs;
    a.causal = causal != 0;
    a.k = static_cast<const uint16_t *>(k_cache), a.k_sb = (uint32_t)(kc_stride_block / 8), a.k_ss = (uint32_t)(kc_stride_slot / 8), a.k_sh = kc_stride_head;
    a.v = static_cast<const uint16_t *>(v_cache), a.v_sb = (uint32_t)(vc_stride_block / 8), a.v_ss = (uint32_t)(vc_stride_slot / 8), a.v_sh = vc_stride_head;
    a.num_blocks = num_blocks;
    a.H = num_kv_heads, a.G = num_q_heads / num_kv_heads, a.block_size = block_size, a.D = head_dim;
    a.bt = block_table, a.max_blocks = max_blocks, a.bt_ss = bt_stride_seq;
    a.seq_lens = seq_lens;
    a.bound = attn_bound(max_seq_len);
    a.cap = std::min<int64_t>(a.bound, max_blocks > a.bound / block_size ? a.bound : max_blocks * block_size);
    a.max_q = (int)max_q_len;
    a.scale = sm_scale * kAttnLog2e;
    a.out = out, a.o_st = out_stride_tok, a.o_sh = out_stride_head;
    const int64_t need = rq_kv16_attention_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len, max_seq_len);
    RQ_CHECK_SPACE(workspace_bytes >= need, "workspace too small: the call needs %lld bytes (got %lld)", (long long)need, (long long)workspace_bytes);
    RQ_CHECK_ARG(need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "workspace must be 16-byte aligned");
    a.part = static_cast<float *>(workspace);
    hipStream_t st = (hipStream_t)stream;
    const Kv16Cut cut = kv16_cut(num_seqs, a.G, a.H, head_dim, a.max_q, a.bound);
    if (dtype == RQ_DTYPE_BF16) launch_kv16_d<RQ_DTYPE_BF16>(a, cut, st);
    else launch_kv16_d<RQ_DTYPE_F16>(a, cut, st);
    return check_launch("kv16_stream_kernel");
}
