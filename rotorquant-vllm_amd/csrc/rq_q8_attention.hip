// Attention over the 8-bit KV cache (rq_q8_attention; format in rq_q8.h): queries of one or a few
// tokens, bound by the stream of codes from HBM.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(sm_scale q_i . k_j) over the keys j that i may see.
//
// Columns are the (token, query head) pairs that share a kv head, 16 to an MFMA.  Per group of 16 keys:
//   S^T = K Q^T   on v_mfma_f32_16x16x32_f16: codes c_k (exact in fp16) times q 2^s (s per column, the row's
//                 largest magnitude near 2^14: fp16 holds what bf16 does), fp32 sums;
//   u = S f + e_v, f = |sm_scale| log2(e) 2^(e_k - s): the score in base 2 plus the V exponent;
//   w = 2^(u - M) in fp16, M a column's running maximum of u (rescaled lazily: w stays under 2^8);
//   O^T += C_v^T w  (codes again exact), l += 2^-e_v sum w.
// So a group's two scales cost one multiplication per column and an addend that the exponent takes anyway, the
// weights are relative to the largest p 2^e_v whatever the groups' scales are, and out = O / l.
// l stays in fp32 whatever the scales: a token whose w underflows has under 2^-26 of the sum of p of the
// one that sets M (e_v is in -40 .. 60).
//
// Operands need neither LDS nor shuffles: a lane's 16 bytes of K and V are its operands' elements (rq_q8.h), and
// the weights come out of S^T in the order that P V takes.
#include <algorithm>

#include "rq_q8_attn.h"

namespace rq {

constexpr int kQ8Waves = 4;     // of a workgroup; tile t of a segment goes to wave t % 4
constexpr int kQ8Cols = 16;     // columns of a workgroup
constexpr int kQ8MinChunk = 8;  // tiles of a workgroup, at least

__device__ __forceinline__ int q8_col_blocks(const Q8AttnArgs &a, int T) { return (T * a.G + kQ8Cols - 1) / kQ8Cols; }

constexpr int kQ8Tile = 32;     // keys of a tile: two groups
__device__ __forceinline__ int q8_tiles(const Q8Seq &s) { return max(1, (s.vis + kQ8Tile - 1) / kQ8Tile); }

// Items are (sequence, block of 16 columns, kv head), in that order; the tiles of all items in a row are cut into
// equal shares.  Tiles of all items, in 64-bit; each workgroup sums over the sequences itself (64 at a time).
__device__ __forceinline__ int64_t q8_seq_tiles(const Q8AttnArgs &a, int64_t b) {
    if (b >= a.num_seqs) return 0;
    const Q8Seq s = q8_seq(a, b);
    return (int64_t)q8_tiles(s) * q8_col_blocks(a, s.T) * a.H;
}
__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ int64_t wave_scan64(int64_t x, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}
__device__ __forceinline__ int64_t q8_share(int64_t tiles, int64_t workgroups) {
    return max((int64_t)kQ8MinChunk, (tiles + workgroups - 1) / workgroups);
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

template <int D>
struct Q8Partial {
    static constexpr int kFloats = kQ8Cols * (D + 2);  // accumulators by column, then (M, l) by column
};

// One column's operands: q 2^s in fp16 in K's dim order, and f without the group's 2^e_k.
template <int DT, int D>
__device__ __forceinline__ float q8_query(const Q8AttnArgs &a, const Q8Seq &s, int c0, int h, int lane, u32x4 (&qop)[D / 32]) {
    const int col = c0 + (lane & 15), g = lane >> 4;
    const int i = col / a.G, hq = h * a.G + col % a.G;
    u32x4 raw[D / 32];
    const bool valid = i < s.T;
    const uint16_t *row = static_cast<const uint16_t *>(a.q) + (int64_t)(s.q0 + (valid ? i : 0)) * a.q_st + (int64_t)(valid ? hq : h * a.G) * a.q_sh;
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
        raw[k] = valid ? *reinterpret_cast<const u32x4 *>(row + 64 * (k >> 1) + 16 * g + 8 * (k & 1)) : u32x4{0u, 0u, 0u, 0u};
        big = q8_max_bits(raw[k], big);
    }
    big = max(big, (uint32_t)__shfl_xor((int)big, 16));
    big = max(big, (uint32_t)__shfl_xor((int)big, 32));
    const int up = q8_query_exp<DT>(big);
    const float f = exp2i(up) * a.q_sign;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) qop[k] = q8_query_f16<DT>(raw[k], f);
    return a.score_scale * exp2i(-up);
}

// Codes and scales of one tile: two groups.
template <int D>
struct Q8Tile {
    u32x4 k[2][D / 64], v[2][D / 64];
    float ks[2], vs[2];
};

template <int DT, int FMT, int D>
__global__ __launch_bounds__(64 * kQ8Waves) void q8_stream_kernel(Q8AttnArgs a) {
    constexpr int kSteps = D / 32, kChunks = D / 64, kBlocks = D / 16;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    __shared__ float lds_acc[kQ8Waves][kQ8Cols][D + 4];
    __shared__ float2 lds_ml[kQ8Waves][kQ8Cols];

    // this workgroup's share [pos, end) of the row of tiles
    int64_t total = 0;
    for (int64_t b = 0; b < a.num_seqs; b += 64) total += wave_sum64(q8_seq_tiles(a, b + lane));
    total = uniform64(total);
    const int64_t share = q8_share(total, gridDim.x);
    int64_t pos = blockIdx.x * share;
    const int64_t end = min(total, pos + share);

    int64_t seq = -1, seq_base = 0, seq_tiles = 0;  // the sequence of pos: its first tile in the row, its tiles
    int64_t scan_b = 0, scan_base = 0;
    while (pos < end) {
        if (seq < 0 || pos >= seq_base + seq_tiles) {
            for (;; scan_b += 64) {
                const int64_t mine = q8_seq_tiles(a, scan_b + lane), upto = wave_scan64(mine, lane);
                const uint64_t hit = __ballot(scan_base + upto > pos);
                if (hit) {
                    const int l = __builtin_ctzll(hit);
                    seq = scan_b + l;
                    seq_tiles = uniform64(__shfl(mine, l));
                    seq_base = uniform64(scan_base + __shfl(upto, l)) - seq_tiles;
                    break;
                }
                scan_base = uniform64(scan_base + __shfl(upto, 63));
            }
        }
        const Q8Seq s = q8_seq(a, seq);
        const int n = q8_tiles(s);
        const int64_t in_seq = pos - seq_base;
        const int64_t item = in_seq / n;
        const int t0 = (int)(in_seq - item * n), t1 = (int)min((int64_t)n, t0 + (end - pos));
        const int h = (int)(item % a.H), c0 = (int)(item / a.H) * kQ8Cols;

        u32x4 qop[kSteps];
        const float colf = q8_query<DT, D>(a, s, c0, h, lane, qop);
        // keys that this lane's column sees, and the fewest that any column of the block sees
        const int i_mine = (c0 + col) / a.G, i_first = c0 / a.G;
        const int lim = a.causal ? min(s.vis, s.L - s.T + i_mine + 1) : s.vis;
        const int lim_first = a.causal ? min(s.vis, s.L - s.T + i_first + 1) : s.vis;

        f32x4 acc[kBlocks];
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
        float M = -INFINITY, l_run = 0.f;

        const Q8Layout lay(a.H, D, a.block_size);
        // tiles of this wave: t0 + wave, + 4, ...; lane l looks up group l % 2 of the (l / 2)-th of the next 32
        const int last_group = max(0, (s.vis + kQ8Group - 1) / kQ8Group - 1);
        int64_t at = 0;
        float2 sc = make_float2(0.f, 0.f);
        auto look_up = [&](int first) {
            const int gi = min(2 * (first + kQ8Waves * (lane >> 1)) + (lane & 1), last_group);
            const int p = gi / a.groups;
            int64_t page = s.vis > 0 ? a.bt[seq * a.bt_ss + p] : 0;
            page = page < 0 || page >= a.num_blocks ? 0 : page;
            at = page * a.stride_block + lay.codes_at(gi - p * a.groups, h);
            sc = *reinterpret_cast<const float2 *>(a.cache + page * a.stride_block + lay.scale_at(gi - p * a.groups, h));
        };
        Q8Tile<D> next;
        auto fetch = [&](int t) {  // tile t of the segment, slot (t - t0) / 4 % 32 of the looked-up ones
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const int from = 2 * (((t - t0) / kQ8Waves) & 31) + gr;
                const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at, from), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)at >> 32), from);
                const uint8_t *p = a.cache + ((uint64_t)hi << 32 | lo);
                next.ks[gr] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.x), from));
                next.vs[gr] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sc.y), from));
#pragma unroll
                for (int j = 0; j < kChunks; ++j) {
                    next.k[gr][j] = *reinterpret_cast<const u32x4 *>(p + 1024 * j + 16 * lane);
                    next.v[gr][j] = *reinterpret_cast<const u32x4 *>(p + kQ8Group * D + 1024 * j + 16 * lane);
                }
            }
        };
        int t = t0 + wave;
        if (t < t1) {
            look_up(t);
            fetch(t);
        }
        for (; t < t1; t += kQ8Waves) {
            Q8Tile<D> cur = next;
            const int tn = t + kQ8Waves;
            if (tn < t1) {
                if ((((tn - t0) / kQ8Waves) & 31) == 0) look_up(tn);
                fetch(tn);
            }
            const int k0 = t * kQ8Tile;
            // scores
            f32x4 S[2];
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                S[gr] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    u32x4 op;
                    const u32x4 w = cur.k[gr][k >> 1];
                    uint32_t x[4];
                    q8_to_f16<FMT>(w[2 * (k & 1)], x[0], x[1]);
                    q8_to_f16<FMT>(w[2 * (k & 1) + 1], x[2], x[3]);
                    op = u32x4{x[0], x[1], x[2], x[3]};
                    S[gr] = mfma_f16(op, qop[k], S[gr]);
                }
            }
            if (k0 + kQ8Tile > lim_first) {
#pragma unroll
                for (int gr = 0; gr < 2; ++gr)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[gr][i] = k0 + 16 * gr + 4 * g + i < lim ? S[gr][i] : -INFINITY;
                if (FMT == RQ_Q8_E4M3 && k0 + kQ8Tile > s.vis) {
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
            int ev[2];
            float f[2], tmax = -INFINITY;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                ev[gr] = q8_scale_exp(cur.vs[gr]);
                f[gr] = colf * exp2i(q8_scale_exp(cur.ks[gr]));
                const float m = fmaxf(fmaxf(S[gr][0], S[gr][1]), fmaxf(S[gr][2], S[gr][3]));
                tmax = fmaxf(tmax, __builtin_fmaf(m, f[gr], (float)ev[gr]));
            }
            if (__any(tmax - M > 8.f)) {
                const float m_new = fmaxf(M, rows_max(tmax));
                const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(M - m_new);
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) acc[m] *= alpha;
                l_run *= alpha;
                M = m_new;
            }
            const float bias = M == -INFINITY ? 0.f : -M;
            u32x4 pw;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
                const float add = bias + (float)ev[gr];
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[gr][i], f[gr], add));
                pw[2 * gr] = pack_f16(w[0], w[1]);
                pw[2 * gr + 1] = pack_f16(w[2], w[3]);
                // the sum of the weights before their rounding to fp16 (which has no bias)
                l_run = __builtin_fmaf((w[0] + w[1]) + (w[2] + w[3]), exp2i(-ev[gr]), l_run);
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t x[4];
                    q8_to_f16<FMT>(cur.v[0][j][i], x[0], x[1]);
                    q8_to_f16<FMT>(cur.v[1][j][i], x[2], x[3]);
                    acc[4 * j + i] = mfma_f16(u32x4{x[0], x[1], x[2], x[3]}, pw, acc[4 * j + i]);
                }
        }

        // the four waves' sums of this segment
        l_run = rows_sum(l_run);
        __syncthreads();  // (the previous segment's are read)
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) *reinterpret_cast<f32x4 *>(&lds_acc[wave][col][16 * m + 4 * g]) = acc[m];
        if (g == 0) lds_ml[wave][col] = make_float2(M, l_run);
        __syncthreads();
        {
            constexpr int kDims = D / 16;  // dims of a thread
            const int c = tid >> 4, d0 = (tid & 15) * kDims;
            float Mt = -INFINITY, l = 0.f, o[kDims] = {};
#pragma unroll
            for (int w = 0; w < kQ8Waves; ++w) Mt = fmaxf(Mt, lds_ml[w][c].x);
#pragma unroll
            for (int w = 0; w < kQ8Waves; ++w) {
                const float2 ml = lds_ml[w][c];
                const float r = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - Mt);
                l += r * ml.y;
#pragma unroll
                for (int k = 0; k < kDims; ++k) o[k] += r * lds_acc[w][c][d0 + k];
            }
            const int i = (c0 + c) / a.G;
            if (t0 == 0 && t1 == n) {
                const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key: zeros
                if (i < s.T) {
                    uint16_t *row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + i) * a.o_st + (int64_t)(h * a.G + (c0 + c) % a.G) * a.o_sh + d0;
#pragma unroll
                    for (int k = 0; k < kDims; k += 4)
                        *reinterpret_cast<uint2 *>(row + k) = make_uint2(Elem<DT>::from_f32(o[k] * inv) | Elem<DT>::from_f32(o[k + 1] * inv) << 16,
                                                                         Elem<DT>::from_f32(o[k + 2] * inv) | Elem<DT>::from_f32(o[k + 3] * inv) << 16);
                }
            } else {
                // an item cut in two or more: the share that begins it ends with it, the others begin with it
                float *pt = a.part + (2 * (int64_t)blockIdx.x + (t0 == 0 ? 1 : 0)) * Q8Partial<D>::kFloats;
#pragma unroll
                for (int k = 0; k < kDims; k += 4) *reinterpret_cast<float4 *>(pt + c * D + d0 + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                if ((tid & 15) == 0) *reinterpret_cast<float2 *>(pt + kQ8Cols * D + 2 * c) = make_float2(Mt, l);
            }
        }
        pos += t1 - t0;
    }
}

// Adds up the partials of the items that were cut: one workgroup per item, thread (column, part).
template <int DT, int D>
__global__ __launch_bounds__(256) void q8_merge_kernel(Q8AttnArgs a, int workgroups) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t b = blockIdx.y;
    const Q8Seq s = q8_seq(a, b);
    if ((int64_t)blockIdx.x >= (int64_t)q8_col_blocks(a, s.T) * a.H) return;
    const int n = q8_tiles(s);
    int64_t total = 0, before = 0;
    for (int64_t b0 = 0; b0 < a.num_seqs; b0 += 64) {
        const int64_t mine = q8_seq_tiles(a, b0 + lane);
        total += wave_sum64(mine);
        before += wave_sum64(b0 + lane < b ? mine : 0);
    }
    const int64_t share = q8_share(total, workgroups);
    const int64_t first = before + (int64_t)blockIdx.x * n;
    const int64_t w0 = first / share, w1 = (first + n - 1) / share;
    if (w0 == w1) return;
    constexpr int kDims = D / 16;
    const int h = blockIdx.x % a.H, c0 = (blockIdx.x / a.H) * kQ8Cols;
    const int c = tid >> 4, d0 = (tid & 15) * kDims;
    float M = -INFINITY, l = 0.f, o[kDims] = {};
    for (int64_t w = w0; w <= w1; ++w) {
        const float *pt = a.part + (2 * w + (w == w0 ? 1 : 0)) * Q8Partial<D>::kFloats;
        const float2 ml = *reinterpret_cast<const float2 *>(pt + kQ8Cols * D + 2 * c);
        const float Mn = fmaxf(M, ml.x);
        const float keep = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - Mn);
        const float r = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - Mn);
        M = Mn;
        l = l * keep + r * ml.y;
#pragma unroll
        for (int k = 0; k < kDims; k += 4) {
            const float4 x = *reinterpret_cast<const float4 *>(pt + c * D + d0 + k);
            o[k] = o[k] * keep + r * x.x, o[k + 1] = o[k + 1] * keep + r * x.y;
            o[k + 2] = o[k + 2] * keep + r * x.z, o[k + 3] = o[k + 3] * keep + r * x.w;
        }
    }
    const int i = (c0 + c) / a.G;
    if (i >= s.T) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *row = static_cast<uint16_t *>(a.out) + (int64_t)(s.q0 + i) * a.o_st + (int64_t)(h * a.G + (c0 + c) % a.G) * a.o_sh + d0;
#pragma unroll
    for (int k = 0; k < kDims; k += 4)
        *reinterpret_cast<uint2 *>(row + k) = make_uint2(Elem<DT>::from_f32(o[k] * inv) | Elem<DT>::from_f32(o[k + 1] * inv) << 16,
                                                         Elem<DT>::from_f32(o[k + 2] * inv) | Elem<DT>::from_f32(o[k + 3] * inv) << 16);
}

// Workgroups of the stream kernel: what the GPU holds at once, or fewer where the bound on the lengths gives less work.
static int64_t q8_workgroups(int64_t num_seqs, int G, int H, int64_t max_q_len, int64_t max_keys) {
    const int64_t tiles = std::max<int64_t>(1, (max_keys + kQ8Tile - 1) / kQ8Tile), cols = (max_q_len * G + kQ8Cols - 1) / kQ8Cols;
    const int64_t work = num_seqs * cols * H * tiles;
    return std::max<int64_t>(1, std::min<int64_t>(3 * (int64_t)device_cus(), (work + kQ8MinChunk - 1) / kQ8MinChunk));
}

template <int DT, int FMT, int D>
static void launch_stream(const Q8AttnArgs &a, int64_t workgroups, hipStream_t st) {
    hipLaunchKernelGGL((q8_stream_kernel<DT, FMT, D>), dim3((unsigned)workgroups), dim3(64 * kQ8Waves), 0, st, a);
    const int64_t items = (int64_t)((int64_t)a.max_q * a.G + kQ8Cols - 1) / kQ8Cols * a.H;
    hipLaunchKernelGGL((q8_merge_kernel<DT, D>), dim3((unsigned)items, (unsigned)a.num_seqs), dim3(256), 0, st, a, (int)workgroups);
}
template <int DT, int FMT>
static void launch_stream_d(const Q8AttnArgs &a, int D, int64_t wgs, hipStream_t st) {
    D == 128 ? launch_stream<DT, FMT, 128>(a, wgs, st) : launch_stream<DT, FMT, 64>(a, wgs, st);
}
template <int DT>
static void launch_stream_f(const Q8AttnArgs &a, int fmt, int D, int64_t wgs, hipStream_t st) {
    fmt == RQ_Q8_INT8 ? launch_stream_d<DT, RQ_Q8_INT8>(a, D, wgs, st) : launch_stream_d<DT, RQ_Q8_E4M3>(a, D, wgs, st);
}

// Calls of so many columns per kv head or more go to the prefill kernels.
constexpr int64_t kQ8PromptCols = 128;
static bool q8_is_prompt(int64_t max_q_len, int G) { return max_q_len > 1 && max_q_len * G >= kQ8PromptCols; }

}  // namespace rq

using namespace rq;

extern "C" int64_t rq_q8_attention_workspace_bytes(int64_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                                   int32_t head_dim, int64_t max_q_len, int64_t max_seq_len) {
    if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0 || max_q_len <= 0 || max_seq_len < 0) return 0;
    const int G = num_q_heads / num_kv_heads;
    if (q8_is_prompt(max_q_len, G)) return q8_prefill_workspace(num_seqs, G, num_kv_heads, head_dim, max_q_len, max_seq_len);
    const int64_t wgs = q8_workgroups(num_seqs, G, num_kv_heads, max_q_len, max_seq_len);
    return 2 * wgs * kQ8Cols * (head_dim + 2) * 4;
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
    RQ_CHECK_ARG(cu_seqlens_q != nullptr || total_q == num_seqs, "without cu_seqlens_q there is one query token per sequence");
    uint32_t scale_bits;  // (by its bits: this file is compiled for arithmetic without NaN)
    __builtin_memcpy(&scale_bits, &sm_scale, 4);
    RQ_CHECK_ARG((scale_bits & 0x7f800000u) != 0x7f800000u, "sm_scale must be finite");
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
    a.cap = std::min<int64_t>(std::min<int64_t>(max_blocks * block_size, max_seq_len), INT32_MAX - 64);
    a.max_q = (int)(cu_seqlens_q ? max_q_len : 1);
    a.score_scale = sm_scale == 0.f ? 1.f : __builtin_fabsf(sm_scale) * kAttnLog2e;
    a.q_sign = sm_scale > 0.f ? 1.f : sm_scale < 0.f ? -1.f : 0.f;
    a.out = out, a.o_st = out_stride_tok, a.o_sh = out_stride_head;
    const int64_t need = rq_q8_attention_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, a.max_q, a.cap);
    RQ_CHECK_SPACE(workspace_bytes >= need, "workspace too small: the call needs %lld bytes (got %lld)", (long long)need, (long long)workspace_bytes);
    RQ_CHECK_ARG(workspace != nullptr && (uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
    a.part = static_cast<float *>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if (q8_is_prompt(a.max_q, a.G)) return q8_prefill(a, dtype, format, head_dim, workspace, st);
    const int64_t wgs = q8_workgroups(num_seqs, a.G, a.H, a.max_q, a.cap);
    if (dtype == RQ_DTYPE_BF16) launch_stream_f<RQ_DTYPE_BF16>(a, format, head_dim, wgs, st);
    else launch_stream_f<RQ_DTYPE_F16>(a, format, head_dim, wgs, st);
    return check_launch("q8_stream_kernel");
}
