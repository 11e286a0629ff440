// The 8-bit KV cache written (rq_q8_store) and read back (rq_q8_read); the format is in rq_q8.h.
//
// Both move bytes and do little else: a token of H heads costs 4 H D bytes on its 16-bit side and
// 2 H D in the cache.  One wave takes one unit -- the K or the V codes of a (group, head), 2 KB at
// head_dim 128; both at 64 -- so that a group's amax, its old codes and its new ones stay in one wave's
// registers: no LDS tile, no barrier.  Rows become codes in the layout of the rows (lane = token t, 8 dims of each
// of four 16-dim parts); the K order needs no more, and the V order, whose dwords hold one dim of
// four tokens, takes one 4 x 4 byte transposition within quads of lanes.
#include <algorithm>

#include "rq_q8.h"

namespace rq {

typedef __attribute__((ext_vector_type(4))) uint32_t q8_u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t q8_u32x2;

struct Q8StoreArgs {
    const void *key, *value;
    int64_t k_st, k_sh, v_st, v_sh;
    int64_t n_tokens;
    const int64_t *slots;
    uint8_t *cache;
    int64_t num_slots, stride_block;
    int H, groups, block_size;  // groups of a page
    int per_wave;  // units of a wave
    // calls of many tokens: per group of the cache the last run of tokens linked to it, per token the
    // run linked before its own (-1: none), and of each group written the token linked first and the group
    int32_t *last, *before, *count;
    int2 *list;
};

constexpr int kStoreWaves = 4;

// Group of token t (slot / 16), or -1 for a slot outside the cache (padding).
__device__ __forceinline__ int64_t q8_group_of(const Q8StoreArgs &a, int64_t t) {
    const int64_t s = a.slots[t];
    return s >= 0 && s < a.num_slots ? s >> 4 : -1;
}

// ---- which tokens a group gets ------------------------------------------------
// Tokens come as runs: consecutive ones of the same group (one run per group in any call that a
// server makes).  Few tokens: every wave looks at all of them (below).  Many: two launches first link the
// runs of each group, and list the groups, each with the token of the run that was linked first.
__device__ __forceinline__ int64_t q8_run_start(const Q8StoreArgs &a, int64_t t) {
    const int64_t g = q8_group_of(a, t);
    return g >= 0 && (t == 0 || q8_group_of(a, t - 1) != g) ? g : -1;
}
constexpr int kLinkThreads = 1024;
__global__ __launch_bounds__(kLinkThreads) void q8_unlink_kernel(Q8StoreArgs a) {
    const int64_t t = (int64_t)blockIdx.x * kLinkThreads + threadIdx.x;
    if (t == 0) *a.count = 0;
    if (t >= a.n_tokens) return;
    const int64_t g = q8_run_start(a, t);
    if (g >= 0) a.last[g] = -1;
}
// The list's places come from one addition per workgroup: additions of every wave to the one counter took 3 us of 8 (32768 tokens).
__global__ __launch_bounds__(kLinkThreads) void q8_link_kernel(Q8StoreArgs a) {
    __shared__ int found, base;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    const int64_t t = (int64_t)blockIdx.x * kLinkThreads + threadIdx.x;
    const int64_t g = t < a.n_tokens ? q8_run_start(a, t) : -1;
    int place = -1;
    if (g >= 0) {
        const int32_t p = atomicExch(a.last + g, (int32_t)t);
        a.before[t] = p;
        if (p < 0) place = atomicAdd(&found, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0 && found > 0) base = atomicAdd(a.count, found);
    __syncthreads();
    if (place >= 0) a.list[base + place] = make_int2((int)t, (int)g);
}

// rows[r] = the last token that writes row r of group g, -1 for none.  LINKED: t0 is the token of the group's list entry.  Otherwise
// from all tokens; false if one before t0 is of the same group (its wave does the work).
template <bool LINKED>
__device__ __forceinline__ bool q8_find_rows(const Q8StoreArgs &a, int64_t t0, int64_t g, int *rows, int lane) {
    if (lane < kQ8Group) rows[lane] = -1;
    __builtin_amdgcn_wave_barrier();
    if constexpr (LINKED) {
        const int64_t s0 = t0 + lane < a.n_tokens ? a.slots[t0 + lane] : -1;
        int64_t r = a.last[g];
        if (r == t0) {  // the only run (its slots are loaded beside the link); of 64 tokens or more: below
            const uint64_t out = ~__ballot(s0 >= 0 && s0 >> 4 == g);
            if (out) {
                if (lane < __builtin_ctzll(out)) atomicMax(rows + (s0 & 15), (int)(t0 + lane));
                r = -1;
            }
        }
        // (each run is linked once, so the walk ends by itself; the bounds hold also where slots change under the call)
        for (int64_t left = a.n_tokens; r >= 0 && r < a.n_tokens && left > 0; r = a.before[r], --left) {
            for (int64_t s = r;; s += 64) {  // the run: up to the first token of another group
                const bool in = s + lane < a.n_tokens && q8_group_of(a, s + lane) == g;
                const uint64_t out = ~__ballot(in);
                const int n = out ? __builtin_ctzll(out) : 64;
                if (lane < n) atomicMax(rows + (a.slots[s + lane] & 15), (int)(s + lane));
                if (n < 64) break;
            }
        }
    } else {
        bool earlier = false;
        for (int64_t s = lane; s < a.n_tokens; s += 256) {
            int64_t at[4];  // (four loads in flight)
#pragma unroll
            for (int u = 0; u < 4; ++u) at[u] = s + 64 * u < a.n_tokens ? a.slots[s + 64 * u] : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (at[u] < 0 || at[u] >> 4 != g) continue;
                earlier |= s + 64 * u < t0;
                atomicMax(rows + (at[u] & 15), (int)(s + 64 * u));
            }
        }
        if (__any(earlier)) return false;
    }
    __builtin_amdgcn_wave_barrier();
    return true;
}

// Eight elements (16-byte aligned), as loaded and as fp32.
template <int DT>
struct Q8Raw {
    q8_u32x4 w[DT == RQ_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Q8Raw<DT> q8_load8(const void *p, int64_t at) {
    Q8Raw<DT> r;
    const q8_u32x4 *q = reinterpret_cast<const q8_u32x4 *>(static_cast<const uint8_t *>(p) + at * (DT == RQ_DTYPE_F32 ? 4 : 2));
    r.w[0] = *q;
    if constexpr (DT == RQ_DTYPE_F32) r.w[1] = q[1];
    return r;
}
template <int DT>
__device__ __forceinline__ void q8_floats(const Q8Raw<DT> &r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (DT == RQ_DTYPE_F32) x[i] = __uint_as_float(r.w[i >> 2][i & 3]);
        else x[i] = Elem<DT>::to_f32((r.w[0][i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
}

// A wave takes a.per_wave units of one group, the next one's rows on their way while one is coded.  Lane: token row
// t = lane % 16, half = (lane / 16) % 2 of the 16-dim parts; the wave's upper 32 lanes are the second 64-dim chunk
// (D = 128) or the V side (D = 64).
// Bound by memory: 32768 tokens of 8 heads (134 MB in, 67 out) in 47 us beside 10 for the two link launches (graph replays of all three: 48).  Non-temporal loads
// here: 56 us (a row's 128 bytes are loaded by four instructions, which then miss the L1).
template <int DT, int FMT, int D, bool LINKED>
__global__ __launch_bounds__(64 * kStoreWaves) void q8_store_kernel(Q8StoreArgs a) {
    constexpr int kUnits = D == 128 ? 2 : 1;  // units per head
    __shared__ int rows_of[kStoreWaves][kQ8Group];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int *const rows = rows_of[wave];
    const int t = lane & 15, half = (lane >> 4) & 1, q = t & 3;
    const int units = kUnits * a.H, waves = (units + a.per_wave - 1) / a.per_wave;  // of a group
    const int64_t entries = LINKED ? *a.count : a.n_tokens;
    const Q8Layout lay(a.H, D, a.block_size);
    for (int64_t item = (int64_t)blockIdx.x * kStoreWaves + wave; item < entries * waves; item += (int64_t)gridDim.x * kStoreWaves) {
        const uint32_t entry = (uint32_t)item / (uint32_t)waves;
        const int first = (int)((uint32_t)item - entry * waves) * a.per_wave, end = min(units, first + a.per_wave);
        int64_t t0 = entry, g;
        if constexpr (LINKED) {
            const int2 e = a.list[entry];
            t0 = e.x, g = e.y;
        } else {
            g = q8_group_of(a, t0);
            if (g < 0 || (t0 > 0 && q8_group_of(a, t0 - 1) == g)) continue;
        }
        if (!q8_find_rows<LINKED>(a, t0, g, rows, lane)) continue;
        const int tok = rows[t];
        const bool anew = rows[0] >= 0;
        const uint64_t written = __ballot(tok >= 0);
        const bool quad_hit = (written >> (lane & 60)) & 15;  // four tokens share their V dwords
        const uint32_t page = (uint32_t)g / (uint32_t)a.groups, gi = (uint32_t)g - page * a.groups;
        uint8_t *const base = a.cache + (int64_t)page * a.stride_block;

        auto side_of = [&](int unit) { return D == 128 ? unit & 1 : lane >> 5; };
        const int chunk = D == 128 ? lane >> 5 : 0;
        Q8Raw<DT> raw[4];
        float old_next;
        auto scale_at = [&](int unit) { return reinterpret_cast<float *>(base + lay.scale_at(gi, unit / kUnits)) + side_of(unit); };
        auto load = [&](int unit) {  // dims 64 chunk + 16 i + 8 half .. of this lane's row
            const int h = unit / kUnits, side = side_of(unit);
            old_next = *scale_at(unit);
            const int64_t at = (int64_t)tok * (side ? a.v_st : a.k_st) + (int64_t)h * (side ? a.v_sh : a.k_sh) + 64 * chunk + 8 * half;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (tok >= 0) raw[i] = q8_load8<DT>(side ? a.value : a.key, at + 16 * i);
        };
        load(first);
        for (int unit = first; unit < end; ++unit) {
            const int h = unit / kUnits, side = side_of(unit);
            uint8_t *const tile = base + lay.codes_at(gi, h) + side * (kQ8Group * D) + chunk * 1024;
            const float old_scale = old_next;
            float x[4][8];
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q8_floats<DT>(raw[i], x[i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (tok < 0) x[i][k] = 0.f;
                    const uint32_t b = __float_as_uint(x[i][k]) & 0x7fffffffu;
                    big = max(big, b < 0x7f800000u ? b : 0u);  // infinities and NaN do not set the scale
                }
            }
            if (unit + 1 < end) load(unit + 1);
#pragma unroll
            for (int o = D == 128 ? 32 : 16; o >= 1; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o));
            const bool begun = !anew && old_scale != 0.f;  // the rows not written keep their tokens
            const int e_old = q8_scale_exp(old_scale), e_new = max(q8_exponent<FMT>(big), begun ? e_old : kQ8MinExp);
            const bool moved = !begun || e_new != e_old;   // every row is written
            const float inv = exp2i(-e_new);
            uint32_t c[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo[4] = {x[i][0], x[i][1], x[i][2], x[i][3]}, hi[4] = {x[i][4], x[i][5], x[i][6], x[i][7]};
                c[i][0] = q8_encode4<FMT>(lo, inv);
                c[i][1] = q8_encode4<FMT>(hi, inv);
            }
            uint8_t *const krow = tile + 16 * t + 8 * half;                     // + 256 i: dims 16 i + 8 half ..
            uint8_t *const vrow = tile + 256 * (t >> 2) + 16 * (8 * half + q);  // + 64 k: dim 8 half + 4 k + q of four parts
            if ((uint32_t)(written & 0xffff) != 0xffffu && __any(begun)) {
                // codes of the rows that stay, in this lane's order, moved to the new scale
                uint32_t old[4][2];
                if (side == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const q8_u32x2 w = *reinterpret_cast<const q8_u32x2 *>(krow + 256 * i);
                        old[i][0] = w[0], old[i][1] = w[1];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const q8_u32x4 w = *reinterpret_cast<const q8_u32x4 *>(vrow + 64 * k);
#pragma unroll
                        for (int i = 0; i < 4; ++i) old[i][k] = quad_transpose(w[i], q);
                    }
                }
                const float shift = exp2i(e_old - e_new);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (tok >= 0 || !begun) continue;
                        float y[4];
                        q8_decode4<FMT>(old[i][k], y);
                        c[i][k] = moved ? q8_encode4<FMT>(y, shift) : old[i][k];
                    }
            }
            if (side == 0) {
                if (tok >= 0 || moved) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<q8_u32x2 *>(krow + 256 * i) = q8_u32x2{c[i][0], c[i][1]};
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    q8_u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = quad_transpose(c[i][k], q);
                    if (moved || quad_hit) *reinterpret_cast<q8_u32x4 *>(vrow + 64 * k) = w;
                }
            }
            if (t == 0 && half == 0 && chunk == 0) *scale_at(unit) = exp2i(e_new);
        }
    }
}

// ---- read back ------------------------------------------------------------------
struct Q8ReadArgs {
    const uint8_t *cache;
    int64_t num_blocks, stride_block;
    int H, groups, block_size;
    const int32_t *bt;
    int64_t max_blocks, bt_ss;
    const int32_t *seq_lens, *starts;
    int64_t num_seqs, total;
    void *out_k, *out_v;
};

constexpr int kReadWaves = 4;

// Units of the sequences: sequence b's group i is number starts[b] / 16 + b + i.  A sequence of n rows has
// at most ceil(n / 16) groups, which is what lies between two sequences' first numbers or less, so
// the numbers need no prefix sum over the lengths; those in between stay idle.
__device__ __forceinline__ int64_t q8_first_unit(const Q8ReadArgs &a, int64_t b) { return (int64_t)(a.starts[b] >> 4) + b; }

// Eight codes (two dwords) times scale as eight consecutive elements.
template <int DT, int FMT>
__device__ __forceinline__ void q8_put8(void *p, int64_t at, uint32_t w0, uint32_t w1, float scale) {
    float x[8], lo[4], hi[4];
    q8_decode4<FMT>(w0, lo);
    q8_decode4<FMT>(w1, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = lo[k] * scale, x[4 + k] = hi[k] * scale;
    if constexpr (DT == RQ_DTYPE_F32) {
        float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + at);
        q[0] = make_float4(x[0], x[1], x[2], x[3]);
        q[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        q8_u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = Elem<DT>::from_f32(x[2 * k]) | Elem<DT>::from_f32(x[2 * k + 1]) << 16;
        *reinterpret_cast<q8_u32x4 *>(static_cast<uint16_t *>(p) + at) = w;
    }
}
// The value of lane l ^ 4.
__device__ __forceinline__ uint32_t lane_xor4(uint32_t x) {
    const int from_above = __builtin_amdgcn_update_dpp(0, (int)x, 0x104, 0xf, 0x5, false);             // lanes with bit 2 clear: row_shl 4
    return (uint32_t)__builtin_amdgcn_update_dpp(from_above, (int)x, 0x114, 0xf, 0xa, false);          // the others: row_shr 4
}

// One wave per (group of a sequence, head).  Codes change lanes (and bytes of V, quads) so that every store is 16 bytes a
// lane (8 elements of 16 bits) and four lanes' are 64 consecutive bytes of a row.
// Bound by memory: 131072 tokens of 8 heads (270 MB in, 537 out) in 164 us, 4.9 TB/s (a copy: 5.1); 32768 in 46.  Two or
// four heads a wave, the next one's codes loaded ahead: 167 and 183 us; non-temporal stores: 182.
template <int DT, int FMT, int D>
__global__ __launch_bounds__(64 * kReadWaves) void q8_read_kernel(Q8ReadArgs a) {
    constexpr int kChunks = D / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * kReadWaves + wave;  // (fits 32 bits)
    const uint32_t unit = (uint32_t)item / (uint32_t)a.H;
    const int h = (int)((uint32_t)item - unit * a.H);
    // the last sequence whose first unit is not past this one, 64 at a time
    int64_t lo = 0, n = a.num_seqs;
    while (n > 1) {
        const int64_t step = (n + 63) / 64, b = lo + lane * step;
        const uint64_t in = __ballot(b < lo + n && q8_first_unit(a, b) <= unit);
        if (in == 0) return;
        const int64_t next = lo + (63 - __builtin_clzll(in)) * step;
        n = min(step, lo + n - next);
        lo = next;
    }
    const int64_t i = unit - q8_first_unit(a, lo);
    const int64_t len = min((int64_t)a.seq_lens[lo], a.max_blocks * a.block_size);
    if (i < 0 || i * kQ8Group >= len) return;
    const int rows = (int)min((int64_t)kQ8Group, len - i * kQ8Group);
    const int64_t out0 = a.starts[lo] + i * kQ8Group;
    const uint32_t slot_page = (uint32_t)i / (uint32_t)a.groups, gi = (uint32_t)i - slot_page * a.groups;
    int64_t page = a.bt[lo * a.bt_ss + slot_page];
    page = page < 0 || page >= a.num_blocks ? 0 : page;
    const Q8Layout lay(a.H, D, a.block_size);
    const uint8_t *const base = a.cache + page * a.stride_block;
    const uint8_t *const tile = base + lay.codes_at(gi, h) + 16 * lane;
    q8_u32x4 kc[kChunks], vc[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        kc[j] = __builtin_nontemporal_load(reinterpret_cast<const q8_u32x4 *>(tile + 1024 * j));
        vc[j] = __builtin_nontemporal_load(reinterpret_cast<const q8_u32x4 *>(tile + kQ8Group * D + 1024 * j));
    }
    const float2 scale = *reinterpret_cast<const float2 *>(base + lay.scale_at(gi, h));
    const int g = lane >> 4, c = lane & 15, q = lane & 3;
    const bool upper = lane & 4;
    auto inside = [&](int row) { return row < rows && out0 + row >= 0 && out0 + row < a.total; };
    const bool k_in = inside(c), v_in = inside(4 * g + q);
    const int64_t k_row = ((out0 + c) * a.H + h) * D, v_row = ((out0 + 4 * g + q) * a.H + h) * D;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        // K: lane group g has dims 16 g .. + 15 of token c -> dims 8 g .. + 7 and 32 + 8 g .. + 7
        uint32_t p[2][2];
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            auto x = __builtin_amdgcn_permlane16_swap(kc[j][d], kc[j][2 + d], false, false);
            auto y = __builtin_amdgcn_permlane32_swap(x[0], x[1], false, false);
            p[0][d] = y[0], p[1][d] = y[1];
        }
        if (k_in) {
#pragma unroll
            for (int u = 0; u < 2; ++u) q8_put8<DT, FMT>(a.out_k, k_row + 64 * j + 32 * u + 8 * g, p[u][0], p[u][1], scale.x);
        }
        // V: four tokens of dim 16 k + c -> dims 16 k + (c & 12) .. + 3 of token 4 g + q -> 8 dims, of part k or k + 1
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint32_t w0 = quad_transpose(vc[j][k], q), w1 = quad_transpose(vc[j][k + 1], q);
            const uint32_t other = lane_xor4(upper ? w0 : w1);
            if (v_in)
                q8_put8<DT, FMT>(a.out_v, v_row + 64 * j + 16 * (k + (upper ? 1 : 0)) + (c & 8), upper ? other : w0, upper ? w1 : other, scale.y);
        }
    }
}

// Units of a wave in a long call: two once one each would be more waves than the GPU holds (about 24 a CU).  GPU time of the store
// alone, 8 heads, one / two / four units: 1024 tokens 9.7 / 10.7 / 13.5 us, 4096: 14.4 / 14.5 / 15.8, 8192 (just under the border):
// 20.1 / 19.3 / 19.1, 32768: 54.0 / 48.3 / 49.5.
static int q8_per_wave(int64_t groups, int units) { return groups * units >= 48 * (int64_t)device_cus() ? 2 : 1; }

template <int DT, int FMT, int D>
static void launch_store(Q8StoreArgs a, bool linked, hipStream_t st) {
    const int units = (D == 128 ? 2 : 1) * a.H;
    a.per_wave = linked ? q8_per_wave(a.n_tokens / kQ8Group, units) : 1;
    const int64_t blocks = (a.n_tokens * ((units + a.per_wave - 1) / a.per_wave) + kStoreWaves - 1) / kStoreWaves;
    if (linked) {
        const dim3 tb((unsigned)((a.n_tokens + kLinkThreads - 1) / kLinkThreads));
        hipLaunchKernelGGL(q8_unlink_kernel, tb, dim3(kLinkThreads), 0, st, a);
        hipLaunchKernelGGL(q8_link_kernel, tb, dim3(kLinkThreads), 0, st, a);
        const unsigned grid = (unsigned)std::min<int64_t>(blocks, 8 * device_cus());
        hipLaunchKernelGGL((q8_store_kernel<DT, FMT, D, true>), dim3(grid), dim3(64 * kStoreWaves), 0, st, a);
    } else {
        hipLaunchKernelGGL((q8_store_kernel<DT, FMT, D, false>), dim3((unsigned)blocks), dim3(64 * kStoreWaves), 0, st, a);
    }
}
template <int DT, int FMT>
static void launch_store_d(const Q8StoreArgs &a, int D, bool linked, hipStream_t st) {
    D == 128 ? launch_store<DT, FMT, 128>(a, linked, st) : launch_store<DT, FMT, 64>(a, linked, st);
}
template <int DT>
static void launch_store_f(const Q8StoreArgs &a, int fmt, int D, bool linked, hipStream_t st) {
    fmt == RQ_Q8_INT8 ? launch_store_d<DT, RQ_Q8_INT8>(a, D, linked, st) : launch_store_d<DT, RQ_Q8_E4M3>(a, D, linked, st);
}

template <int DT, int FMT>
static void launch_read_d(const Q8ReadArgs &a, int D, hipStream_t st) {
    const int64_t items = (a.total / kQ8Group + a.num_seqs) * a.H;
    const dim3 grid((unsigned)((items + kReadWaves - 1) / kReadWaves)), block(64 * kReadWaves);
    if (D == 128) hipLaunchKernelGGL((q8_read_kernel<DT, FMT, 128>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((q8_read_kernel<DT, FMT, 64>), grid, block, 0, st, a);
}
template <int DT>
static void launch_read_f(const Q8ReadArgs &a, int fmt, int D, hipStream_t st) {
    fmt == RQ_Q8_INT8 ? launch_read_d<DT, RQ_Q8_INT8>(a, D, st) : launch_read_d<DT, RQ_Q8_E4M3>(a, D, st);
}

// Tokens up to which every wave looks through all slots itself: one launch, no workspace.  GPU time of the store alone, 8 heads, itself /
// linked: appended tokens (a group each) 16: 4.9 / 8.8 us, 128: 5.8 / 10.0, 256: 7.9 / 12.0, 512: 13.5 / 17.3, 1024: 27.5 / 28.0;
// prompts 256: 7.3 / 8.9, 512: 9.7 / 9.3, 1024: 17.7 / 9.6, 2048: 39 / 10.7.  (Its work grows with the square of the tokens.)
constexpr int64_t kStoreScan = 512;

}  // namespace rq

using namespace rq;

extern "C" int rq_q8_slot_bytes(int32_t num_kv_heads, int32_t head_dim) {
    if (num_kv_heads < 1 || head_dim < 1) return 0;
    const int64_t bytes = (num_kv_heads * (2 * (int64_t)head_dim + 1) + 7) / 8 * 8;
    return bytes <= INT32_MAX ? (int)bytes : 0;
}

extern "C" int64_t rq_q8_store_workspace_bytes(int64_t n_tokens, int64_t num_blocks, int32_t block_size) {
    if (n_tokens <= kStoreScan || num_blocks <= 0 || block_size <= 0) return 0;
    return (num_blocks * (block_size / kQ8Group) + 3 * n_tokens + 4) * 4;
}

extern "C" int rq_q8_store(const void *key, const void *value, int32_t dtype, int64_t n_tokens,
                           int64_t k_stride_token, int64_t k_stride_head, int64_t v_stride_token, int64_t v_stride_head,
                           int32_t num_kv_heads, int32_t head_dim, int32_t format, const int64_t *slot_mapping,
                           uint8_t *kv_cache, int64_t num_blocks, int32_t block_size, int64_t stride_block,
                           void *workspace, int64_t workspace_bytes, void *stream) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_F16 || dtype == RQ_DTYPE_BF16 || dtype == RQ_DTYPE_F32, "bad dtype %d", dtype);
    const int rc = check_q8_cache(head_dim, num_kv_heads, block_size, num_blocks, kv_cache, stride_block, format);
    if (rc) return rc;
    RQ_CHECK_ARG(n_tokens >= 0 && n_tokens <= (1 << 30) / num_kv_heads, "n_tokens %lld out of range", (long long)n_tokens);
    if (n_tokens == 0 || num_blocks == 0) return RQ_OK;
    RQ_CHECK_ARG(key && value && slot_mapping, "null pointer");
    const int eb = dtype == RQ_DTYPE_F32 ? 4 : 2;
    RQ_CHECK_ARG((uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0 && k_stride_token * eb % 16 == 0 &&
                     k_stride_head * eb % 16 == 0 && v_stride_token * eb % 16 == 0 && v_stride_head * eb % 16 == 0,
                 "key/value rows must be 16-byte aligned");
    const int64_t need = rq_q8_store_workspace_bytes(n_tokens, num_blocks, block_size);
    RQ_CHECK_SPACE(workspace_bytes >= need, "workspace too small: the call needs %lld bytes (got %lld)", (long long)need,
                   (long long)workspace_bytes);
    RQ_CHECK_ARG(need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "workspace must be 16-byte aligned");
    Q8StoreArgs a{};
    a.key = key, a.value = value;
    a.k_st = k_stride_token, a.k_sh = k_stride_head, a.v_st = v_stride_token, a.v_sh = v_stride_head;
    a.n_tokens = n_tokens;
    a.slots = slot_mapping;
    a.cache = kv_cache;
    a.num_slots = num_blocks * block_size;
    a.stride_block = stride_block;
    a.H = num_kv_heads;
    a.block_size = block_size;
    a.groups = block_size / kQ8Group;
    if (need) {
        a.count = static_cast<int32_t *>(workspace);
        a.list = reinterpret_cast<int2 *>(a.count + 4);
        a.before = reinterpret_cast<int32_t *>(a.list + n_tokens);
        a.last = a.before + n_tokens;
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RQ_DTYPE_F16) launch_store_f<RQ_DTYPE_F16>(a, format, head_dim, need > 0, st);
    else if (dtype == RQ_DTYPE_BF16) launch_store_f<RQ_DTYPE_BF16>(a, format, head_dim, need > 0, st);
    else launch_store_f<RQ_DTYPE_F32>(a, format, head_dim, need > 0, st);
    return check_launch("q8_store_kernel");
}

extern "C" int rq_q8_read(const uint8_t *kv_cache, int64_t num_blocks, int32_t block_size, int64_t stride_block,
                          int32_t num_kv_heads, int32_t head_dim, int32_t format, const int32_t *block_table,
                          int64_t max_blocks, int64_t bt_stride_seq, const int32_t *seq_lens, const int32_t *starts,
                          int64_t num_seqs, int64_t total, void *out_k, void *out_v, int32_t out_dtype, void *stream) {
    RQ_CHECK_ARG(out_dtype == RQ_DTYPE_F16 || out_dtype == RQ_DTYPE_BF16 || out_dtype == RQ_DTYPE_F32, "bad dtype %d", out_dtype);
    const int rc = check_q8_cache(head_dim, num_kv_heads, block_size, num_blocks, kv_cache, stride_block, format);
    if (rc) return rc;
    RQ_CHECK_ARG(num_seqs >= 0 && num_seqs <= (1 << 24) && total >= 0 && total <= INT32_MAX && max_blocks >= 0, "bad sizes");
    RQ_CHECK_ARG((total / kQ8Group + num_seqs) * num_kv_heads <= INT32_MAX, "too many rows and heads for one call");
    if (num_seqs == 0 || total == 0 || max_blocks == 0 || num_blocks == 0) return RQ_OK;
    RQ_CHECK_ARG(block_table && seq_lens && starts && out_k && out_v, "null pointer");
    RQ_CHECK_ARG((uintptr_t)out_k % 16 == 0 && (uintptr_t)out_v % 16 == 0, "outputs must be 16-byte aligned");
    Q8ReadArgs a{};
    a.cache = kv_cache;
    a.num_blocks = num_blocks;
    a.stride_block = stride_block;
    a.H = num_kv_heads;
    a.block_size = block_size;
    a.groups = block_size / kQ8Group;
    a.bt = block_table;
    a.max_blocks = max_blocks;
    a.bt_ss = bt_stride_seq;
    a.seq_lens = seq_lens;
    a.starts = starts;
    a.num_seqs = num_seqs;
    a.total = total;
    a.out_k = out_k, a.out_v = out_v;
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == RQ_DTYPE_F16) launch_read_f<RQ_DTYPE_F16>(a, format, head_dim, st);
    else if (out_dtype == RQ_DTYPE_BF16) launch_read_f<RQ_DTYPE_BF16>(a, format, head_dim, st);
    else launch_read_f<RQ_DTYPE_F32>(a, format, head_dim, st);
    return check_launch("q8_read_kernel");
}
