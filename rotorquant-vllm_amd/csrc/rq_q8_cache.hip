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
    // calls of many tokens: per group of the cache the last run of tokens linked to it, per token the
    // run linked before its own (-1: none), and the first run's token of each group written
    int32_t *last, *before, *list, *count;
};

constexpr int kStoreWaves = 4;

// Group of token t (slot / 16), or -1 for a slot outside the cache (padding).
__device__ __forceinline__ int64_t q8_group_of(const Q8StoreArgs &a, int64_t t) {
    const int64_t s = a.slots[t];
    return s >= 0 && s < a.num_slots ? s >> 4 : -1;
}

// ---- which tokens a group gets ------------------------------------------------
// Tokens come as runs: consecutive ones of the same group (one run per group in any call that a
// server makes).  Few tokens: every unit looks at all of them (below).  Many: two launches first link the
// runs of each group, and list the groups, each by the token of the run that was linked first.
__device__ __forceinline__ int64_t q8_run_start(const Q8StoreArgs &a, int64_t t) {
    const int64_t g = q8_group_of(a, t);
    return g >= 0 && (t == 0 || q8_group_of(a, t - 1) != g) ? g : -1;
}
__global__ __launch_bounds__(256) void q8_unlink_kernel(Q8StoreArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t == 0) *a.count = 0;
    if (t >= a.n_tokens) return;
    const int64_t g = q8_run_start(a, t);
    if (g >= 0) a.last[g] = -1;
}
__global__ __launch_bounds__(256) void q8_link_kernel(Q8StoreArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.n_tokens) return;
    const int64_t g = q8_run_start(a, t);
    if (g < 0) return;
    const int32_t p = atomicExch(a.last + g, (int32_t)t);
    a.before[t] = p;
    if (p < 0) a.list[atomicAdd(a.count, 1)] = (int32_t)t;
}

// rows[r] = the last token that writes row r of group g, -1 for none.  LINKED: from the group's runs.
// Otherwise from all tokens; false if a token before t0 is of the same group (its unit does the work).
template <bool LINKED>
__device__ __forceinline__ bool q8_find_rows(const Q8StoreArgs &a, int64_t t0, int64_t g, int *rows, int lane) {
    if (lane < kQ8Group) rows[lane] = -1;
    __builtin_amdgcn_wave_barrier();
    if constexpr (LINKED) {
        for (int64_t r = a.last[g]; r >= 0; r = a.before[r]) {
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

// Eight elements (16-byte aligned) as fp32.
template <int DT>
__device__ __forceinline__ void q8_load8(const void *p, int64_t at, float (&x)[8]) {
    if constexpr (DT == RQ_DTYPE_F32) {
        const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at + 4);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
        const q8_u32x4 u = *reinterpret_cast<const q8_u32x4 *>(static_cast<const uint16_t *>(p) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = Elem<DT>::to_f32((u[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    }
}

// One unit per wave.  Lane: token row t = lane % 16, half = (lane / 16) % 2 of the 16-dim parts; the wave's
// upper 32 lanes are the second 64-dim chunk (D = 128) or the V side (D = 64).
template <int DT, int FMT, int D, bool LINKED>
__global__ __launch_bounds__(64 * kStoreWaves) void q8_store_kernel(Q8StoreArgs a) {
    constexpr int kUnits = D == 128 ? 2 : 1;  // units per head
    __shared__ int rows_of[kStoreWaves][kQ8Group];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int *const rows = rows_of[wave];
    const int t = lane & 15, half = (lane >> 4) & 1, q = t & 3;
    const uint32_t per = kUnits * a.H;
    const int64_t entries = LINKED ? *a.count : a.n_tokens;
    for (int64_t unit = (int64_t)blockIdx.x * kStoreWaves + wave; unit < entries * per; unit += (int64_t)gridDim.x * kStoreWaves) {
        const int64_t entry = unit / per;
        const int of_entry = (int)(unit - entry * per), h = of_entry / kUnits;
        const int side = D == 128 ? of_entry & 1 : lane >> 5, chunk = D == 128 ? lane >> 5 : 0;
        const int64_t t0 = LINKED ? a.list[entry] : entry;
        const int64_t g = q8_group_of(a, t0);
        if (g < 0 || (!LINKED && t0 > 0 && q8_group_of(a, t0 - 1) == g)) continue;
        if (!q8_find_rows<LINKED>(a, t0, g, rows, lane)) continue;
        const int tok = rows[t];
        const bool anew = rows[0] >= 0;
        const bool quad_hit = (__ballot(tok >= 0) >> (lane & 60)) & 15;  // four tokens share their V dwords
        const uint32_t page = (uint32_t)g / (uint32_t)a.groups, gi = (uint32_t)g - page * a.groups;
        const Q8Layout lay(a.H, D, a.block_size);
        uint8_t *const base = a.cache + (int64_t)page * a.stride_block;
        uint8_t *const tile = base + lay.codes_at(gi, h) + side * (kQ8Group * D) + chunk * 1024;
        float *const scale = reinterpret_cast<float *>(base + lay.scale_at(gi, h)) + side;
        const float old_scale = *scale;

        float x[4][8];  // dims 64 chunk + 16 i + 8 half + ...
        uint32_t big = 0;
        const void *src = side ? a.value : a.key;
        const int64_t at = (int64_t)max(tok, 0) * (side ? a.v_st : a.k_st) + (int64_t)h * (side ? a.v_sh : a.k_sh) + 64 * chunk + 8 * half;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (tok >= 0) {
                q8_load8<DT>(src, at + 16 * i, x[i]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[i][k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t b = __float_as_uint(x[i][k]) & 0x7fffffffu;
                big = max(big, b < 0x7f800000u ? b : 0u);  // infinities and NaN do not set the scale
            }
        }
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
        uint8_t *const krow = tile + 16 * t + 8 * half;              // + 256 i: dims 16 i + 8 half ..
        uint8_t *const vrow = tile + 256 * (t >> 2) + 16 * (8 * half + q);  // + 64 k: dim 8 half + 4 k + q of four parts
        if (begun && __any(tok < 0)) {
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
                    if (tok >= 0) continue;
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
        if (t == 0 && half == 0 && chunk == 0) *scale = exp2i(e_new);
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

// Stores n (2 or 4) consecutive elements.
template <int DT>
__device__ __forceinline__ void q8_put4(void *p, int64_t at, const float (&x)[4]) {
    if constexpr (DT == RQ_DTYPE_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        const uint32_t lo = Elem<DT>::from_f32(x[0]) | Elem<DT>::from_f32(x[1]) << 16;
        const uint32_t hi = Elem<DT>::from_f32(x[2]) | Elem<DT>::from_f32(x[3]) << 16;
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) = make_uint2(lo, hi);
    }
}

// One wave per (group of a sequence, head).
template <int DT, int FMT, int D>
__global__ __launch_bounds__(64 * kReadWaves) void q8_read_kernel(Q8ReadArgs a) {
    constexpr int kChunks = D / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * kReadWaves + wave;
    const int64_t unit = item / a.H;
    const int h = (int)(item - unit * a.H);
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
    const int64_t first = q8_first_unit(a, lo);
    const int64_t i = unit - first;
    const int row0 = a.starts[lo];
    const int64_t len = min((int64_t)a.seq_lens[lo], a.max_blocks * a.block_size);
    if (i < 0 || i * kQ8Group >= len) return;
    const int rows = (int)min((int64_t)kQ8Group, len - i * kQ8Group);
    const int64_t out0 = row0 + i * kQ8Group;
    const uint32_t slot_page = (uint32_t)i / (uint32_t)a.groups, gi = (uint32_t)i - slot_page * a.groups;
    int64_t page = a.bt[lo * a.bt_ss + slot_page];
    page = page < 0 || page >= a.num_blocks ? 0 : page;
    const Q8Layout lay(a.H, D, a.block_size);
    const uint8_t *const base = a.cache + page * a.stride_block;
    const uint8_t *const tile = base + lay.codes_at(gi, h) + 16 * lane;
    q8_u32x4 kw[kChunks], vw[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        kw[j] = *reinterpret_cast<const q8_u32x4 *>(tile + 1024 * j);
        vw[j] = *reinterpret_cast<const q8_u32x4 *>(tile + kQ8Group * D + 1024 * j);
    }
    const float2 s = *reinterpret_cast<const float2 *>(base + lay.scale_at(gi, h));
    const int g = lane >> 4, c = lane & 15, q = lane & 3;
    auto put = [&](void *out, int row, int dim, uint32_t w, float scale) {
        if (row >= rows || out0 + row < 0 || out0 + row >= a.total) return;
        float x[4];
        q8_decode4<FMT>(w, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] *= scale;
        q8_put4<DT>(out, ((out0 + row) * a.H + h) * D + dim, x);
    };
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            put(a.out_k, c, 64 * j + 16 * g + 4 * k, kw[j][k], s.x);
            // V: part k of this lane's dim, four tokens -> token 4 g + q, four dims
            put(a.out_v, 4 * g + q, 64 * j + 16 * k + (c & 12), quad_transpose(vw[j][k], q), s.y);
        }
}

template <int DT, int FMT, int D>
static void launch_store(const Q8StoreArgs &a, bool linked, hipStream_t st) {
    const int64_t per = (D == 128 ? 2 : 1) * (int64_t)a.H, blocks = (a.n_tokens * per + kStoreWaves - 1) / kStoreWaves;
    if (linked) {
        const unsigned tb = (unsigned)((a.n_tokens + 255) / 256);
        hipLaunchKernelGGL(q8_unlink_kernel, dim3(tb), dim3(256), 0, st, a);
        hipLaunchKernelGGL(q8_link_kernel, dim3(tb), dim3(256), 0, st, a);
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

// Tokens up to which every unit looks through all slots itself: one launch, no workspace.
constexpr int64_t kStoreScan = 512;

}  // namespace rq

using namespace rq;

extern "C" int rq_q8_slot_bytes(int32_t num_kv_heads, int32_t head_dim) {
    if (num_kv_heads < 1 || head_dim < 1) return 0;
    return (num_kv_heads * (2 * head_dim + 1) + 7) / 8 * 8;
}

extern "C" int64_t rq_q8_store_workspace_bytes(int64_t n_tokens, int64_t num_blocks, int32_t block_size) {
    if (n_tokens <= kStoreScan || num_blocks <= 0 || block_size <= 0) return 0;
    return (num_blocks * (block_size / kQ8Group) + 2 * n_tokens + 4) * 4;
}

extern "C" int rq_q8_store(const void *key, const void *value, int32_t dtype, int64_t n_tokens,
                           int64_t k_stride_token, int64_t k_stride_head, int64_t v_stride_token, int64_t v_stride_head,
                           int32_t num_kv_heads, int32_t head_dim, int32_t format, const int64_t *slot_mapping,
                           uint8_t *kv_cache, int64_t num_blocks, int32_t block_size, int64_t stride_block,
                           void *workspace, int64_t workspace_bytes, void *stream) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_F16 || dtype == RQ_DTYPE_BF16 || dtype == RQ_DTYPE_F32, "bad dtype %d", dtype);
    const int rc = check_q8_cache(head_dim, num_kv_heads, block_size, num_blocks, kv_cache, stride_block, format);
    if (rc) return rc;
    RQ_CHECK_ARG(n_tokens >= 0 && n_tokens <= (1 << 24), "n_tokens %lld out of range", (long long)n_tokens);
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
        a.list = a.count + 4;
        a.before = a.list + n_tokens;
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
