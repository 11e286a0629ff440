// Position rotation (rotary embedding) of query and key rows on the way into a cache (no counterpart in the reference, whose
// model rotates before the backend is called).
//
// A table row of `rot` numbers per position holds cosines, then sines, of rot / 2 angles.  Angle i turns the pair of dims
// (i, i + rot / 2) ("halves") or (2 i, 2 i + 1):
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,
// in fp32, each product and the sum rounded once (no fma), so that a rotated key is the same number
// wherever it is computed: the codes of all the caches go by it.  Dims from rot on pass unchanged.  A
// position outside the table turns by NaN.
//
// Rows move in pieces of 8 dims.  With halves a piece's partners are the piece rot / 16 further on (or back), so a
// multiple of 16 rotated dims keeps all loads 16 bytes wide.
#pragma once

#include "rq_common.h"

namespace rq {

struct RopeTable {
    const int64_t *positions;  // of each token
    const void *table;
    int64_t stride, rows;  // elements between rows; positions that it holds
    int rot, halves, f32;  // rotated dims; kind of pairs; table of fp32 (else of the rows' type)
};

// N (4 or 8) consecutive numbers of a table row.
template <int DT, int N>
__device__ __forceinline__ void rope_angles(const RopeTable &t, int64_t at, float *x) {
    if (DT == RQ_DTYPE_F32 || t.f32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(t.table) + at);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) x[4 * i] = p[i].x, x[4 * i + 1] = p[i].y, x[4 * i + 2] = p[i].z, x[4 * i + 3] = p[i].w;
    } else if constexpr (DT != RQ_DTYPE_F32) {
        const u32x2 *p = reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(t.table) + at);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint32_t w = p[i >> 1][i & 1];
            x[2 * i] = Elem<DT>::to_f32(w & 0xffffu), x[2 * i + 1] = Elem<DT>::to_f32(w >> 16);
        }
    }
}

// Cosines and sines: of eight pairs, or of four and four.
struct RopeTurn {
    float c[8], s[8];
};

__device__ __forceinline__ float rope_diff(float a, float c, float b, float s) {
#pragma clang fp contract(off)
    const float x = a * c, y = b * s;
    return x - y;
}
__device__ __forceinline__ float rope_sum(float a, float c, float b, float s) {
#pragma clang fp contract(off)
    const float x = a * c, y = b * s;
    return x + y;
}
// A row is worked on in units of two pieces: with halves two that are partners, else two that are as far apart; past the rotated dims two
// that pass.  A row of D dims has D / 16 units.
struct RopeUnit {
    int p0, p1;
    bool turned, also;  // either piece is (with halves both or none)
    __device__ __forceinline__ RopeUnit(const RopeTable &t, int unit) {
        const int hp = t.rot >> 4;
        turned = also = unit < hp;
        p0 = turned ? unit : 2 * unit, p1 = turned ? unit + hp : 2 * unit + 1;
    }
    // Pieces q0 and q1, partners where t is of halves.
    __device__ __forceinline__ RopeUnit(const RopeTable &t, int q0, int q1) : p0(q0), p1(q1), turned(q0 < t.rot >> 3), also(q1 < t.rot >> 3) {}
};
// The angles of a unit that is turned: eight of its pairs with halves, else four of each piece.
template <int DT>
__device__ __forceinline__ RopeTurn rope_unit_turn(const RopeTable &t, int64_t position, const RopeUnit &u) {
    RopeTurn r;
    const bool in = position >= 0 && position < t.rows;
    const int64_t row = (in ? position : 0) * t.stride, half = t.rot >> 1;
    if (t.halves) {
        rope_angles<DT, 8>(t, row + 8 * u.p0, r.c);
        rope_angles<DT, 8>(t, row + half + 8 * u.p0, r.s);
    } else {
        rope_angles<DT, 4>(t, row + 4 * u.p0, r.c);
        rope_angles<DT, 4>(t, row + half + 4 * u.p0, r.s);
        if (u.also) {
            rope_angles<DT, 4>(t, row + 4 * u.p1, r.c + 4);
            rope_angles<DT, 4>(t, row + half + 4 * u.p1, r.s + 4);
        }
    }
    if (!in) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.c[i] = r.s[i] = __builtin_nanf("");
    }
    return r;
}
// Turns a unit that is turned.
__device__ __forceinline__ void rope_unit(float (&x)[8], float (&y)[8], const RopeTurn &r, bool halves, const RopeUnit &u) {
    if (halves) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i], b = y[i];
            x[i] = rope_diff(a, r.c[i], b, r.s[i]);
            y[i] = rope_sum(b, r.c[i], a, r.s[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = rope_diff(a, r.c[i], b, r.s[i]);
            x[2 * i + 1] = rope_sum(b, r.c[i], a, r.s[i]);
            if (!u.also) continue;
            a = y[2 * i], b = y[2 * i + 1];
            y[2 * i] = rope_diff(a, r.c[4 + i], b, r.s[4 + i]);
            y[2 * i + 1] = rope_sum(b, r.c[4 + i], a, r.s[4 + i]);
        }
    }
}

// ---- rows to rows ---------------------------------------------------------------
// Query rows to rotated rows, and K and V rows to plain 16-bit pages (n_kv > 0).
struct RopeRows {
    RopeTable t;
    int64_t n_tokens;
    int n_q, n_kv, D;  // query heads, kv heads (0: queries only)
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // element strides
    void *out;
    int64_t o_st, o_sh;
    const int64_t *slots;
    void *k_cache, *v_cache;
    int64_t num_slots;
    int block_size;
    int64_t kc_sb, kc_ss, kc_sh, vc_sb, vc_ss, vc_sh;  // element strides: page, slot, head
};
constexpr int kRopeThreads = 256;

// A thread takes a unit of a row: its angles come from the caches, and rows that share them, two or four to a thread, are slower (32768 tokens of 32
// query and 8 kv heads, bf16 pages: 144 us, by two 150; 64 tokens 3.2, 3.7, by four 4.7).
__host__ __device__ __forceinline__ int64_t rope_threads(const RopeRows &a) { return a.n_tokens * (a.n_q + 2 * a.n_kv) * (a.D / 16); }
inline int64_t rope_blocks(const RopeRows &a) { return (rope_threads(a) + kRopeThreads - 1) / kRopeThreads; }

template <int DT>
__device__ __forceinline__ void rope_rows(const RopeRows &a, int64_t thread) {
    if (thread >= rope_threads(a)) return;  // (fits 32 bits)
    const uint32_t units = a.D / 16, rows = a.n_q + 2 * a.n_kv;
    const uint32_t row = (uint32_t)thread / units, tok = row / rows;
    const int r = (int)(row - tok * rows);
    const RopeUnit unit(a.t, (int)((uint32_t)thread - row * units));
    const int64_t token = tok, position = a.t.positions[token];
    const void *from = a.q;
    void *to = a.out;
    int64_t src = token * a.q_st + r * a.q_sh, dst = token * a.o_st + r * a.o_sh;
    bool turn = unit.turned;
    if (r >= a.n_q) {
        const int64_t s = a.slots[token];
        if (s < 0 || s >= a.num_slots) return;
        int64_t page;
        if (a.num_slots <= 0x7fffffff) page = (uint32_t)s / (uint32_t)a.block_size;
        else page = s / a.block_size;
        const int64_t in_page = s - page * a.block_size;
        const bool is_v = r >= a.n_q + a.n_kv;
        const int h = r - a.n_q - (is_v ? a.n_kv : 0);
        from = is_v ? a.v : a.k, to = is_v ? a.v_cache : a.k_cache;
        src = is_v ? token * a.v_st + h * a.v_sh : token * a.k_st + h * a.k_sh;
        dst = is_v ? page * a.vc_sb + in_page * a.vc_ss + h * a.vc_sh : page * a.kc_sb + in_page * a.kc_ss + h * a.kc_sh;
        turn = turn && !is_v;
    }
    Row8<DT> x0 = row8_load<DT>(from, src + 8 * unit.p0), x1 = row8_load<DT>(from, src + 8 * unit.p1);
    to = static_cast<uint8_t *>(to) + dst * (DT == RQ_DTYPE_F32 ? 4 : 2);
    if (turn) {
        const RopeTurn t = rope_unit_turn<DT>(a.t, position, unit);
        float f0[8], f1[8];
        row8_floats<DT>(x0, f0);
        row8_floats<DT>(x1, f1);
        rope_unit(f0, f1, t, a.t.halves, unit);
        x0 = row8_round<DT>(f0);
        x1 = row8_round<DT>(f1);
    }
    row8_store<DT>(to, 8 * unit.p0, x0);
    row8_store<DT>(to, 8 * unit.p1, x1);
}

template <int DT>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeRows a) {
    rope_rows<DT>(a, (int64_t)blockIdx.x * kRopeThreads + threadIdx.x);
}
template <int DT>
void launch_rope_rows(const RopeRows &a, hipStream_t st) {
    if (rope_blocks(a) > 0) hipLaunchKernelGGL((rope_rows_kernel<DT>), dim3((unsigned)rope_blocks(a)), dim3(kRopeThreads), 0, st, a);
}

// Whether a store's queries have a launch of their own: where they are long, since beside a store's registers and LDS fewer of their waves fit a CU;
// otherwise workgroups behind the store's fill what it leaves free.  rope_compress_store / rope_q8_store of 8 kv heads of 128, beside / apart, us: 32 query
// heads, 4096 tokens 31 / 36, 29 / 31; 16384 (134 MB of queries) 100 / 101, 82 / 86; 24576 147 / 148, 119 / 117; 32768 211 / 194, 166 / 154; 8 query heads,
// 65536 tokens 244 / 247, 149 / 155; 64, 16384 149 / 146, 130 / 129.
template <int DT>
bool rope_apart(const RopeRows &a) {
    return a.n_tokens * a.n_q * a.D * (DT == RQ_DTYPE_F32 ? 4 : 2) > (int64_t)192 << 20;
}

// The table and the query rows of a call, checked; strides in elements of the rows' type.
inline int rope_queries(RopeRows &a, int dtype, int64_t n_tokens, int head_dim, const int64_t *positions, const void *table, int table_dtype,
                        int64_t table_rows, int64_t table_stride, int rot_dim, int halves, const void *query, int num_q_heads, int64_t q_st,
                        int64_t q_sh, void *out, int64_t o_st, int64_t o_sh) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_F16 || dtype == RQ_DTYPE_BF16 || dtype == RQ_DTYPE_F32, "bad dtype %d", dtype);
    RQ_CHECK_ARG(table_dtype == RQ_DTYPE_F32 || table_dtype == dtype, "the table must be fp32 or of the rows' dtype");
    RQ_CHECK_ARG(head_dim >= 16 && head_dim <= 512 && head_dim % 16 == 0, "head_dim %d must be a multiple of 16 up to 512", head_dim);
    RQ_CHECK_ARG(rot_dim >= 16 && rot_dim <= head_dim && rot_dim % 16 == 0, "rot_dim %d must be a multiple of 16 up to head_dim %d", rot_dim, head_dim);
    RQ_CHECK_ARG(n_tokens >= 0 && n_tokens <= (1 << 24) && num_q_heads >= 0 && num_q_heads <= 65536 && table_rows >= 1, "bad sizes");
    RQ_CHECK_ARG(n_tokens == 0 || (positions && table && (num_q_heads == 0 || (query && out))), "null pointer");
    const int eb = dtype == RQ_DTYPE_F32 ? 4 : 2, tb = table_dtype == RQ_DTYPE_F32 ? 4 : 2;
    RQ_CHECK_ARG((uintptr_t)table % 16 == 0 && (table_rows == 1 || (table_stride >= rot_dim && table_stride * tb % 16 == 0)),
                 "table rows must be 16-byte aligned, %d numbers or more apart", rot_dim);
    RQ_CHECK_ARG(num_q_heads == 0 || ((uintptr_t)query % 16 == 0 && q_st * eb % 16 == 0 && q_sh * eb % 16 == 0 && (uintptr_t)out % 16 == 0 &&
                                      o_st * eb % 16 == 0 && o_sh * eb % 16 == 0),
                 "query and rotated query rows must be 16-byte aligned");
    a = RopeRows{};
    a.t = {positions, table, table_stride, table_rows, rot_dim, halves != 0, table_dtype == RQ_DTYPE_F32};
    a.n_tokens = n_tokens;
    a.n_q = num_q_heads, a.D = head_dim;
    a.q = query, a.q_st = q_st, a.q_sh = q_sh;
    a.out = out, a.o_st = o_st, a.o_sh = o_sh;
    RQ_CHECK_ARG(rope_threads(a) <= INT32_MAX - kRopeThreads, "too many rows for one call");
    return RQ_OK;
}

}  // namespace rq
