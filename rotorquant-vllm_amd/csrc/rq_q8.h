// The 8-bit KV cache: format and conversions shared by its kernels (no counterpart in the
// reference, whose cache holds 3- and 4-bit codebook indices).
//
// A group is 16 consecutive slots of a page.  For each (group, kv head) and each of K and V
// the cache holds 16 x head_dim codes c and one scale 2^e; a value is c * 2^e.
//   int8: c in -127 .. 127, stored as c + 128;   e4m3: the OCP 8-bit float (largest 448).
// e is the smallest integer of [kQ8MinExp, kQ8MaxExp] with amax <= Q * 2^e, amax the largest
// finite magnitude written to the group, Q = 127.5 (int8) or 448 (e4m3); c = x * 2^-e rounded to
// even and clamped to the largest code.  With powers of two, x * 2^-e is exact, so a code does not
// depend on how a division rounds; e4m3 codes move to a larger scale without loss (but for
// subnormals), and int8 codes are rounded again only where a group's amax crosses a power of two, which
// tokens after the first few of a group hardly ever do.
// The bounds on e keep every sum of the attention in range: a weight times 2^e and the same weight
// are both held in fp32, 2^100 apart at most.
//
// Page (block_size slots, a multiple of 16; n = block_size / 16 groups):
//   [group][head][K codes: 16 D bytes | V codes: 16 D bytes]      codes
//   [group][head]{float 2^e_k, float 2^e_v, 8 bytes unused}       scales
// A scale of 0 (a zeroed page) marks a group that was never begun.
//
// Codes lie in the order in which the MFMA operands of the attention take them (token t, dim d,
// 64-dim chunk j = d / 64; lane l = 0..63 of a wave loads bytes 16 l .. 16 l + 15 of a 1 KB chunk):
//   K: byte 1024 j + 256 ((d / 16) % 4) + 16 t + d % 16: lane (g, t) holds 16 dims of token t;
//   V: byte 1024 j + 256 (t / 4) + 16 (d % 16) + 4 ((d / 16) % 4) + t % 4: lane (g, c) holds
//      tokens 4g .. 4g + 3 of dims c, c + 16, c + 32 and c + 48, which is what the V^T operand of
//      P V takes beside weights in the order in which Q K^T leaves them.
#pragma once

#include "rq_common.h"

namespace rq {

constexpr int kQ8Group = 16;
constexpr int kQ8MinExp = -40, kQ8MaxExp = 60;

struct Q8Layout {
    int64_t tile, scales;  // bytes of a (group, head)'s codes; offset of the scales in a page
    int H;
    __host__ __device__ Q8Layout(int h, int d, int block_size)
        : tile(2 * kQ8Group * (int64_t)d), scales((int64_t)(block_size / kQ8Group) * h * tile), H(h) {}
    __host__ __device__ int64_t codes_at(int group, int head) const { return ((int64_t)group * H + head) * tile; }
    __host__ __device__ int64_t scale_at(int group, int head) const { return scales + ((int64_t)group * H + head) * 16; }
};

// Exponent of a stored scale (a power of two, 0 in a group never begun, anything in memory that
// no store ever wrote), within the format's bounds.
__device__ __forceinline__ int q8_scale_exp(float s) {
    return min(kQ8MaxExp, max(kQ8MinExp, (int)((__float_as_uint(s) >> 23) & 0xffu) - 127));
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127

// Smallest exponent with amax <= Q * 2^e (bits: those of amax >= 0, finite).
// amax = 1.m * 2^x; Q = 1.9921875 * 2^6 (int8) or 1.75 * 2^8 (e4m3).
template <int FMT>
__device__ __forceinline__ int q8_exponent(uint32_t bits) {
    constexpr uint32_t kMant = FMT == RQ_Q8_INT8 ? 0x7f0000u : 0x600000u;
    constexpr int kExp = FMT == RQ_Q8_INT8 ? 6 : 8;
    const int e = (int)(bits >> 23) - 127 - kExp + ((bits & 0x7fffffu) > kMant ? 1 : 0);
    return min(kQ8MaxExp, max(kQ8MinExp, e));
}

// Four codes of x * 2^-e, one per byte (inv = 2^-e).  NaN becomes 0; what lies past the largest code
// (infinities) takes it.
template <int FMT>
__device__ __forceinline__ uint32_t q8_encode4(const float (&x)[4], float inv) {
    constexpr float kMax = FMT == RQ_Q8_INT8 ? 127.f : 448.f;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = x[i] == x[i] ? x[i] * inv : 0.f;
        y[i] = fminf(fmaxf(v, -kMax), kMax);
    }
    if constexpr (FMT == RQ_Q8_INT8) {
        // y + 1.5 * 2^23 + 128 has its last place at 1: the sum rounds y to an even integer, and
        // its low byte is c + 128.
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[i] + 12583040.f);
        return perm(perm(b[3], b[2], 0x0c0c0400u), perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    }
}

// The four codes of a dword as numbers.
template <int FMT>
__device__ __forceinline__ void q8_decode4(uint32_t w, float (&x)[4]) {
    if constexpr (FMT == RQ_Q8_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)((w >> (8 * i)) & 0xffu) - 128.f;
    } else {
        auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
    }
}

// Transposes the 4 x 4 bytes that the four lanes of a quad (q = lane % 4) hold, one dword each:
// byte k of lane q becomes byte q of lane k.  Its own inverse.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w, int q) {
    const uint32_t p = __builtin_amdgcn_update_dpp(0, w, 0xB1, 0xf, 0xf, true);  // lane q ^ 1
    const uint32_t r = perm(p, w, q & 1 ? 0x03070105u : 0x06020400u);
    const uint32_t s = __builtin_amdgcn_update_dpp(0, r, 0x4E, 0xf, 0xf, true);  // lane q ^ 2
    return perm(s, r, q & 2 ? 0x03020706u : 0x05040100u);
}

// Host checks that every entry point on an 8-bit cache makes.
inline int check_q8_cache(int head_dim, int num_kv_heads, int block_size, int64_t num_blocks, const void *cache,
                          int64_t stride_block, int format) {
    RQ_CHECK_ARG(format == RQ_Q8_INT8 || format == RQ_Q8_E4M3, "8-bit format %d unknown", format);
    RQ_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d unsupported (64 or 128)", head_dim);
    RQ_CHECK_ARG(num_kv_heads >= 1 && num_kv_heads <= 4096, "num_kv_heads %d unsupported", num_kv_heads);
    RQ_CHECK_ARG(block_size >= kQ8Group && block_size % kQ8Group == 0 && block_size <= 65536,
                 "block_size %d must be a multiple of %d", block_size, kQ8Group);
    RQ_CHECK_ARG(num_blocks >= 0 && num_blocks <= INT32_MAX / (block_size / kQ8Group), "num_blocks %lld out of range", (long long)num_blocks);
    const int64_t page = Q8Layout(num_kv_heads, head_dim, block_size).scale_at(block_size / kQ8Group, 0);
    RQ_CHECK_ARG(stride_block >= page && stride_block % 16 == 0,
                 "pages must be %lld bytes or more, a multiple of 16 (got %lld)", (long long)page, (long long)stride_block);
    RQ_CHECK_ARG(num_blocks == 0 || (cache != nullptr && (uintptr_t)cache % 16 == 0), "the cache must be 16-byte aligned");
    return RQ_OK;
}

}  // namespace rq
