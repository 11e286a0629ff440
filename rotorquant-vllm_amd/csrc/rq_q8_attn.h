// Pieces that the attention kernels over the 8-bit KV cache share (rq_q8_attention.hip: short queries;
// rq_q8_prefill.hip: prompts).  The arithmetic is described in rq_q8_attention.hip.
#pragma once

#include "rq_attn_share.h"
#include "rq_q8.h"

namespace rq {

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct Q8AttnArgs : AttnBatch {
    const void *q;
    int64_t q_st, q_sh;
    const uint8_t *cache;
    int64_t num_blocks, stride_block;
    int groups;         // of a page
    float score_scale;  // |sm_scale| log2(e)
    float q_sign;       // sign of sm_scale (0 for 0)
    int max_up;         // largest s of q 2^s (below)
};

// The codes of a dword in fp16: two dwords.  int8: bytes under 0x64 are 1024 + (c + 128).
template <int FMT>
__device__ __forceinline__ void q8_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (FMT == RQ_Q8_INT8) {
        const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, perm(0x64646464u, w, 0x04010400u)) - off);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, perm(0x64646464u, w, 0x04030402u)) - off);
    } else {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true));
    }
}

// Exponent s with which a query row, its largest magnitude given by its bits, goes into fp16: q 2^s has
// its largest magnitude in [2^14, 2^15); smaller rows take max_up.  That is 60, or less where f = score_scale 2^(e_k - s) would fall
// under 2^-126 and to 0 at the smallest e_k (a masked score times 0 is NaN): score_scale 2^-max_up is 2^-86 or more.  A row
// that max_up cuts short loses parts under 2^-25 of 2^max_up, which move no score by more than 2^(-25 - 86 + 67) D.
template <int DT>
__device__ __forceinline__ int q8_query_exp(const Q8AttnArgs &a, uint32_t big) {
    return min(a.max_up, 14 - ((int)((__float_as_uint(Elem<DT>::to_f32(big)) >> 23) & 0xffu) - 127));
}
__device__ __forceinline__ uint32_t q8_max_bits(u32x4 raw, uint32_t big) {
#pragma unroll
    for (int e = 0; e < 4; ++e) big = max(big, max(raw[e] & 0x7fffu, (raw[e] >> 16) & 0x7fffu));
    return big;
}
template <int DT>
__device__ __forceinline__ u32x4 q8_query_f16(u32x4 raw, float f) {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_f16(Elem<DT>::to_f32(raw[e] & 0xffffu) * f, Elem<DT>::to_f32(raw[e] >> 16) * f);
    return o;
}

// Weights are w = 2^(u + B) in fp16.  A column's B begins at kQ8NoBias (no key seen) and becomes kQ8Peak - u at its largest u so far, but only
// when w would pass 2^kQ8Most: the largest w is 2^7 to 2^15 (fp16 ends at 2^16), so weights keep fp16's 11 bits down
// to 2^-21 of it, and those down to 2^-31 count.  The factor 2^B is in O and in l, and so not in O / l.
// With a peak of 1 and the same code a full batch of prompts takes 849 us against 859: small weights then have fewer bits to multiply.
// Where |B| is large, u + B is off by up to 1.5 of its last places (the rounding of u, and of the exponent's addend): the 2^-19 |B|
// leaves room for them up to |B| = 2^26.
constexpr float kQ8Peak = 7.f, kQ8Most = 15.f, kQ8NoBias = 3.402823466e38f;
__device__ __forceinline__ bool q8_passes(float u, float B) { return __builtin_fmaf(__builtin_fabsf(B), 0x1p-19f, u + B) > kQ8Most; }
// What the sums of several waves or workgroups are compared by.
__device__ __forceinline__ float q8_max_of(float B) { return B == kQ8NoBias ? -INFINITY : -B; }

// Prompts and chunks (rq_q8_prefill.hip).  Bytes of the workspace, and the launches.
int64_t q8_prefill_workspace_bound(int D, int64_t max_keys);
int64_t q8_prefill_workspace(int64_t num_seqs, int G, int H, int D, int64_t max_q_len, int64_t max_keys);
int q8_prefill(const Q8AttnArgs &a, int dtype, int format, int D, void *workspace, hipStream_t st);

}  // namespace rq
