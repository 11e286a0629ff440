// Plain 16-bit pages written (rq_rope_kv16_store): keys rotated by their positions and appended, values appended, and the
// query rows rotated, in one launch.  The pages are K and V (page, slot, head, dim) with any strides over whole rows.
#include "rq_rope.h"

using namespace rq;

extern "C" int rq_rope_kv16_store(const void *query, const void *key, const void *value, int32_t dtype, int64_t n_tokens, int32_t num_q_heads,
                                  int64_t q_stride_token, int64_t q_stride_head, int64_t k_stride_token, int64_t k_stride_head,
                                  int64_t v_stride_token, int64_t v_stride_head, int32_t num_kv_heads, int32_t head_dim,
                                  const int64_t *positions, const void *cos_sin, int32_t table_dtype, int64_t table_rows, int64_t table_stride,
                                  int32_t rot_dim, int32_t halves, void *out_q, int64_t out_stride_token, int64_t out_stride_head,
                                  const int64_t *slot_mapping, void *k_cache, void *v_cache, int64_t num_blocks, int32_t block_size,
                                  int64_t kc_stride_block, int64_t kc_stride_slot, int64_t kc_stride_head,
                                  int64_t vc_stride_block, int64_t vc_stride_slot, int64_t vc_stride_head, void *stream) {
    RQ_CHECK_ARG(dtype == RQ_DTYPE_F16 || dtype == RQ_DTYPE_BF16, "rows must be f16 or bf16");
    RopeRows a;
    const int rc = rope_queries(a, dtype, n_tokens, head_dim, positions, cos_sin, table_dtype, table_rows, table_stride, rot_dim, halves, query,
                                num_q_heads, q_stride_token, q_stride_head, out_q, out_stride_token, out_stride_head);
    if (rc) return rc;
    RQ_CHECK_ARG(num_kv_heads >= 1 && num_kv_heads <= 4096, "num_kv_heads %d unsupported", num_kv_heads);
    RQ_CHECK_ARG(block_size >= 1 && block_size <= 65536 && num_blocks >= 0 && num_blocks <= INT32_MAX, "bad cache sizes");
    if (n_tokens == 0) return RQ_OK;
    RQ_CHECK_ARG(key && value && slot_mapping && (num_blocks == 0 || (k_cache && v_cache)), "null pointer");
    const int64_t strides[] = {k_stride_token, k_stride_head, v_stride_token, v_stride_head, kc_stride_block, kc_stride_slot, kc_stride_head,
                               vc_stride_block, vc_stride_slot, vc_stride_head};
    bool aligned = ((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0;
    for (int64_t s : strides) aligned = aligned && s % 8 == 0;
    RQ_CHECK_ARG(aligned, "key, value and cache rows must be 16-byte aligned");
    a.n_kv = num_kv_heads;
    a.k = key, a.k_st = k_stride_token, a.k_sh = k_stride_head;
    a.v = value, a.v_st = v_stride_token, a.v_sh = v_stride_head;
    a.slots = slot_mapping;
    a.k_cache = k_cache, a.kc_sb = kc_stride_block, a.kc_ss = kc_stride_slot, a.kc_sh = kc_stride_head;
    a.v_cache = v_cache, a.vc_sb = vc_stride_block, a.vc_ss = vc_stride_slot, a.vc_sh = vc_stride_head;
    a.num_slots = num_blocks * block_size;
    a.block_size = block_size;
    RQ_CHECK_ARG(rope_threads(a) <= INT32_MAX - kRopeThreads, "too many rows for one call");
    dtype == RQ_DTYPE_F16 ? launch_rope_rows<RQ_DTYPE_F16>(a, (hipStream_t)stream) : launch_rope_rows<RQ_DTYPE_BF16>(a, (hipStream_t)stream);
    return check_launch("rope_rows_kernel");
}
