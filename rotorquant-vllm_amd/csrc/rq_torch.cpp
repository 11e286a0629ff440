// The torch side of the entry points whose calls take less time on the GPU than a Python function takes to look through their tensors
// (rotorquant_vllm._rq_torch; the documented functions are in rotorquant_vllm/kernels/rope.py and kv16.py).  It checks tensors, takes
// the current stream of their device and scratch from torch's allocator, and calls the C ABI of librq_hip.so, which checks
// sizes, strides and alignment.  A rotating store of a decode step, whose kernel takes 4 us: 10.5 us of host time through ctypes, 4.4 through this.
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <sstream>
#include <string>

#include "../../include/rq_abi.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

template <typename... T>
std::string text(const T &...t) {
    std::ostringstream s;
    (s << ... << t);
    return s.str();
}
[[noreturn]] void refuse(const std::string &why) { throw py::value_error(why); }

std::string name_of(at::ScalarType t) { return t == at::kHalf ? "float16" : t == at::kBFloat16 ? "bfloat16" : t == at::kFloat ? "float32" : c10::toString(t); }
std::string shape_of(const Tensor &t) {
    std::ostringstream s;
    s << "(";
    for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
    s << ")";
    return s.str();
}

// The device that all tensors are on.
struct OnDevice {
    const Tensor &first;
    explicit OnDevice(const Tensor &t) : first(t) { cuda(t); }
    static void cuda(const Tensor &t) {
        if (!t.is_cuda())
            throw std::runtime_error(text("rotorquant_vllm.kernels runs only on ROCm device tensors (got a ", c10::DeviceTypeName(t.device().type(), true),
                                          " tensor); there is no CPU path"));
    }
    void also(const Tensor &t) const {
        cuda(t);
        if (t.get_device() != first.get_device()) refuse(text("tensors on ", first.device().str(), " and ", t.device().str()));
    }
    void also(const OptTensor &t) const {
        if (t) also(*t);
    }
};

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return RQ_DTYPE_F16;
        case at::kBFloat16: return RQ_DTYPE_BF16;
        case at::kFloat: return RQ_DTYPE_F32;
        default: throw py::type_error("unsupported dtype " + name_of(t));
    }
}

void check_status(int rc, const char *name) {
    if (rc == RQ_OK) return;
    if (rc == RQ_EINVAL) refuse(text(name, ": ", rq_last_error()));
    throw std::runtime_error(text(name, " failed (status ", rc, "): ", rq_last_error()));
}

// The C ABI takes counts of heads, dims, slots and the like as ints.
int count(int64_t n) {
    if (n > INT32_MAX) refuse(text("a dimension of ", n, " is too large"));
    return (int)n;
}

// Strides over a single token or head may be any number in a view.
int64_t step(const Tensor &t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

// Scratch: the caller's buffer, or of this call from the stream's allocator.
struct Scratch {
    Tensor keep;
    void *at = nullptr;
    int64_t bytes = 0;
    Scratch(const OptTensor &given, int64_t need, const Tensor &like) {
        if (given) {
            if (given->scalar_type() != at::kByte || !given->is_contiguous()) refuse("workspace must be a contiguous uint8 tensor");
            keep = *given;
        } else if (need > 0) {
            keep = at::empty({need}, like.options().dtype(at::kByte));
        }
        if (keep.defined()) at = keep.data_ptr(), bytes = keep.numel();
    }
};

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// ---- position rotation -------------------------------------------------------------
struct Rope {
    const Tensor &key, &value, &positions, &table;
    OptTensor query, out;
    int64_t N, H, D, HQ = 0;
    int dtype;
    Rope(const OptTensor &q, const Tensor &k, const Tensor &v, const Tensor &p, const Tensor &t, const Tensor &slots, const OptTensor &out_q)
        : key(k), value(v), positions(p), table(t), query(q) {
        OnDevice on(k);
        on.also(v), on.also(q), on.also(p), on.also(t), on.also(slots), on.also(out_q);
        const auto type = k.scalar_type();
        if (k.dim() != 3 || !v.sizes().equals(k.sizes()) || v.scalar_type() != type)
            refuse("key and value must have the same (tokens, heads, head_dim) shape and dtype");
        N = k.size(0), H = k.size(1), D = k.size(2);
        if (k.stride(2) != 1 || v.stride(2) != 1) refuse("key and value must be contiguous over head_dim");
        for (const auto &[x, name] : {std::pair<const Tensor &, const char *>(p, "positions"), {slots, "slot_mapping"}})
            if (x.scalar_type() != at::kLong || x.dim() != 1 || x.numel() < N || !x.is_contiguous())
                refuse(text(name, " must be a contiguous int64 tensor of ", N, " tokens or more"));
        if (t.dim() != 2 || t.stride(1) != 1 || (t.scalar_type() != at::kFloat && t.scalar_type() != type))
            refuse("cos_sin must be (positions, rot_dim), contiguous over rot_dim, of float32 or " + name_of(type));
        dtype = dtype_code(type);
        if (!q) {
            if (out_q) refuse("out_q without query");
            return;
        }
        if (q->dim() != 3 || q->size(0) != N || q->size(2) != D || q->scalar_type() != type)
            refuse(text("query must be (", N, ", heads, ", D, ") of ", name_of(type), ", as key is"));
        HQ = q->size(1);
        out = out_q ? *out_q : at::empty(q->sizes(), q->options());
        if (!out->sizes().equals(q->sizes()) || out->scalar_type() != type) refuse("out_q must have query's shape and dtype");
        if (q->stride(2) != 1 || out->stride(2) != 1) refuse("query and out_q must be contiguous over head_dim");
    }
    // fn(the arguments that every store begins with, more...)
    template <typename F, typename... T>
    void call(F fn, const char *name, bool neox, T... more) const {
        const bool q = query.has_value();
        check_status(fn(q ? query->data_ptr() : nullptr, key.data_ptr(), value.data_ptr(), dtype, N, count(HQ), q ? step(*query, 0) : 0,
                        q ? step(*query, 1) : 0, step(key, 0), step(key, 1), step(value, 0), step(value, 1), count(H), count(D),
                        positions.data_ptr<int64_t>(), table.data_ptr(), dtype_code(table.scalar_type()), table.size(0), table.stride(0),
                        count(table.size(1)), neox ? 1 : 0, q ? out->data_ptr() : nullptr, q ? step(*out, 0) : 0, q ? step(*out, 1) : 0, more...),
                     name);
    }
};

void check_bytes(const Tensor &cache, const char *what) {
    if (cache.scalar_type() != at::kByte || cache.dim() != 3) refuse(text("kv_cache must be a (num_blocks, block_size, ", what, ") uint8 tensor"));
}

Tensor to_f32(const Tensor &t, const Tensor &like) {
    return t.scalar_type() == at::kFloat && t.device() == like.device() && t.is_contiguous() ? t : t.to(like.device(), at::kFloat).contiguous();
}

OptTensor rope_compress_store(const OptTensor &query, const Tensor &key, const Tensor &value, const Tensor &positions, const Tensor &cos_sin,
                              const Tensor &cache, const Tensor &slots, const Tensor &rot_even, const Tensor &rot_odd, const Tensor &k_bounds,
                              const Tensor &v_bounds, bool neox, const OptTensor &out_q, int64_t rot_block, bool dense3) {
    const Rope r(query, key, value, positions, cos_sin, slots, out_q);
    OnDevice(key).also(cache);
    check_bytes(cache, "total_bytes");
    if (cache.stride(2) != 1) refuse("the bytes of a slot must be contiguous");
    for (const Tensor *t : {&rot_even, &rot_odd})
        if (t->dim() != 2 || t->size(0) != r.D || t->size(1) != r.D / 2) refuse(text("rot_T_even and rot_T_odd must be (", r.D, ", ", r.D / 2, ")"));
    const c10::hip::HIPGuard guard(key.get_device());
    const Tensor even = to_f32(rot_even, key), odd = to_f32(rot_odd, key), kb = to_f32(k_bounds, key), vb = to_f32(v_bounds, key);
    r.call(rq_rope_compress_store, "rq_rope_compress_store", neox, (int)(dense3 ? RQ_INDEX_DENSE3 : RQ_INDEX_NIBBLE), slots.data_ptr<int64_t>(),
           cache.data_ptr<uint8_t>(), cache.size(0), count(cache.size(1)), cache.stride(0), cache.stride(1), count(cache.size(2)), even.data_ptr<float>(),
           odd.data_ptr<float>(), count(rot_block), kb.data_ptr<float>(), count(kb.numel()), vb.data_ptr<float>(), count(vb.numel()), stream_of(key));
    return r.out;
}

OptTensor rope_q8_store(const OptTensor &query, const Tensor &key, const Tensor &value, const Tensor &positions, const Tensor &cos_sin,
                        const Tensor &cache, const Tensor &slots, int64_t format, bool neox, const OptTensor &out_q, const OptTensor &workspace) {
    const Rope r(query, key, value, positions, cos_sin, slots, out_q);
    const OnDevice on(key);
    on.also(cache), on.also(workspace);
    check_bytes(cache, "q8_slot_bytes");
    if (cache.size(2) < r.H * (2 * r.D + 1))
        refuse(text("cache slots of ", cache.size(2), " bytes; ", r.H, " heads of ", r.D, " take ", (r.H * (2 * r.D + 1) + 7) / 8 * 8));
    if (cache.stride(2) != 1 || cache.stride(1) != cache.size(2)) refuse("the slots of a page must be contiguous");
    const c10::hip::HIPGuard guard(key.get_device());
    const Scratch ws(workspace, rq_q8_store_workspace_bytes(r.N, cache.size(0), count(cache.size(1))), key);
    r.call(rq_rope_q8_store, "rq_rope_q8_store", neox, count(format), slots.data_ptr<int64_t>(), cache.data_ptr<uint8_t>(), cache.size(0),
           count(cache.size(1)), cache.stride(0), ws.at, ws.bytes, stream_of(key));
    return r.out;
}

// ---- plain 16-bit pages ---------------------------------------------------------------
void check_pages(const Tensor &k, const Tensor &v, int64_t heads, int64_t head_dim) {
    if (k.dim() != 4 || !v.sizes().equals(k.sizes()) || v.scalar_type() != k.scalar_type())
        refuse("k_cache and v_cache must have the same (num_blocks, block_size, heads, head_dim) shape and dtype");
    if (k.size(2) != heads || k.size(3) != head_dim || k.stride(3) != 1 || v.stride(3) != 1)
        refuse(text("the pages must hold ", heads, " heads of ", head_dim, ", contiguous over head_dim"));
}

OptTensor rope_kv16_store(const OptTensor &query, const Tensor &key, const Tensor &value, const Tensor &positions, const Tensor &cos_sin,
                          const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots, bool neox, const OptTensor &out_q) {
    const Rope r(query, key, value, positions, cos_sin, slots, out_q);
    const OnDevice on(key);
    on.also(k_cache), on.also(v_cache);
    if (k_cache.scalar_type() != key.scalar_type()) refuse("the pages must be of " + name_of(key.scalar_type()) + ", as key is");
    check_pages(k_cache, v_cache, r.H, r.D);
    const c10::hip::HIPGuard guard(key.get_device());
    r.call(rq_rope_kv16_store, "rq_rope_kv16_store", neox, slots.data_ptr<int64_t>(), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.size(0),
           count(k_cache.size(1)), step(k_cache, 0), step(k_cache, 1), step(k_cache, 2), step(v_cache, 0), step(v_cache, 1), step(v_cache, 2),
           stream_of(key));
    return r.out;
}

// An int32 tensor, contiguous over its last dimension.
Tensor index_of(const Tensor &t, const char *name, int64_t dim) {
    if (t.scalar_type() != at::kInt || t.dim() != dim)
        refuse(text(name, " must be a ", dim, "-dimensional torch.int32 tensor, got ", t.dim(), " dimensions of ", name_of(t.scalar_type())));
    return t.is_contiguous() || t.stride(-1) == 1 ? t : t.contiguous();
}

Tensor kv16_attention(const Tensor &q_, const Tensor &k_cache, const Tensor &v_cache, const Tensor &block_table, const Tensor &seq_lens,
                      std::optional<double> sm_scale, bool causal, const OptTensor &cu_seqlens_q, std::optional<int64_t> max_q_len,
                      std::optional<int64_t> max_seq_len, const OptTensor &out_, const OptTensor &workspace) {
    const OnDevice on(q_);
    on.also(k_cache), on.also(v_cache), on.also(block_table), on.also(seq_lens), on.also(cu_seqlens_q), on.also(out_), on.also(workspace);
    const int64_t H = k_cache.dim() == 4 ? k_cache.size(2) : 0;
    if (q_.dim() != 3 || H < 1 || q_.size(1) % H != 0 || k_cache.scalar_type() != q_.scalar_type())
        refuse(text("q must be (tokens, a multiple of the pages' heads, head_dim) of the pages' dtype, got ", shape_of(q_), " of ", name_of(q_.scalar_type())));
    const int64_t T = q_.size(0), HQ = q_.size(1), D = q_.size(2);
    check_pages(k_cache, v_cache, H, D);
    const Tensor bt = index_of(block_table, "block_table", 2), sl = index_of(seq_lens, "seq_lens", 1);
    const int64_t B = sl.numel(), max_blocks = bt.size(1);
    if (bt.size(0) != B) refuse("block_table and seq_lens differ in the number of sequences");
    const c10::hip::HIPGuard guard(q_.get_device());
    Tensor cu;
    int64_t most = 1;
    if (cu_seqlens_q) {
        cu = index_of(*cu_seqlens_q, "cu_seqlens_q", 1);
        if (cu.numel() != B + 1) refuse(text("cu_seqlens_q must have ", B + 1, " entries, got ", cu.numel()));
        most = max_q_len ? std::min(*max_q_len, T) : T;
    } else if (T != B) {
        refuse(text(T, " query tokens and ", B, " sequences: cu_seqlens_q is needed"));
    }
    const Tensor q = q_.stride(2) == 1 ? q_ : q_.contiguous();
    Tensor out = out_ ? *out_ : at::empty(q.sizes(), q.options());
    if (!out.sizes().equals(q.sizes()) || out.scalar_type() != q.scalar_type() || out.stride(2) != 1)
        refuse("out must have q's shape and dtype and be contiguous over head_dim");
    const int64_t capacity = max_blocks * k_cache.size(1), longest = max_seq_len ? std::min(*max_seq_len, capacity) : capacity;
    const Scratch ws(workspace, rq_kv16_attention_workspace_bytes(B, count(HQ), count(H), count(D), most, longest), q);
    const float scale = sm_scale ? (float)*sm_scale : D > 0 ? (float)(1.0 / std::sqrt((double)D)) : 0.f;
    check_status(rq_kv16_attention(q.data_ptr(), dtype_code(q.scalar_type()), T, count(HQ), step(q, 0), step(q, 1),
                                   cu.defined() ? cu.data_ptr<int32_t>() : nullptr, B, most, causal ? 1 : 0, k_cache.data_ptr(), v_cache.data_ptr(),
                                   k_cache.size(0), count(k_cache.size(1)), step(k_cache, 0), step(k_cache, 1), step(k_cache, 2), step(v_cache, 0),
                                   step(v_cache, 1), step(v_cache, 2), count(H), count(D), bt.data_ptr<int32_t>(), max_blocks, bt.stride(0),
                                   sl.data_ptr<int32_t>(), longest, scale, out.data_ptr(), step(out, 0), step(out, 1), ws.at, ws.bytes, stream_of(q)),
                 "rq_kv16_attention");
    return out;
}

}  // namespace

PYBIND11_MODULE(_rq_torch, m) {
    m.def("rope_compress_store", &rope_compress_store);
    m.def("rope_q8_store", &rope_q8_store);
    m.def("rope_kv16_store", &rope_kv16_store);
    m.def("kv16_attention", &kv16_attention);
}
