// binding.cpp -- the Python side of the 4-bit and cache operators
// (mxfp4.py, kv_cache.py): argument checks, output allocation and the call into
// the C ABI, on the current stream of the tensors' device.
//
// These operators are called once a layer on a few rows, where a call costs
// the host more than the GPU: the same checks and allocations in Python with
// ctypes took 9 to 19 us a call.  The library itself is still loaded by
// _capi.lib(); bind() takes its entries' addresses, and the function that turns
// a status code into an exception.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "../../include/mxfp4.h"
#include "../../include/mxfp8_cache.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Api {
    decltype(&mxfp4_quantize) fp4_quantize;
    decltype(&mxfp4_dequantize) fp4_dequantize;
    decltype(&mxfp4_gemm) fp4_gemm;
    decltype(&mxfp8_cache_write) cache_write;
    decltype(&mxfp8_cache_read) cache_read;
    decltype(&mxfp8_cache_attention_workspace) attention_workspace;
    decltype(&mxfp8_cache_attention) attention;
    py::object* check;  // check(code, context) raises; lives as long as the process
};
Api api;

void bind(const py::dict& entries, const py::object& check) {
    auto at = [&](const char* name) { return reinterpret_cast<void*>(entries[name].cast<uintptr_t>()); };
    api.fp4_quantize = reinterpret_cast<decltype(api.fp4_quantize)>(at("mxfp4_quantize"));
    api.fp4_dequantize = reinterpret_cast<decltype(api.fp4_dequantize)>(at("mxfp4_dequantize"));
    api.fp4_gemm = reinterpret_cast<decltype(api.fp4_gemm)>(at("mxfp4_gemm"));
    api.cache_write = reinterpret_cast<decltype(api.cache_write)>(at("mxfp8_cache_write"));
    api.cache_read = reinterpret_cast<decltype(api.cache_read)>(at("mxfp8_cache_read"));
    api.attention_workspace = reinterpret_cast<decltype(api.attention_workspace)>(at("mxfp8_cache_attention_workspace"));
    api.attention = reinterpret_cast<decltype(api.attention)>(at("mxfp8_cache_attention"));
    if (!api.check) api.check = new py::object(check);
}

// The C call without the GIL (a full launch queue blocks); its error raised.
template <typename F>
void call(const char* context, F f) {
    int rc;
    {
        py::gil_scoped_release release;
        rc = f();
    }
    if (rc != MXFP8_OK) (*api.check)(rc, context);
}


void same_device(const Tensor& first, const Tensor& t) {
    TORCH_CHECK_VALUE(t.device() == first.device(), "all tensors must be on ", first.device(), ", got one on ", t.device());
}
void same_device(const Tensor& first, const OptTensor& t) {
    if (t) same_device(first, *t);
}

template <typename... T>
void* enter(c10::cuda::OptionalCUDAGuard& guard, const Tensor& first, const T&... others) {
    TORCH_CHECK_VALUE(first.is_cuda(), "the operator runs on CUDA tensors, got one on ", first.device());
    (same_device(first, others), ...);
    guard.set_device(first.device());
    return c10::cuda::getCurrentCUDAStream(first.device().index()).stream();
}

// A new contiguous tensor beside t, from torch's allocator without the way
// through its dispatcher.
Tensor new_empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& t) {
    return at::detail::empty_cuda(sizes, type, t.device(), std::nullopt);
}

int in_dtype(const char* name, const Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return MXFP8_BF16;
    if (t.scalar_type() == at::kHalf) return MXFP8_FP16;
    TORCH_CHECK_VALUE(false, name, " must be torch.bfloat16 or torch.float16, got ", t.scalar_type());
}

int out_dtype(at::ScalarType type) {
    switch (type) {
        case at::kFloat: return MXFP8_F32;
        case at::kBFloat16: return MXFP8_BF16;
        case at::kHalf: return MXFP8_FP16;
        default: TORCH_CHECK_VALUE(false, "out_dtype must be torch.float32, torch.bfloat16 or torch.float16");
    }
}

// ---------------------------------------------------------------------------
// MXFP4
// ---------------------------------------------------------------------------

struct Payload {
    int64_t rows, cols, ld;
};

// Row stride; a single row's own means nothing, and may be any number.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

Payload payload(const char* name, const Tensor& q) {
    const auto type = q.scalar_type();
    TORCH_CHECK_VALUE(q.dim() == 2 && (type == at::kByte || type == at::kChar || type == at::kFloat4_e2m1fn_x2) &&
                          (q.stride(1) == 1 || q.size(1) <= 1),
                      name, " must be a row-major matrix of bytes, got ", q.sizes(), " ", type);
    TORCH_CHECK_VALUE(q.size(1) % 16 == 0, name, " must have a multiple of 32 columns (16 bytes), got ", 2 * q.size(1));
    return Payload{q.size(0), 2 * q.size(1), row_stride(q)};
}

// The library checks the size.
void check_scales(const char* name, const Tensor& s) {
    TORCH_CHECK_VALUE(s.element_size() == 1 && s.is_contiguous(), name, " must be a contiguous buffer of bytes");
}

std::tuple<Tensor, Tensor> quantize_mxfp4(const Tensor& x_in, const OptTensor& q_in, const OptTensor& s_in) {
    Tensor x = x_in;
    TORCH_CHECK_VALUE(x.dim() == 2, "X must be 2-D, got shape ", x.sizes());
    const int code = in_dtype("X", x);
    const int64_t m = x.size(0), k = x.size(1), q_cols = (k + 31) / 32 * 32;
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, x, q_in, s_in);
    if ((x.stride(1) != 1 && k > 1) || (m > 1 && x.stride(0) < k)) x = x.contiguous();
    Tensor q = q_in ? *q_in : new_empty({m, q_cols / 2}, at::kByte, x);
    if (q_in) {
        const Payload p = payload("q", q);
        TORCH_CHECK_VALUE(p.rows == m && p.cols == q_cols, "q must be (", m, ", ", q_cols / 2, ") bytes, got ", q.sizes());
    }
    Tensor s = s_in ? *s_in : new_empty({(m + 127) / 128 * 128 * ((q_cols + 127) / 128 * 4)}, at::kByte, x);
    if (s_in) check_scales("s", s);
    const int64_t ld_x = row_stride(x), ld_q = row_stride(q), s_bytes = s.numel();
    call("MXFP4 quantizer launch", [&] {
        return api.fp4_quantize(x.data_ptr(), code, m, k, ld_x, q.data_ptr(), ld_q, s.data_ptr(), s_bytes, stream);
    });
    return {q, s};
}

Tensor dequantize_mxfp4(const Tensor& q, const Tensor& s, at::ScalarType type) {
    const Payload p = payload("q", q);
    check_scales("s", s);
    const int code = out_dtype(type);
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, q, s);
    Tensor out = new_empty({p.rows, p.cols}, type, q);
    call("MXFP4 dequantizer launch", [&] {
        return api.fp4_dequantize(q.data_ptr(), p.rows, p.cols, p.ld, s.data_ptr(), s.numel(), out.data_ptr(), code,
                                  p.cols, stream);
    });
    return out;
}

Tensor gemm_mxfp4(const Tensor& a_q, const Tensor& b_q, const Tensor& a_s, const Tensor& b_s, at::ScalarType type,
                  const OptTensor& out_in) {
    const Payload a = payload("a_q", a_q), b = payload("b_q", b_q);
    TORCH_CHECK_VALUE(a.cols == b.cols, "a_q and b_q must have the same number of columns, got ", a.cols, " and ", b.cols);
    check_scales("a_s", a_s);
    check_scales("b_s", b_s);
    if (out_in) {
        const Tensor& o = *out_in;
        TORCH_CHECK_VALUE(o.dim() == 2 && o.size(0) == a.rows && o.size(1) == b.rows && (o.stride(1) == 1 || b.rows <= 1),
                          "out must be a row-major (", a.rows, ", ", b.rows, ") matrix, got ", o.sizes());
        type = o.scalar_type();
    }
    const int code = out_dtype(type);
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, a_q, b_q, a_s, b_s, out_in);
    Tensor out = out_in ? *out_in : new_empty({a.rows, b.rows}, type, a_q);
    const int64_t ld_out = row_stride(out);
    call("MXFP4 product launch", [&] {
        return api.fp4_gemm(a_q.data_ptr(), a.rows, a.ld, a_s.data_ptr(), a_s.numel(), b_q.data_ptr(), b.rows, b.ld,
                            b_s.data_ptr(), b_s.numel(), a.cols, out.data_ptr(), code, ld_out, stream);
    });
    return out;
}

// ---------------------------------------------------------------------------
// the cache
// ---------------------------------------------------------------------------

mxfp8_cache describe(const Tensor& k, const Tensor& v, const Tensor& k_scales, const Tensor& v_scales) {
    auto e4m3 = [](const Tensor& t) {  // or its bytes; another 8-bit format would be misread
        return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte || t.scalar_type() == at::kChar;
    };
    TORCH_CHECK_VALUE(k.dim() == 4 && e4m3(k) && e4m3(v) && v.sizes() == k.sizes(),
                      "k and v must be (num_pages, heads, page_size, dim) float8_e4m3fn or bytes, got ", k.sizes(), " ",
                      k.scalar_type(), " and ", v.sizes(), " ", v.scalar_type());
    const int64_t dim = k.size(3);
    for (const Tensor* s : {&k_scales, &v_scales}) {
        TORCH_CHECK_VALUE(dim % 32 == 0 && s->dim() == 4 && s->size(0) == k.size(0) && s->size(1) == k.size(1) &&
                              s->size(2) == k.size(2) && s->size(3) == dim / 32,
                          "the scales must be (num_pages, heads, page_size, dim / 32) for dim a multiple of 32, got ",
                          s->sizes(), " beside ", k.sizes());
        TORCH_CHECK_VALUE(s->element_size() == 1, "the scales must be bytes");
    }
    TORCH_CHECK_VALUE(k.is_contiguous() && v.is_contiguous() && k_scales.is_contiguous() && v_scales.is_contiguous(),
                      "the cache's buffers must be contiguous");
    constexpr int64_t kMost = 2147483647;
    TORCH_CHECK_VALUE(k.size(1) <= kMost && k.size(2) <= kMost && dim <= kMost, "the cache's sizes are out of range");
    return mxfp8_cache{k.data_ptr(),   v.data_ptr(),       k_scales.data_ptr(), v_scales.data_ptr(),
                       k.size(0),      (int32_t)k.size(1), (int32_t)k.size(2),  (int32_t)dim};
}

void check_index(const char* name, const Tensor& t, at::ScalarType type, int64_t dims) {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == dims && (t.stride(-1) == 1 || t.size(-1) <= 1), name,
                      " must be a ", dims, "-D ", type == at::kInt ? "int32" : "int64",
                      " tensor with a contiguous last dimension, got ", t.sizes(), " ", t.scalar_type());
}

void check_rows(const char* name, const Tensor& t, int64_t heads, int64_t dim) {
    TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == dim && (heads < 0 || t.size(1) == heads), name, " must be (rows, ",
                      heads < 0 ? std::string("heads") : std::to_string(heads), ", ", dim, "), got ", t.sizes());
}

// t with a contiguous last dimension.
Tensor rows(const Tensor& t) { return t.stride(2) == 1 ? t : t.contiguous(); }

int64_t table_stride(const Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

const int32_t* int32s(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

void cache_write(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& k_in,
                 const Tensor& v_in, const Tensor& slots) {
    const mxfp8_cache c = describe(ck, cv, cks, cvs);
    check_rows("k", k_in, c.heads, c.dim);
    check_rows("v", v_in, c.heads, c.dim);
    check_index("slots", slots, at::kLong, 1);
    const int64_t tokens = k_in.size(0);
    TORCH_CHECK_VALUE(v_in.size(0) == tokens && slots.size(0) == tokens && v_in.scalar_type() == k_in.scalar_type(),
                      "k, v and slots must have the same number of tokens and k and v one type, got ", k_in.sizes(), " ",
                      k_in.scalar_type(), ", ", v_in.sizes(), " ", v_in.scalar_type(), ", ", slots.sizes());
    const int code = in_dtype("k", k_in);
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, k_in, v_in, slots, ck, cv, cks, cvs);
    const Tensor k = rows(k_in), v = rows(v_in);
    call("cache write launch", [&] {
        return api.cache_write(&c, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), code,
                               tokens, static_cast<const int64_t*>(slots.data_ptr()), stream);
    });
}

std::tuple<Tensor, Tensor> cache_read(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs,
                                      const Tensor& table, const Tensor& starts, int64_t total, at::ScalarType type,
                                      const OptTensor& k_given, const OptTensor& v_given) {
    const mxfp8_cache c = describe(ck, cv, cks, cvs);
    check_index("page_table", table, at::kInt, 2);
    check_index("starts", starts, at::kInt, 1);
    const int64_t batch = table.size(0);
    TORCH_CHECK_VALUE(starts.size(0) == batch + 1, "starts must have batch + 1 = ", batch + 1, " values, got ",
                      starts.size(0));
    TORCH_CHECK_VALUE(total >= 0, "total must be >= 0, got ", total);
    if (k_given || v_given) {  // both are written: one alone is refused
        for (const OptTensor* t : {&k_given, &v_given})
            TORCH_CHECK_VALUE(k_given && *t && (*t)->dim() == 3 && (*t)->size(0) == total && (*t)->size(1) == c.heads &&
                                  (*t)->size(2) == c.dim && (*t)->is_contiguous() &&
                                  (*t)->scalar_type() == k_given->scalar_type(),
                              "out must be a pair of contiguous (", total, ", ", c.heads, ", ", c.dim,
                              ") tensors of one type");
        type = k_given->scalar_type();
    }
    const int code = out_dtype(type);
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, table, starts, ck, cv, cks, cvs, k_given, v_given);
    Tensor k = k_given ? *k_given : new_empty({total, c.heads, c.dim}, type, table);
    Tensor v = v_given ? *v_given : new_empty({total, c.heads, c.dim}, type, table);
    call("cache read launch", [&] {
        return api.cache_read(&c, int32s(table), table_stride(table), table.size(1), batch, int32s(starts), total,
                              k.data_ptr(), v.data_ptr(), code, stream);
    });
    return {k, v};
}

std::tuple<Tensor, OptTensor> cache_attention(const Tensor& q_in, const Tensor& ck, const Tensor& cv, const Tensor& cks,
                                              const Tensor& cvs, const Tensor& table, const Tensor& lengths,
                                              std::optional<double> scale, bool return_lse) {
    const mxfp8_cache c = describe(ck, cv, cks, cvs);
    check_rows("q", q_in, -1, c.dim);
    check_index("page_table", table, at::kInt, 2);
    check_index("lengths", lengths, at::kInt, 1);
    const int64_t batch = q_in.size(0), q_heads = q_in.size(1);
    TORCH_CHECK_VALUE(table.size(0) == batch && lengths.size(0) == batch,
                      "page_table and lengths must have q's batch of ", batch, ", got ", table.sizes(), " and ",
                      lengths.sizes());
    TORCH_CHECK_VALUE(q_heads >= 1 && c.heads >= 1 && q_heads % c.heads == 0, "q must have a multiple of the cache's ",
                      c.heads, " heads, got ", q_heads);
    TORCH_CHECK_VALUE((c.dim == 64 || c.dim == 128 || c.dim == 192 || c.dim == 256) && c.page_size >= 2,
                      "attention needs dim 64, 128, 192 or 256 and page_size >= 2, got ", c.dim, " and ", c.page_size);
    const int code = in_dtype("q", q_in);
    c10::cuda::OptionalCUDAGuard guard;
    void* stream = enter(guard, q_in, table, lengths, ck, cv, cks, cvs);
    const Tensor q = rows(q_in);
    Tensor out = new_empty({batch, q_heads, c.dim}, q.scalar_type(), q);
    OptTensor lse;
    if (return_lse) lse = new_empty({batch, q_heads}, at::kFloat, q);
    int64_t size = 0;
    call("cache attention workspace", [&] {
        size = api.attention_workspace(&c, batch, q_heads);
        return size < 0 ? (int)size : MXFP8_OK;
    });
    // scratch of this call: its memory may serve others once the stream has passed it
    Tensor workspace = new_empty({size}, at::kByte, q);
    const float factor = (float)(scale ? *scale : 1.0 / std::sqrt((double)c.dim));
    call("cache attention launch", [&] {
        return api.attention(&c, q.data_ptr(), q.stride(0), q.stride(1), code, batch, q_heads, int32s(table),
                             table_stride(table), table.size(1), int32s(lengths), factor, out.data_ptr(),
                             lse ? static_cast<float*>(lse->data_ptr()) : nullptr, workspace.data_ptr(), size, stream);
    });
    return {out, lse};
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    m.def("bind", &bind);
    m.def("quantize_mxfp4", &quantize_mxfp4);
    m.def("dequantize_mxfp4", &dequantize_mxfp4);
    m.def("mxfp4_gemm", &gemm_mxfp4);
    m.def("cache_write", &cache_write);
    m.def("cache_read", &cache_read);
    m.def("cache_attention", &cache_attention);
}
