// What the translation units of the serving entries check and fill in alike.
// Internal header, included once per translation unit.
#pragma once

#include "onednn_flash_hip.h"

#include <hip/hip_runtime.h>

#include <string>

#include "capi_shared.h"
#include "serving_kernels.h"

namespace {

#define OFH_HIP_CHECK(expr)                                                                   \
    do {                                                                                      \
        const hipError_t e_ = (expr);                                                         \
        if (e_ != hipSuccess)                                                                 \
            return ofh::api_error(OFH_ERROR_HIP, std::string(#expr " failed: ") + hipGetErrorString(e_)); \
    } while (0)

inline int invalid(const std::string& msg) { return ofh::api_error(OFH_ERROR_INVALID_ARGUMENT, msg); }
inline int unsupported(const std::string& msg) { return ofh::api_error(OFH_ERROR_UNSUPPORTED, msg); }

constexpr int64_t kMaxTokens = (int64_t)1 << 30;  // of a sequence; positions and keys are 32-bit
constexpr int64_t kMaxOffset = ((int64_t)1 << 31) - 1;

inline int elem_size(int dtype) { return dtype == OFH_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype >= OFH_DTYPE_F32 && dtype <= OFH_DTYPE_F16; }

// All-zero strides mean a contiguous [A, B, T, last] tensor.
inline void resolve_strides(int64_t out[3], const int64_t in[3], size_t b, size_t t, size_t last) {
    const bool none = in[0] == 0 && in[1] == 0 && in[2] == 0;
    out[0] = none ? (int64_t)(b * t * last) : in[0];
    out[1] = none ? (int64_t)(t * last) : in[1];
    out[2] = none ? (int64_t)last : in[2];
}

// The pool's geometry, as both paged_attention and cache_write ask.
inline int check_pages(size_t num_pages, size_t page_size, size_t max_pages, int64_t table_stride, const int32_t* table,
                const int32_t* lengths, bool check_ptrs) {
    if (num_pages == 0 || max_pages == 0) return invalid("num_pages and max_pages must be non-zero");
    if (page_size < (size_t)ofh::kStreamKeys || (page_size & (page_size - 1)) != 0)
        return unsupported("page_size must be a power of two, 16 or more");
    if (num_pages > (size_t)kMaxOffset || page_size > (size_t)kMaxTokens || max_pages > (size_t)kMaxTokens ||
        max_pages * page_size > (size_t)kMaxTokens)
        return unsupported("pages exceed the 32-bit index range (2^30 tokens per sequence)");
    if (table_stride < 0) return invalid("table_stride must be non-negative");
    if (check_ptrs && (table == nullptr || lengths == nullptr)) return invalid("page_table and lengths must be non-null");
    return OFH_SUCCESS;
}

inline int log2_of(size_t n) {
    int s = 0;
    while (((size_t)1 << s) < n) ++s;
    return s;
}

// Checks a call that writes new rows into pages and fills its arguments.
inline int cache_write_args(const ofh_cache_write_params* p, const void* k, const void* v, void* k_pages, void* v_pages,
                            ofh::CacheWriteArgs& a) {
    if (p == nullptr) return invalid("params must be non-null");
    if (p->struct_size != sizeof(*p))
        return invalid("ofh_cache_write_params.struct_size mismatch (call ofh_cache_write_params_init)");
    if (p->batch == 0 || p->kv_heads == 0 || p->tokens == 0 || p->head_dim == 0 || p->value_dim == 0)
        return invalid("cache dimensions must be non-zero");
    if (!known_dtype(p->dtype)) return invalid("unknown dtype");
    if (p->batch > (size_t)kMaxTokens || p->kv_heads > (size_t)kMaxTokens || p->tokens > (size_t)kMaxTokens ||
        p->head_dim > ((size_t)1 << 20) || p->value_dim > ((size_t)1 << 20))
        return unsupported("cache dimensions exceed the 32-bit index range");
    if (int rc = check_pages(p->num_pages, p->page_size, p->max_pages, p->table_stride, p->page_table, p->lengths,
                             true))
        return rc;
    if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr)
        return invalid("cache pointers must be non-null");
    int64_t ks[3], vs[3], kp[3], vp[3];
    resolve_strides(ks, p->k_strides, p->kv_heads, p->tokens, p->head_dim);
    resolve_strides(vs, p->v_strides, p->kv_heads, p->tokens, p->value_dim);
    resolve_strides(kp, p->k_page_strides, p->kv_heads, p->page_size, p->head_dim);
    resolve_strides(vp, p->v_page_strides, p->kv_heads, p->page_size, p->value_dim);
    for (const int64_t* s : {ks, vs, kp, vp})
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0) return invalid("cache strides must be non-negative");
    a = ofh::CacheWriteArgs{};
    a.k = k;
    a.v = v;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.k_sb = ks[0]; a.k_sh = ks[1]; a.k_st = ks[2];
    a.v_sb = vs[0]; a.v_sh = vs[1]; a.v_st = vs[2];
    a.kp_sp = kp[0]; a.kp_sh = kp[1]; a.kp_st = kp[2];
    a.vp_sp = vp[0]; a.vp_sh = vp[1]; a.vp_st = vp[2];
    a.table = p->page_table;
    a.table_stride = p->table_stride != 0 ? p->table_stride : (int64_t)p->max_pages;
    a.num_pages = (int)p->num_pages;
    a.page_shift = log2_of(p->page_size);
    a.max_pages = (int)p->max_pages;
    a.lengths = p->lengths;
    a.counts = p->counts;
    a.B = (int)p->batch;
    a.Hkv = (int)p->kv_heads;
    a.T = (int)p->tokens;
    a.elem = elem_size(p->dtype);
    a.k_bytes = (int)p->head_dim * a.elem;
    a.v_bytes = (int)p->value_dim * a.elem;
    return OFH_SUCCESS;
}

// No C++ exception (a message that finds no memory) leaves the C ABI.
template <typename F>
int guarded(F&& body) {
    try {
        return body();
    } catch (...) {
        return OFH_ERROR_HIP;
    }
}

}  // namespace
