// C ABI of what stands around attention in a decode step
// (include/onednn_flash_hip.h): rotary positions and appending to a cache.
// Argument checks, layout resolution.

#include <cmath>
#include <cstring>
#include <limits>

#include "serving_checks.h"

namespace {

int check_rotary(const ofh_rotary& r, size_t head_dim, ofh::Rotation& out) {
    if (head_dim == 0 || head_dim > (size_t)ofh::kRotaryMaxDim)
        return unsupported("head_dim must be at most " + std::to_string(ofh::kRotaryMaxDim));
    if (r.rotary_dim < 2 || r.rotary_dim % 2 != 0 || r.rotary_dim > head_dim)
        return invalid("rotary_dim must be even, from 2 to head_dim");
    if (r.frequencies == nullptr) return invalid("frequencies must be non-null");
    if ((uintptr_t)r.frequencies % sizeof(double) != 0) return invalid("frequencies must be aligned");
    if (!std::isfinite(r.magnitude)) return invalid("magnitude must be finite");
    out = ofh::Rotation{};
    out.freq = r.frequencies;
    out.R = (int)r.rotary_dim;
    out.interleaved = r.interleaved != 0;
    out.magnitude = r.magnitude;
    return OFH_SUCCESS;
}

int check_strides(const int64_t s[3], const char* name) {
    for (int i = 0; i < 3; ++i)
        if (s[i] < 0) return invalid(std::string(name) + " strides must be non-negative");
    return OFH_SUCCESS;
}

// A row read and its result: the same rows, or rows apart.
int check_rows(const void* x, const int64_t xs[3], const void* out, const int64_t os[3], int elem, const char* name) {
    if (x == nullptr || out == nullptr) return invalid(std::string(name) + " and its output must be non-null");
    if ((uintptr_t)x % (size_t)elem != 0 || (uintptr_t)out % (size_t)elem != 0)
        return unsupported(std::string(name) + " and its output must be aligned to their elements");
    if (x == out && std::memcmp(xs, os, 3 * sizeof(int64_t)) != 0)
        return invalid(std::string(name) + " turned in place must keep its strides");
    return OFH_SUCCESS;
}

}  // namespace

extern "C" {

void ofh_rotary_params_init(ofh_rotary_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
    p->rotary.magnitude = 1.0f;
}

int ofh_rotary_fwd(const ofh_rotary_params* p, const void* x, void* out, void* stream) {
    return guarded([&]() -> int {
        if (p == nullptr) return invalid("params must be non-null");
        if (p->struct_size != sizeof(*p))
            return invalid("ofh_rotary_params.struct_size mismatch (call ofh_rotary_params_init)");
        if (p->batch == 0 || p->heads == 0 || p->tokens == 0 || p->head_dim == 0)
            return invalid("rotary dimensions must be non-zero");
        if (!known_dtype(p->dtype)) return invalid("unknown dtype");
        if (p->batch > (size_t)kMaxTokens || p->heads > (size_t)kMaxTokens || p->tokens > (size_t)kMaxTokens)
            return unsupported("rotary dimensions exceed the 32-bit index range");
        ofh::RotaryArgs a{};
        if (int rc = check_rotary(p->rotary, p->head_dim, a.r)) return rc;
        if (p->positions != nullptr && p->lengths != nullptr) return invalid("either positions or lengths, not both");
        if (p->position_stride < 0) return invalid("position_stride must be non-negative");
        if (p->offset < std::numeric_limits<int32_t>::min() || p->offset > std::numeric_limits<int32_t>::max())
            return unsupported("offset exceeds the 32-bit index range");
        int64_t xs[3], os[3];
        resolve_strides(xs, p->x_strides, p->heads, p->tokens, p->head_dim);
        resolve_strides(os, p->o_strides, p->heads, p->tokens, p->head_dim);
        if (int rc = check_strides(xs, "x")) return rc;
        if (int rc = check_strides(os, "out")) return rc;
        if (int rc = check_rows(x, xs, out, os, elem_size(p->dtype), "x")) return rc;
        a.x = x;
        a.o = out;
        a.x_sb = xs[0]; a.x_sh = xs[1]; a.x_st = xs[2];
        a.o_sb = os[0]; a.o_sh = os[1]; a.o_st = os[2];
        a.B = (int)p->batch;
        a.H = (int)p->heads;
        a.T = (int)p->tokens;
        a.D = (int)p->head_dim;
        a.r.transpose = p->transpose != 0;
        a.positions = p->positions;
        a.pos_sb = p->position_stride;
        a.lengths = p->lengths;
        a.offset = p->offset;
        if (!ofh::rotary_fits(a)) return unsupported("rotary call exceeds the launch range");
        OFH_HIP_CHECK(ofh::launch_rotary(a, p->dtype, static_cast<hipStream_t>(stream)));
        return OFH_SUCCESS;
    });
}

void ofh_cache_append_params_init(ofh_cache_append_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
    ofh_cache_write_params_init(&p->cache);
    p->rotary.magnitude = 1.0f;
}

int ofh_cache_append(const ofh_cache_append_params* p, const void* k, const void* v, const void* q, void* k_pages,
                     void* v_pages, void* q_out, void* stream) {
    return guarded([&]() -> int {
        if (p == nullptr) return invalid("params must be non-null");
        if (p->struct_size != sizeof(*p))
            return invalid("ofh_cache_append_params.struct_size mismatch (call ofh_cache_append_params_init)");
        ofh::CacheAppendArgs a{};
        if (int rc = cache_write_args(&p->cache, k, v, k_pages, v_pages, a.w)) return rc;
        if (int rc = check_rotary(p->rotary, p->cache.head_dim, a.r)) return rc;
        if (p->heads > (size_t)kMaxTokens) return unsupported("cache dimensions exceed the 32-bit index range");
        const int es = elem_size(p->cache.dtype);
        if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_pages | (uintptr_t)v_pages) % (size_t)es != 0)
            return unsupported("cache pointers must be aligned to their elements");
        if (p->heads > 0) {
            int64_t qs[3], os[3];
            resolve_strides(qs, p->q_strides, p->heads, p->cache.tokens, p->cache.head_dim);
            resolve_strides(os, p->o_strides, p->heads, p->cache.tokens, p->cache.head_dim);
            if (int rc = check_strides(qs, "q")) return rc;
            if (int rc = check_strides(os, "q_out")) return rc;
            if (int rc = check_rows(q, qs, q_out, os, es, "q")) return rc;
            a.q = q;
            a.q_out = q_out;
            a.q_sb = qs[0]; a.q_sh = qs[1]; a.q_st = qs[2];
            a.o_sb = os[0]; a.o_sh = os[1]; a.o_st = os[2];
        }
        a.H = (int)p->heads;
        a.D = (int)p->cache.head_dim;
        a.Dv = (int)p->cache.value_dim;
        if (!ofh::cache_append_fits(a)) return unsupported("cache append exceeds the launch range");
        OFH_HIP_CHECK(ofh::launch_cache_append(a, p->cache.dtype, static_cast<hipStream_t>(stream)));
        return OFH_SUCCESS;
    });
}

}  // extern "C"
