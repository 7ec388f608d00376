// Writing new rows into the pages of a key-value cache, and copying pages.
// Both only move bytes: bound by reading and writing each once, or for a few
// rows by the launch.

#include "serving_kernels.h"

namespace ofh {
namespace {

constexpr int kCacheThreads = 256;

template <int W>
struct Chunk;
template <>
struct Chunk<16> {
    typedef unsigned int type __attribute__((ext_vector_type(4)));
};
template <>
struct Chunk<8> {
    typedef unsigned int type __attribute__((ext_vector_type(2)));
};
template <>
struct Chunk<4> {
    typedef unsigned int type;
};
template <>
struct Chunk<2> {
    typedef unsigned short type;
};

// A thread moves one W-byte chunk of a K or V row: consecutive threads take the
// chunks of a row, then the heads of a token (which is how a projection lays K
// and V out). W is the widest that every address allows.
template <int W>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheWriteArgs a, int k_chunks, int v_chunks) {
    using C = typename Chunk<W>::type;
    const int row_chunks = k_chunks + v_chunks;
    const int64_t item = (int64_t)blockIdx.x * kCacheThreads + threadIdx.x;
    const int64_t row = item / row_chunks;
    int c = (int)(item - row * row_chunks);
    const int64_t token = row / a.Hkv;
    const int h = (int)(row - token * a.Hkv);
    const int b = (int)(token / a.T), t = (int)(token - (int64_t)b * a.T);
    if (b >= a.B) return;
    const int count = a.counts != nullptr ? max(0, min(a.counts[b], a.T)) : a.T;
    if (t >= count) return;
    const int64_t pos = (int64_t)a.lengths[b] - count + t;
    const int64_t slot = pos >> a.page_shift;
    if (pos < 0 || slot >= a.max_pages) return;
    const int page = a.table[b * a.table_stride + slot];
    if ((unsigned)page >= (unsigned)a.num_pages) return;
    const int64_t in_page = pos & (((int64_t)1 << a.page_shift) - 1);
    if (c < k_chunks) {
        const char* src = (const char*)a.k + (b * a.k_sb + h * a.k_sh + t * a.k_st) * a.elem;
        char* dst = (char*)a.k_pages + (page * a.kp_sp + h * a.kp_sh + in_page * a.kp_st) * a.elem;
        *(C*)(dst + W * c) = *(const C*)(src + W * c);
    } else {
        c -= k_chunks;
        const char* src = (const char*)a.v + (b * a.v_sb + h * a.v_sh + t * a.v_st) * a.elem;
        char* dst = (char*)a.v_pages + (page * a.vp_sp + h * a.vp_sh + in_page * a.vp_st) * a.elem;
        *(C*)(dst + W * c) = *(const C*)(src + W * c);
    }
}

template <int W>
hipError_t launch_write(const CacheWriteArgs& a, hipStream_t s) {
    const int kc = a.k_bytes / W, vc = a.v_bytes / W;
    const int64_t items = (int64_t)a.B * a.T * a.Hkv * (kc + vc);
    const int64_t wgs = (items + kCacheThreads - 1) / kCacheThreads;
    if (!grid_fits(wgs, kCacheThreads)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((cache_write_kernel<W>), dim3((unsigned)wgs), dim3(kCacheThreads), 0, s, a, kc, vc);
    return hipGetLastError();
}

// A workgroup copies kPart bytes of one page of one pool, four chunks per
// thread in flight.
constexpr int kUnroll = 4;
template <int W>
constexpr int part_bytes() {
    return W * kUnroll * kCacheThreads;
}

template <int W>
__global__ __launch_bounds__(kCacheThreads) void copy_pages_kernel(CopyPagesArgs a, int parts) {
    using C = typename Chunk<W>::type;
    const unsigned part = blockIdx.x % parts, rest = blockIdx.x / parts;
    const unsigned pool = rest % a.num_pools, pair = rest / a.num_pools;
    const char* src = a.pools[pool] + a.src[pair] * a.page_stride;
    char* dst = a.pools[pool] + a.dst[pair] * a.page_stride;
    const int64_t first = (int64_t)part * part_bytes<W>() + W * threadIdx.x;
    C x[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t at = first + i * W * kCacheThreads;
        if (at < a.page_bytes) x[i] = *(const C*)(src + at);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t at = first + i * W * kCacheThreads;
        if (at < a.page_bytes) *(C*)(dst + at) = x[i];
    }
}

template <int W>
hipError_t launch_copy(const CopyPagesArgs& a, hipStream_t s) {
    const int64_t parts = (a.page_bytes + part_bytes<W>() - 1) / part_bytes<W>();
    const int64_t wgs = parts * a.num_pools * a.num_pairs;
    if (!grid_fits(wgs, kCacheThreads)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((copy_pages_kernel<W>), dim3((unsigned)wgs), dim3(kCacheThreads), 0, s, a, (int)parts);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_write(const CacheWriteArgs& a, hipStream_t s) {
    const int64_t strides = a.k_sb | a.k_sh | a.k_st | a.v_sb | a.v_sh | a.v_st | a.kp_sp | a.kp_sh | a.kp_st |
                            a.vp_sp | a.vp_sh | a.vp_st;
    const uint64_t all = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages |
                         (uint64_t)(strides * a.elem) | (uint64_t)a.k_bytes | (uint64_t)a.v_bytes;
    if (all % 16 == 0) return launch_write<16>(a, s);
    if (all % 8 == 0) return launch_write<8>(a, s);
    if (all % 4 == 0) return launch_write<4>(a, s);
    return launch_write<2>(a, s);
}

hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t s) {
    uint64_t all = (uint64_t)a.page_stride | (uint64_t)a.page_bytes;
    for (int i = 0; i < a.num_pools; ++i) all |= (uintptr_t)a.pools[i];
    if (all % 16 == 0) return launch_copy<16>(a, s);
    if (all % 4 == 0) return launch_copy<4>(a, s);
    return launch_copy<2>(a, s);
}

}  // namespace ofh
