// Writing new rows into the pages of a key-value cache, and copying pages.
// Both only move bytes: bound by reading and writing each once (1700 pages of 32 KB in
// four pools 91 us, 4.9 TB/s; a copy of 1 GiB reaches 5.1), or for a few
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

// A workgroup takes TOKENS tokens, so that their place (length, count, page) is
// three scalar loads; its threads take the W-byte chunks of a token's K and V rows
// of all heads. W is the widest that every address allows. A workgroup per token
// spreads a decode step's few; four have their loads in flight together: 8
// prompts (93 MB) 30.4 -> 21.8 us (4.3 TB/s), a step of 64 sequences 2.9 us.
template <int W, int TOKENS>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheWriteArgs a, unsigned k_chunks, unsigned v_chunks) {
    using C = typename Chunk<W>::type;
    const unsigned row_chunks = k_chunks + v_chunks, chunks = row_chunks * (unsigned)a.Hkv;
    const unsigned blocks = (chunks + kCacheThreads - 1) / kCacheThreads;  // workgroups of a token
    const unsigned group = blockIdx.x / blocks, chunk = (blockIdx.x - group * blocks) * kCacheThreads + threadIdx.x;
    const unsigned h = chunk / row_chunks;
    unsigned c = chunk - h * row_chunks;
    const bool is_v = c >= k_chunks;
    if (is_v) c -= k_chunks;
    const char* src = (const char*)(is_v ? a.v : a.k) + (h * (is_v ? a.v_sh : a.k_sh)) * a.elem + (uint64_t)W * c;
    char* dst = (char*)(is_v ? a.v_pages : a.k_pages) + (h * (is_v ? a.vp_sh : a.kp_sh)) * a.elem + (uint64_t)W * c;
    C x[TOKENS];
    int64_t to[TOKENS];  // byte offset, -1: not written
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        to[i] = -1;
        const int64_t token = (int64_t)group * TOKENS + i;
        if (token >= (int64_t)a.B * a.T) continue;
        const int b = (int)((unsigned)token / (unsigned)a.T), t = (int)(token - (int64_t)b * a.T);
        const int count = a.counts != nullptr ? max(0, min(a.counts[b], a.T)) : a.T;
        if (t >= count) continue;
        const int64_t pos = (int64_t)a.lengths[b] - count + t;
        const int64_t slot = pos >> a.page_shift;
        if (pos < 0 || slot >= a.max_pages) continue;
        const int page = a.table[b * a.table_stride + slot];
        if ((unsigned)page >= (unsigned)a.num_pages) continue;
        const int64_t row = pos & (((int64_t)1 << a.page_shift) - 1);
        to[i] = (is_v ? page * a.vp_sp + row * a.vp_st : page * a.kp_sp + row * a.kp_st) * a.elem;
        if (chunk < chunks) x[i] = *(const C*)(src + (is_v ? b * a.v_sb + t * a.v_st : b * a.k_sb + t * a.k_st) * a.elem);
    }
#pragma unroll
    for (int i = 0; i < TOKENS; ++i)
        if (to[i] >= 0 && chunk < chunks) *(C*)(dst + to[i]) = x[i];
}

// The widest chunk that every address allows.
int write_chunk(const CacheWriteArgs& a) {
    const int64_t strides = a.k_sb | a.k_sh | a.k_st | a.v_sb | a.v_sh | a.v_st | a.kp_sp | a.kp_sh | a.kp_st |
                            a.vp_sp | a.vp_sh | a.vp_st;
    const uint64_t all = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages |
                         (uint64_t)(strides * a.elem) | (uint64_t)a.k_bytes | (uint64_t)a.v_bytes;
    return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// Workgroups of a call, and whether each takes four tokens (0: past what a launch holds).
int64_t write_grid(const CacheWriteArgs& a, bool& many) {
    const int w = write_chunk(a);
    const int64_t tokens = (int64_t)a.B * a.T, chunks = (int64_t)a.Hkv * (a.k_bytes / w + a.v_bytes / w);
    const int64_t blocks = (chunks + kCacheThreads - 1) / kCacheThreads;
    // (chunks of a token, tokens and workgroups are 32-bit in the kernel)
    if (chunks >= ((int64_t)1 << 31) || tokens >= ((int64_t)1 << 32)) return 0;
    many = tokens * blocks >= 16 * kComputeUnits;
    const int64_t wgs = (many ? (tokens + 3) / 4 : tokens) * blocks;
    return grid_fits(wgs, kCacheThreads) ? wgs : 0;
}

template <int W>
hipError_t launch_write(const CacheWriteArgs& a, hipStream_t s) {
    const int kc = a.k_bytes / W, vc = a.v_bytes / W;
    bool many = false;
    const int64_t wgs = write_grid(a, many);
    if (wgs == 0) return hipErrorInvalidValue;
    if (many) hipLaunchKernelGGL((cache_write_kernel<W, 4>), dim3((unsigned)wgs), dim3(kCacheThreads), 0, s, a, kc, vc);
    else hipLaunchKernelGGL((cache_write_kernel<W, 1>), dim3((unsigned)wgs), dim3(kCacheThreads), 0, s, a, kc, vc);
    return hipGetLastError();
}

// A workgroup copies one part of one page of one pool, four chunks per thread in
// flight. The pools and the pairs come with the launch: nothing is uploaded.
constexpr int kUnroll = 4;
template <int W>
constexpr int part_bytes() {
    return W * kUnroll * kCacheThreads;
}

template <int W>
__global__ __launch_bounds__(kCacheThreads) void copy_pages_kernel(CopyPagesArgs a, unsigned parts) {
    using C = typename Chunk<W>::type;
    const unsigned rest = blockIdx.x / parts, part = blockIdx.x - rest * parts;
    const unsigned pair = rest / (unsigned)a.num_pools, pool = rest - pair * (unsigned)a.num_pools;
    char* base = (char*)(uintptr_t)(((uint64_t)a.words[2 * pool + 1] << 32) | a.words[2 * pool]);
    const uint32_t* pairs = a.words + 2 * a.num_pools;
    const int64_t from = a.wide ? pairs[2 * pair] : pairs[pair] & 0xffffu;
    const int64_t to = a.wide ? pairs[2 * pair + 1] : pairs[pair] >> 16;
    const char* src = base + from * a.page_stride;
    char* dst = base + to * a.page_stride;
    const int64_t first = (int64_t)part * part_bytes<W>() + W * threadIdx.x;
    C x[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t at = first + i * W * kCacheThreads;
        if (at < a.page_bytes) x[i] = __builtin_nontemporal_load((const C*)(src + at));
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t at = first + i * W * kCacheThreads;
        if (at < a.page_bytes) __builtin_nontemporal_store(x[i], (C*)(dst + at));
    }
}

template <int W>
hipError_t launch_copy(const CopyPagesArgs& a, hipStream_t s) {
    const int64_t parts = (a.page_bytes + part_bytes<W>() - 1) / part_bytes<W>();
    const int64_t wgs = parts * a.num_pools * a.num_pairs;
    if (!grid_fits(wgs, kCacheThreads)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((copy_pages_kernel<W>), dim3((unsigned)wgs), dim3(kCacheThreads), 0, s, a, (unsigned)parts);
    return hipGetLastError();
}

}  // namespace

bool cache_write_fits(const CacheWriteArgs& a) {
    bool many = false;
    return write_grid(a, many) > 0;
}

hipError_t launch_cache_write(const CacheWriteArgs& a, hipStream_t s) {
    switch (write_chunk(a)) {
        case 16: return launch_write<16>(a, s);
        case 8: return launch_write<8>(a, s);
        case 4: return launch_write<4>(a, s);
        default: return launch_write<2>(a, s);
    }
}

hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t s) {
    uint64_t all = (uint64_t)a.page_stride | (uint64_t)a.page_bytes;
    for (int i = 0; i < a.num_pools; ++i) all |= a.words[2 * i];
    if (all % 16 == 0) return launch_copy<16>(a, s);
    if (all % 4 == 0) return launch_copy<4>(a, s);
    return launch_copy<2>(a, s);
}

}  // namespace ofh
