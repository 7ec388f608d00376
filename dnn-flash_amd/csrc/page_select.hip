// Selection of pages by a cheap score: the bounds of a page's keys, the scores of
// a sequence's pages for a token, and the choice of the highest.
//
// Score of a page for a token and key-value head, an upper bound of q.k over the
// page's keys k when q is a head of its group:
//     max over the group's heads of sum_d q_d (q_d > 0 ? hi_d : lo_d),
// hi and lo the columns' largest and smallest values in the page. The sum is
// formed in 64 bits and rounded to fp32. Products of 16-bit numbers are exact there
// (bf16 16 bits, fp16 22), and so are sums of up to 256 while the products' exponents
// lie within 29 (bf16) or 23 (fp16) of each other: their order then decides nothing.
// Otherwise, and in fp32, another order moves the last of the sum's 64-bit digits, and
// a score, a tie or a rank only where the sum is that near to the middle between two
// fp32 numbers.

#include <algorithm>
#include <type_traits>

#include "flash_wave32.h"
#include "serving_kernels.h"

namespace ofh {
namespace {

constexpr int kSelectThreads = 256;
constexpr int kSelectWaves = kSelectThreads / 64;

// Elements of a 16-byte word, as floats.
template <typename T>
struct Words {
    static constexpr int W = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W)));
    static __device__ __forceinline__ void get(u32x4 x, float (&f)[W]) {
        const vec v = __builtin_bit_cast(vec, x);
#pragma unroll
        for (int i = 0; i < W; ++i) f[i] = (float)v[i];
    }
    static __device__ __forceinline__ u32x4 put(const float (&f)[W]) {
        vec v;
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = (T)f[i];
        return __builtin_bit_cast(u32x4, v);
    }
};

// A NaN stays.
__device__ __forceinline__ float lower(float a, float b) { return b < a || b != b ? b : a; }
__device__ __forceinline__ float upper(float a, float b) { return b > a || b != b ? b : a; }

// Lanes per row of `words` 16-byte words: a power of two.
__device__ __forceinline__ int row_lanes(int words) { return words <= 1 ? 1 : 1 << (32 - __builtin_clz(words - 1)); }

// A wavefront per touched page and key-value head: its lanes take the words of a
// row and, beside each other, several rows, four or eight of which are in flight per lane.
// Bound by reading the page's keys once (us: fp16, 8 prompts of 1500 new tokens up to 2048
// long, H8 D128, pages of 32, 26 MB, 8.7, 3.0 TB/s; a wavefront per page and
// head is 12 per CU, one round of the GPU, so a wavefront's own loads in flight count);
// a decode step's few pages by the launch (64 sequences 4.2).
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void page_bounds_kernel(PageBoundsArgs a) {
    using X = Words<T>;
    constexpr int W = X::W;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * kSelectWaves + (threadIdx.x >> 6);
    const int64_t bi = item / a.Hkv;
    const int hk = (int)(item - bi * a.Hkv), b = (int)(bi / a.touched), i = (int)(bi - (int64_t)b * a.touched);
    if (b >= a.B) return;
    const int size = 1 << a.page_shift;
    const int count = a.counts != nullptr ? max(0, min(a.counts[b], a.T)) : a.T;
    const int64_t length = a.lengths[b], first = max((int64_t)0, length - count);
    const int64_t place = (first >> a.page_shift) + i;
    if (count == 0 || place >= a.max_pages || place << a.page_shift >= length) return;
    const int page = a.table[b * a.table_stride + place];
    if ((unsigned)page >= (unsigned)a.num_pages) return;
    const int rows = (int)min((int64_t)size, length - (place << a.page_shift));
    const int words = a.D / W, lanes = row_lanes(words), groups = 64 / lanes;
    const int word = min(lane % lanes, words - 1), group = lane / lanes;
    const T* keys = (const T*)a.k_pages + page * a.k_sp + hk * a.k_sh + word * W;
    float lo[W], hi[W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        lo[j] = __builtin_huge_valf();
        hi[j] = kNegInf;
    }
    auto read = [&](auto ahead) {  // rows of a lane in flight
        constexpr int AHEAD = decltype(ahead)::value;
        for (int r = group; r < rows; r += AHEAD * groups) {
            u32x4 x[AHEAD];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) x[n] = *(const u32x4*)(keys + (int64_t)min(r + n * groups, rows - 1) * a.k_st);
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                float f[W];
                X::get(x[n], f);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    lo[j] = lower(lo[j], f[j]);
                    hi[j] = upper(hi[j], f[j]);
                }
            }
        }
    };
    if (rows > 4 * groups) read(std::integral_constant<int, 8>{});
    else read(std::integral_constant<int, 4>{});
    for (int d = lanes; d < 64; d *= 2)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            lo[j] = lower(lo[j], __shfl_xor(lo[j], d));
            hi[j] = upper(hi[j], __shfl_xor(hi[j], d));
        }
    if (lane >= words) return;
    T* out = (T*)a.bounds + page * a.b_sp + hk * a.b_sh + word * W;
    *(u32x4*)out = X::put(lo);
    *(u32x4*)(out + a.b_st) = X::put(hi);
}

// Pages with keys up to token (b, t): the candidates.
__device__ __forceinline__ int candidates(const SelectArgs& a, int b, int t) {
    const int capacity = a.max_pages << a.page_shift;
    const int seen = max(0, min(a.lengths[b], capacity)) - a.T + t + 1;
    return (max(0, seen) + (1 << a.page_shift) - 1) >> a.page_shift;
}

// Scores as numbers whose order is theirs: -0 counts as 0, NaN is above all. 0 is
// below every score: pages without a place in the pool.
__device__ __forceinline__ unsigned score_rank(float x) {
    if (x != x) return ~0u;
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, 0xf, 0xf, true);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over `lanes` neighbouring lanes (up to 16), valid in the first of them.
__device__ __forceinline__ double sum_lanes(double x, int lanes) {
    if (lanes >= 2) x += dpp<0xB1>(x);   // quad_perm [1,0,3,2]
    if (lanes >= 4) x += dpp<0x4E>(x);   // quad_perm [2,3,0,1]
    if (lanes >= 8) x += dpp<0x104>(x);  // row_shl:4
    if (lanes >= 16) x += dpp<0x108>(x); // row_shl:8
    return x;
}

// Bits of x where m has ones, of y elsewhere. (Written as such: the compiler takes
// the select apart again into two masks and an or for every other column.)
__device__ __forceinline__ unsigned bit_select(unsigned m, unsigned x, unsigned y) {
    unsigned r;
    asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(m), "v"(x), "v"(y));
    return r;
}

constexpr int kScoreWords = 4;      // of a bounds row that a lane takes
constexpr int kScoreQuery = 4096;   // numbers of Q that a workgroup keeps at most: 32 KB

// A workgroup scores up to `per` pages for one token and key-value head. `lanes`
// neighbouring lanes share a page, each with four words of lo and of hi, so that a
// sum takes few lane exchanges. Q is in LDS in 64 bits, beside it a mask of its
// positive numbers in the layout of the bounds, so that hi or lo is one bit select
// for a word. Tokens that see no more pages than they may take need no scores.
//
// What bounds it (bf16, 32 sequences of 2000-32768 tokens, pages of 32, H32/8 D128: 71 MB
// of bounds, 23.9 us in a trace): the reading of 512 bytes here and there, and beside it
// the sums (without them 19.8; in fp32 22.8). Workgroups are numbered chunk by chunk,
// since row by row the late chunks, which only long sequences have, fall on the same
// XCDs: 29.0.
template <typename T>
__global__ __launch_bounds__(kSelectThreads) void page_score_kernel(SelectArgs a, int per, int lanes, int heads_kept) {
    using X = Words<T>;
    constexpr int W = X::W;
    extern __shared__ __attribute__((aligned(16))) double q[];
    // rows of Q in the layout of the lanes: `slots` words, 0 past the row
    const int slots = lanes * kScoreWords;
    u32x4* masks = (u32x4*)(q + heads_kept * slots * W);
    const int rows = a.B * a.Hkv * a.T, chunk = blockIdx.x / rows;
    const int64_t row = blockIdx.x - (int64_t)chunk * rows;  // (b, hk, t)
    const int t = (int)(row % a.T), hk = (int)(row / a.T % a.Hkv), b = (int)(row / a.T / a.Hkv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int words = a.D / W, beside = 64 / lanes;
    const int sub = lane & (lanes - 1), slot = lane / lanes;
    // (the first page's table entry is read beside the length, not after it)
    const int page0 = chunk * per, start = page0 + wave * beside + slot;
    const int first_page = a.table[b * a.table_stride + min(start, a.max_pages - 1)];
    const int have = candidates(a, b, t), page1 = min(have, page0 + per);
    if (have <= a.pages || page0 >= have) return;
    for (int g0 = 0; g0 < a.G; g0 += heads_kept) {
        const int heads = min(heads_kept, a.G - g0);
        __syncthreads();
        for (int n = threadIdx.x; n < heads * slots; n += kSelectThreads) {
            const int g = n >> __builtin_ctz(slots), w = n & (slots - 1);
            const T* at = (const T*)a.q + b * a.q_sb + (int64_t)(hk * a.G + g0 + g) * a.q_sh + t * a.q_st + w * W;
            if (w >= words) {
#pragma unroll
                for (int j = 0; j < W; ++j) q[n * W + j] = 0.0;
                masks[n] = u32x4{0u, 0u, 0u, 0u};
                continue;
            }
            unsigned on[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float x = a.negative ? -(float)at[j] : (float)at[j];
                q[n * W + j] = (double)x;
                on[j] = x > 0.0f ? ~0u : 0u;
            }
            u32x4 m;
#pragma unroll
            for (int j = 0; j < 4; ++j) m[j] = sizeof(T) == 4 ? on[j] : bit_select(0xffffu, on[2 * j % W], on[(2 * j + 1) % W]);
            masks[n] = m;
        }
        __syncthreads();
        for (int p = start; p - slot < page1; p += kSelectWaves * beside) {
            // (lanes past the last page score some page of the table, for nothing)
            const int page = p == start ? first_page : a.table[b * a.table_stride + min(p, page1 - 1)];
            const bool ok = (unsigned)page < (unsigned)a.num_pages;
            const T* at = (const T*)a.bounds + (ok ? page : 0) * a.b_sp + hk * a.b_sh;
            u32x4 lo[kScoreWords], hi[kScoreWords];
#pragma unroll
            for (int c = 0; c < kScoreWords; ++c) {
                const int word = min(sub + lanes * c, words - 1);
                lo[c] = *(const u32x4*)(at + word * W);
                hi[c] = *(const u32x4*)(at + a.b_st + word * W);
            }
#pragma unroll
            for (int c = 0; c < kScoreWords; ++c)  // a word past the row is 0, as Q's is
                if (sub + lanes * c >= words) lo[c] = hi[c] = u32x4{0u, 0u, 0u, 0u};
            unsigned best = 0;
            for (int g = 0; g < heads; ++g) {
                double sum[2] = {0.0, 0.0};
#pragma unroll
                for (int c = 0; c < kScoreWords; ++c) {
                    const int word = g * slots + sub + lanes * c;
                    const u32x4 m = masks[word];
                    u32x4 bound;
#pragma unroll
                    for (int j = 0; j < 4; ++j) bound[j] = bit_select(m[j], hi[c][j], lo[c][j]);
                    float f[W];
                    X::get(bound, f);
#pragma unroll
                    for (int j = 0; j < W; ++j) sum[j & 1] = __builtin_fma(q[word * W + j], (double)f[j], sum[j & 1]);
                }
                best = max(best, score_rank((float)sum_lanes(sum[0] + sum[1], lanes)));
            }
            if (sub == 0 && p < page1) {
                uint32_t* out = a.scores + row * a.max_pages + p;
                if (!ok) best = 0;
                *out = g0 > 0 ? max(*out, best) : best;
            }
        }
    }
}

constexpr int kSelectKept = 16384;  // scores that a workgroup keeps in LDS

// (us, 256 / 512 / 1024 threads: one sequence of 2047 pages 10.8 / 9.4 / 9.9, 32 of up to
// 1024 pages 8.5 / 8.4 / 9.7)
constexpr int kPickThreads = 512, kPickWaves = kPickThreads / 64;

// A workgroup per token and key-value head. The need-th highest score of the
// candidates between the first and the recent ones is found from counts of the
// scores' bits; then each thread takes a stretch of the candidates, counts what is
// above and what is equal to it, and after a sum over the threads before writes its
// share: ascending, ties to the lower page. Bound by its barriers, 7-7.5 us with the
// launch: eight bits a round take four rounds at most.
__global__ __launch_bounds__(kPickThreads) void page_select_kernel(SelectArgs a) {
    __shared__ uint32_t kept[kSelectKept];
    __shared__ int count[256];
    __shared__ int found[3];
    __shared__ int sums[2][kPickWaves];
    __shared__ uint32_t ends[2][kPickWaves];
    constexpr int EARLY = 4;
    const int64_t row = blockIdx.x;
    const int t = (int)(row % a.T), b = (int)(row / a.T / a.Hkv);
    int32_t* out = a.selected + row * a.pages;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the first scores are read beside the length (what is there past the candidates is
    // not used; no scores are there when every sequence of the table may take all)
    uint32_t early[EARLY] = {};
    if (a.max_pages > a.pages)
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            early[i] = a.scores[row * a.max_pages + min(a.first_pages + tid + i * kPickThreads, a.max_pages - 1)];
    const int have = candidates(a, b, t);
    if (have <= a.pages) {
        for (int i = tid; i < a.pages; i += kPickThreads) out[i] = i < have ? i : -1;
        return;
    }
    const uint32_t* scores = a.scores + row * a.max_pages + a.first_pages;
    const int n = have - a.first_pages - a.recent_pages, need = a.pages - a.first_pages - a.recent_pages;
    const bool keep = n <= kSelectKept;
    uint32_t low = ~0u, high = 0;
    if (need > 0) {
        auto take = [&](int i, uint32_t x) {
            if (keep) kept[i] = x;
            low = min(low, x);
            high = max(high, x);
        };
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            if (tid + i * kPickThreads < n) take(tid + i * kPickThreads, early[i]);
        for (int i = tid + EARLY * kPickThreads; i < n; i += kPickThreads) take(i, scores[i]);
    }
    // (the first and the recent pages)
    for (int i = tid; i < a.first_pages; i += kPickThreads) out[i] = i;
    for (int i = tid; i < a.recent_pages; i += kPickThreads) out[a.pages - a.recent_pages + i] = have - a.recent_pages + i;
    if (need == 0) return;
    auto score = [&](int i) { return keep ? kept[i] : scores[i]; };
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        low = min(low, (uint32_t)__shfl_xor((int)low, d));
        high = max(high, (uint32_t)__shfl_xor((int)high, d));
    }
    if (lane == 0) {
        ends[0][wave] = low;
        ends[1][wave] = high;
    }
    __syncthreads();
    for (int w = 0; w < kPickWaves; ++w) {
        low = min(low, ends[0][w]);
        high = max(high, ends[1][w]);
    }
    // The need-th highest score, eight bits at a time from the first that differs: of
    // the scores whose bits from `shift` up are `limit`, `rest` are taken.
    int shift = low == high ? 0 : 32 - __builtin_clz(low ^ high), rest = need;
    uint64_t limit = (uint64_t)high >> shift;
    while (shift > 0) {
        const int width = min(shift, 8), next = shift - width;
        if (tid < 256) count[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kPickThreads) {
            const uint64_t x = score(i);
            if (x >> shift == limit) atomicAdd(&count[(x >> next) & 255 >> (8 - width)], 1);
        }
        __syncthreads();
        // of the values from the highest down: the first at which `rest` are reached
        const int mine = tid < 256 ? count[255 - tid] : 0;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        if (lane == 63) sums[0][wave] = upto;
        __syncthreads();
        for (int w = 0; w < wave; ++w) upto += sums[0][w];
        if (upto >= rest && upto - mine < rest) {
            found[0] = 255 - tid;
            found[1] = rest - (upto - mine);
            found[2] = mine;
        }
        __syncthreads();
        limit = limit << width | (uint32_t)found[0];
        rest = found[1];
        shift = next;
        if (found[2] == rest) break;  // all of them
    }
    // all above the limit, and the first `rest` equal to it
    const int per = (n + kPickThreads - 1) / kPickThreads, begin = min(n, tid * per), end = min(n, begin + per);
    int above = 0, equal = 0;
    for (int i = begin; i < end; ++i) {
        const uint64_t x = (uint64_t)score(i) >> shift;
        above += x > limit;
        equal += x == limit;
    }
    int above_upto = above, equal_upto = equal;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(above_upto, d), y = __shfl_up(equal_upto, d);
        if (lane >= d) {
            above_upto += x;
            equal_upto += y;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sums[0][wave] = above_upto;
        sums[1][wave] = equal_upto;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        above_upto += sums[0][w];
        equal_upto += sums[1][w];
    }
    int ties = equal_upto - equal;
    int at = a.first_pages + above_upto - above + min(ties, rest);
    for (int i = begin; i < end; ++i) {
        const uint64_t x = (uint64_t)score(i) >> shift;
        if (x > limit || (x == limit && ties++ < rest)) out[at++] = a.first_pages + i;
    }
}

// Lanes that share a page's bounds of `words` words.
int score_lanes(int words) {
    int lanes = 1;
    while (lanes * kScoreWords < words) lanes *= 2;
    return lanes;
}

// Pages of a workgroup: one round of its lanes, more where the workgroups then still
// fill the GPU a few times (us of a selection, 64 pages / one round: f32 D256 B2 H64/4, 512
// pages 35.2 / 16.3; f16 D64 B32 H32/8, 1875 pages 34.2 / 30.3).
int score_pages(const SelectArgs& a, int lanes) {
    const int64_t rows = (int64_t)a.B * a.Hkv * a.T, want = 16 * (int64_t)kComputeUnits;
    int per = kSelectWaves * (64 / lanes);
    while (per < 1024 && rows * ((a.max_pages + 2 * per - 1) / (2 * per)) >= want) per *= 2;
    return per;
}
int score_chunks(const SelectArgs& a, int lanes) {
    const int per = score_pages(a, lanes);
    return (a.max_pages + per - 1) / per;
}

template <typename T>
hipError_t launch_score(const SelectArgs& a, hipStream_t s) {
    const int words = a.D / Words<T>::W, lanes = score_lanes(words), slots = lanes * kScoreWords;
    const int heads = std::min(a.G, kScoreQuery / (slots * Words<T>::W)), chunks = score_chunks(a, lanes);
    hipLaunchKernelGGL((page_score_kernel<T>), dim3((unsigned)((int64_t)a.B * a.Hkv * a.T * chunks)), dim3(kSelectThreads),
                       heads * slots * (Words<T>::W * (int)sizeof(double) + 16), s, a, score_pages(a, lanes), lanes, heads);
    return hipGetLastError();
}

int64_t bounds_grid(const PageBoundsArgs& a) {
    return ((int64_t)a.B * a.touched * a.Hkv + kSelectWaves - 1) / kSelectWaves;
}

}  // namespace

bool page_bounds_fits(const PageBoundsArgs& a) { return grid_fits(bounds_grid(a), kSelectThreads); }

hipError_t launch_page_bounds(const PageBoundsArgs& a, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)bounds_grid(a)), block(kSelectThreads);
    switch (dtype) {
        case DT_F32: hipLaunchKernelGGL((page_bounds_kernel<float>), grid, block, 0, s, a); break;
        case DT_BF16: hipLaunchKernelGGL((page_bounds_kernel<__bf16>), grid, block, 0, s, a); break;
        case DT_F16: hipLaunchKernelGGL((page_bounds_kernel<_Float16>), grid, block, 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

bool page_select_fits(const SelectArgs& a, int dtype) {
    const int64_t rows = (int64_t)a.B * a.Hkv * a.T;
    const int lanes = score_lanes(a.D * (dtype == DT_F32 ? 4 : 2) / 16);
    return grid_fits(rows * score_chunks(a, lanes), kSelectThreads) && grid_fits(rows, kPickThreads);
}

hipError_t launch_page_select(const SelectArgs& a, int dtype, hipStream_t s) {
    if (a.max_pages > a.pages) {
        hipError_t e;
        switch (dtype) {
            case DT_F32: e = launch_score<float>(a, s); break;
            case DT_BF16: e = launch_score<__bf16>(a, s); break;
            case DT_F16: e = launch_score<_Float16>(a, s); break;
            default: return hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(page_select_kernel, dim3((unsigned)((int64_t)a.B * a.Hkv * a.T)), dim3(kPickThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace ofh
