// Rotary positions: on rows by themselves, and on new keys and queries on the
// way into a paged cache.
//
// Pair (x, y) at position p becomes m (x cos a - y sin a, y cos a + x sin a),
// a = p f_i, or with -a in the transposed form (the gradient of the other).
// The angle is formed in 64 bits in turns and brought within half a turn
// there, so that far positions keep their digits: p f_i / 2 pi takes three roundings
// (of 1 / 2 pi, times f_i, times p), each 2^-53 of it at most. At p = 2^21 and f_i = 1, 2^18.3
// turns, they are 2^-33 turns together, where each of 32 bits could be 2^-5.7,
// a fiftieth of a turn. Sine and cosine are then fp32, with what the angle's rounding to fp32 takes
// off put back to first order, and so are the products; the result is rounded once.
//
// Both kernels are bound by reading and writing each row once. A wavefront (or,
// with few tokens, each of four) takes a token: its place and position are scalars,
// its sines and cosines are computed once for all heads and kept in LDS, and the
// first rows are on their way meanwhile. A lane keeps its columns for all rows.
// Measured (us): rows by themselves, bf16 B4 H32 T2048 D128, 134 MB, 26.2, which is 5.1
// TB/s, a copy's rate (kernel 23.4); into the cache, fp16 B8 H16/8 T2048 of which 700-2048
// count, 207 MB, 48.8 (kernel 43.8, 4.7 TB/s); one token of 64 sequences, bf16 H32/8 D128,
// 7.9 (kernel 4.9): the launch, then length, place in the table, page and store in turn.

#include "serving_kernels.h"

namespace ofh {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryWaves = kRotaryThreads / 64;
constexpr int kInFlight = 4;  // rows of a lane whose loads are issued together
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
constexpr double kHalfTurn = 3.14159265358979323846;

template <int BYTES>
struct Word;
template <>
struct Word<16> {
    typedef unsigned int type __attribute__((ext_vector_type(4)));
};
template <>
struct Word<4> {
    typedef unsigned int type;
};
template <>
struct Word<2> {
    typedef unsigned short type;
};

// How a row of D columns, R of them turned, is cut into items. W columns are 16
// bytes, or one column where an address or a size does not allow that.
//   halves:      an item is W pairs: W columns of either half
//   interleaved: W / 2 pairs in W columns; with W = 1 a pair
// then (D - R) / W items that are copied.
template <typename T, int W, bool INTERLEAVED>
struct Row {
    static constexpr int BYTES = W * (int)sizeof(T);
    using C = typename Word<BYTES>::type;
    static constexpr int PAIRS = INTERLEAVED && W > 1 ? W / 2 : W;  // of an item
    static constexpr bool ONE = INTERLEAVED && W > 1;               // word of an item
    struct Item {
        C a, b;
    };
    int ca, cb, pair;  // columns of the item's two words, its first pair; copied: pair -1
    __device__ __forceinline__ Row(const Rotation& r, int item) {
        const int turned = r.R / 2 / PAIRS;
        pair = item < turned ? item * PAIRS : -1;
        if (pair < 0) {
            ca = cb = r.R + (item - turned) * W;
        } else if (INTERLEAVED) {
            ca = item * 2 * PAIRS;
            cb = W > 1 ? ca : ca + 1;
        } else {
            ca = item * W;
            cb = ca + r.R / 2;
        }
    }
    __device__ __forceinline__ Item load(const T* row) const {
        Item x;
        x.a = *(const C*)(row + ca);
        x.b = ONE ? x.a : *(const C*)(row + cb);
        return x;
    }
    __device__ __forceinline__ void clear(T* row) const {
        *(C*)(row + ca) = C{};
        if (!ONE) *(C*)(row + cb) = C{};
    }
    // cs: cosines and sines of the row's token
    __device__ __forceinline__ void store(T* row, const Item& x, const float2* cs) const {
        if (pair < 0) {
            *(C*)(row + ca) = x.a;
            return;
        }
        union U {
            C c;
            T t[W];
        } a, b;
        a.c = x.a;
        b.c = x.b;
        cs += pair;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const float2 t = cs[i];
            T& p = ONE ? a.t[2 * i] : a.t[i];
            T& q = ONE ? a.t[2 * i + 1] : b.t[i];
            const float u = (float)p, v = (float)q;
            p = (T)(u * t.x - v * t.y);
            q = (T)(v * t.x + u * t.y);
        }
        *(C*)(row + ca) = a.c;
        if (!ONE) *(C*)(row + cb) = b.c;
    }
};

__device__ __forceinline__ float2 turn(const Rotation& r, int pair, int64_t position) {
    const double turns = (double)position * (r.freq[pair] * kTurn), halves = 2.0 * (turns - __builtin_rint(turns));
    const float x = (float)halves, off = (float)((halves - (double)x) * kHalfTurn);
    float s, c;
    sincospif(x, &s, &c);
    const float s1 = __builtin_fmaf(c, off, s), c1 = __builtin_fmaf(-s, off, c);
    return float2{c1 * r.magnitude, (r.transpose ? -s1 : s1) * r.magnitude};
}

// Items of a row.
inline __host__ __device__ int row_items(const Rotation& r, int D, int W) {
    const int pairs = r.interleaved && W > 1 ? W / 2 : W;
    return r.R / 2 / pairs + (D - r.R) / W;
}

// The wavefront's token and its share of the token's rows. PER_TOKEN wavefronts
// share a token; `beside` rows of `lanes` lanes stand beside each other in one.
template <int PER_TOKEN>
struct Share {
    int lanes, beside, lane, slot;
    int64_t token;
    __device__ __forceinline__ Share(int items) {
        lanes = 1;
        while (lanes < items && lanes < 64) lanes *= 2;
        beside = 64 / lanes;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
        token = (int64_t)blockIdx.x * (kRotaryWaves / PER_TOKEN) + wave / PER_TOKEN;
        lane = l & (lanes - 1);
        slot = (wave % PER_TOKEN) * beside + l / lanes;
    }
    __device__ __forceinline__ int stride() const { return PER_TOKEN * beside; }
};

// Cosines and sines of a position, by the wavefront for itself.
__device__ __forceinline__ void turns(const Rotation& r, int64_t position, float2* cs) {
    for (int n = threadIdx.x & 63; n < r.R / 2; n += 64) cs[n] = turn(r, n, position);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Turns rows 0 .. rows - 1 of a token: from(row) is a row, to(row) where it goes (null:
// nowhere), padding(row) whether it is cleared instead. `before` runs once, when the
// first rows are on their way, and leaves cs.
template <typename X, typename S, typename From, typename To, typename Padding, typename Before>
__device__ __forceinline__ void turn_rows(const Rotation& r, const S& share, int items, int rows, const float2* cs, From from,
                                          To to, Padding padding, Before before) {
    bool first = true;
    for (int base = 0; base < items; base += share.lanes) {
        const int item = base + share.lane;
        const X x(r, min(item, items - 1));
        for (int row0 = share.slot; row0 - share.slot < rows; row0 += kInFlight * share.stride()) {
            typename X::Item v[kInFlight];
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) {
                const int row = min(row0 + i * share.stride(), rows - 1);
                if (!padding(row)) v[i] = x.load(from(row));
            }
            if (first) before();
            first = false;
#pragma unroll
            for (int i = 0; i < kInFlight; ++i) {
                const int row = row0 + i * share.stride();
                if (row >= rows || item >= items) continue;
                auto* out = to(row);
                if (out == nullptr) continue;
                if (padding(row)) x.clear(out);
                else x.store(out, v[i], cs);
            }
        }
    }
}

template <typename T, int W, bool INTERLEAVED, int PER_TOKEN>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 table[kRotaryWaves][kRotaryMaxDim / 2];
    const int items = row_items(a.r, a.D, W);
    const Share<PER_TOKEN> share(items);
    if (share.token >= (int64_t)a.B * a.T) return;
    const int b = (int)((unsigned)share.token / (unsigned)a.T), t = (int)share.token - b * a.T;
    float2* cs = table[threadIdx.x >> 6];
    const T* x = (const T*)a.x + b * a.x_sb + t * a.x_st;
    T* o = (T*)a.o + b * a.o_sb + t * a.o_st;
    turn_rows<Row<T, W, INTERLEAVED>>(
        a.r, share, items, a.H, cs, [&](int h) { return x + h * a.x_sh; }, [&](int h) { return o + h * a.o_sh; },
        [](int) { return false; },
        [&] {
            turns(a.r, a.positions != nullptr ? (int64_t)a.positions[b * a.pos_sb + t]
                       : a.lengths != nullptr ? (int64_t)a.lengths[b] - a.T + t
                                              : a.offset + t, cs);
        });
}

template <typename T, int W, bool INTERLEAVED, int PER_TOKEN>
__global__ __launch_bounds__(kRotaryThreads) void cache_append_kernel(CacheAppendArgs a) {
    using X = Row<T, W, INTERLEAVED>;
    using C = typename X::C;
    __shared__ float2 table[kRotaryWaves][kRotaryMaxDim / 2];
    const CacheWriteArgs& w = a.w;
    const int items = row_items(a.r, a.D, W), words = a.Dv / W;
    const Share<PER_TOKEN> share(items), v_share(words);
    if (share.token >= (int64_t)w.B * w.T) return;
    const int b = (int)((unsigned)share.token / (unsigned)w.T), t = (int)share.token - b * w.T;
    const int count = w.counts != nullptr ? max(0, min(w.counts[b], w.T)) : w.T;
    const bool padding = t >= count;
    float2* cs = table[threadIdx.x >> 6];

    const int64_t position = (int64_t)w.lengths[b] - count + t, place = position >> w.page_shift;
    int page = -1;
    if (!padding && position >= 0 && place < w.max_pages) page = w.table[b * w.table_stride + place];
    const bool placed = (unsigned)page < (unsigned)w.num_pages;
    const int64_t in_page = position & (((int64_t)1 << w.page_shift) - 1);
    T* k_to = (T*)w.k_pages + page * w.kp_sp + in_page * w.kp_st;
    T* v_to = (T*)w.v_pages + page * w.vp_sp + in_page * w.vp_st;

    const T* k = (const T*)w.k + b * w.k_sb + t * w.k_st;
    const T* q = (const T*)a.q + b * a.q_sb + t * a.q_st;
    T* q_to = (T*)a.q_out + b * a.o_sb + t * a.o_st;
    // V rows are copied, K rows and Q rows turned
    const T* v = (const T*)w.v + b * w.v_sb + t * w.v_st;
    if (placed)
        for (int base = 0; base < words; base += v_share.lanes) {
            const int word = base + v_share.lane;
            for (int h0 = v_share.slot; h0 - v_share.slot < w.Hkv; h0 += kInFlight * v_share.stride()) {
                C x[kInFlight];
#pragma unroll
                for (int i = 0; i < kInFlight; ++i)
                    x[i] = *(const C*)(v + min(h0 + i * v_share.stride(), w.Hkv - 1) * w.v_sh + min(word, words - 1) * W);
#pragma unroll
                for (int i = 0; i < kInFlight; ++i) {
                    const int h = h0 + i * v_share.stride();
                    if (h < w.Hkv && word < words) *(C*)(v_to + h * w.vp_sh + word * W) = x[i];
                }
            }
        }
    turn_rows<X>(
        a.r, share, items, w.Hkv + a.H, cs,
        [&](int row) { return row < w.Hkv ? k + row * w.k_sh : q + (row - w.Hkv) * a.q_sh; },
        [&](int row) -> T* {
            if (row >= w.Hkv) return q_to + (row - w.Hkv) * a.o_sh;
            return placed ? k_to + row * w.kp_sh : nullptr;
        },
        [&](int) { return padding; },
        [&] {
            if (!padding) turns(a.r, position, cs);
        });
}

bool turns_in_words(const Rotation& r, int D, int elem) {
    const int words = 16 / elem;
    return (r.interleaved ? r.R : r.R / 2) % words == 0 && D % words == 0;
}
bool aligned(uint64_t addresses, int64_t strides, int elem) {
    return addresses % 16 == 0 && (uint64_t)(strides * elem) % 16 == 0;
}
bool rotary_in_words(const RotaryArgs& a, int elem) {
    return turns_in_words(a.r, a.D, elem) && aligned((uintptr_t)a.x | (uintptr_t)a.o,
                                                     a.x_sb | a.x_sh | a.x_st | a.o_sb | a.o_sh | a.o_st, elem);
}
bool append_in_words(const CacheAppendArgs& a, int elem) {
    const CacheWriteArgs& w = a.w;
    uint64_t all = (uintptr_t)w.k | (uintptr_t)w.v | (uintptr_t)w.k_pages | (uintptr_t)w.v_pages;
    int64_t strides = w.k_sb | w.k_sh | w.k_st | w.v_sb | w.v_sh | w.v_st | w.kp_sp | w.kp_sh | w.kp_st | w.vp_sp |
                      w.vp_sh | w.vp_st;
    if (a.H > 0) {
        all |= (uintptr_t)a.q | (uintptr_t)a.q_out;
        strides |= a.q_sb | a.q_sh | a.q_st | a.o_sb | a.o_sh | a.o_st;
    }
    return turns_in_words(a.r, a.D, elem) && a.Dv % (16 / elem) == 0 && aligned(all, strides, elem);
}

// A wavefront per token once that fills the GPU, a workgroup before (us, a workgroup /
// a wavefront: the 8192 tokens of 32 heads above 29.3 / 26.2, the prompts 62.7 / 48.8).
bool many_tokens(int64_t tokens) { return tokens >= 16 * (int64_t)kComputeUnits; }
int64_t rotary_grid(int64_t tokens) { return many_tokens(tokens) ? (tokens + kRotaryWaves - 1) / kRotaryWaves : tokens; }

// Tokens and rows of a token are 32-bit in the kernels.
bool fits(int64_t tokens, int64_t rows) {
    return tokens < ((int64_t)1 << 31) && rows < ((int64_t)1 << 30) && grid_fits(rotary_grid(tokens), kRotaryThreads);
}

#define OFH_ROTARY_LAUNCH(KERNEL, T, W, INTER)                                                          \
    do {                                                                                                \
        const dim3 grid((unsigned)rotary_grid(tokens)), block(kRotaryThreads);                          \
        if (many_tokens(tokens)) hipLaunchKernelGGL((KERNEL<T, W, INTER, 1>), grid, block, 0, s, a);    \
        else hipLaunchKernelGGL((KERNEL<T, W, INTER, kRotaryWaves>), grid, block, 0, s, a);             \
    } while (0)

template <typename T>
hipError_t launch_rotary_type(const RotaryArgs& a, hipStream_t s) {
    constexpr int W = 16 / (int)sizeof(T);
    const int64_t tokens = (int64_t)a.B * a.T;
    const bool words = rotary_in_words(a, sizeof(T));
    if (words && a.r.interleaved) OFH_ROTARY_LAUNCH(rotary_kernel, T, W, true);
    else if (words) OFH_ROTARY_LAUNCH(rotary_kernel, T, W, false);
    else if (a.r.interleaved) OFH_ROTARY_LAUNCH(rotary_kernel, T, 1, true);
    else OFH_ROTARY_LAUNCH(rotary_kernel, T, 1, false);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_append_type(const CacheAppendArgs& a, hipStream_t s) {
    constexpr int W = 16 / (int)sizeof(T);
    const int64_t tokens = (int64_t)a.w.B * a.w.T;
    const bool words = append_in_words(a, sizeof(T));
    if (words && a.r.interleaved) OFH_ROTARY_LAUNCH(cache_append_kernel, T, W, true);
    else if (words) OFH_ROTARY_LAUNCH(cache_append_kernel, T, W, false);
    else if (a.r.interleaved) OFH_ROTARY_LAUNCH(cache_append_kernel, T, 1, true);
    else OFH_ROTARY_LAUNCH(cache_append_kernel, T, 1, false);
    return hipGetLastError();
}

}  // namespace

bool rotary_fits(const RotaryArgs& a) { return fits((int64_t)a.B * a.T, a.H); }
bool cache_append_fits(const CacheAppendArgs& a) { return fits((int64_t)a.w.B * a.w.T, (int64_t)a.w.Hkv + a.H); }

hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DT_F32: return launch_rotary_type<float>(a, s);
        case DT_BF16: return launch_rotary_type<__bf16>(a, s);
        case DT_F16: return launch_rotary_type<_Float16>(a, s);
        default: return hipErrorInvalidValue;
    }
}
hipError_t launch_cache_append(const CacheAppendArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DT_F32: return launch_append_type<float>(a, s);
        case DT_BF16: return launch_append_type<__bf16>(a, s);
        case DT_F16: return launch_append_type<_Float16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ofh
