// Rotary positions: on rows by themselves, and on new keys and queries on the
// way into a paged cache.
//
// Pair (x, y) at position p becomes m (x cos a - y sin a, y cos a + x sin a),
// a = p f_i, or with -a in the transposed form (the gradient of the other).
// The angle is formed in 64 bits in turns and brought within half a turn
// there, so that far positions keep their digits: p f_i / 2 pi is off by 2^-52 of
// itself, 2^-31 turns at p = 2^21, where 32 bits would be off by a sixteenth of
// a turn. Sine and cosine are then fp32, like the products; the result is rounded once.
//
// Both kernels are bound by reading and writing each row once. A workgroup
// takes one token or four, so the sines and cosines of a token, one per pair, are
// computed once for all heads and shared through LDS; the first rows are on
// their way meanwhile.

#include "serving_kernels.h"

namespace ofh {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kInFlight = 4;  // items of a thread whose loads are issued together
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

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
    // columns of the item's two words
    static __device__ __forceinline__ void columns(const Rotation& r, int item, int& ca, int& cb) {
        const int turned = r.R / 2 / PAIRS;
        if (item >= turned) {
            ca = cb = r.R + (item - turned) * W;
        } else if (INTERLEAVED) {
            ca = item * 2 * PAIRS;
            cb = W > 1 ? ca : ca + 1;
        } else {
            ca = item * W;
            cb = ca + r.R / 2;
        }
    }
    static __device__ __forceinline__ Item load(const Rotation& r, const T* row, int item) {
        int ca, cb;
        columns(r, item, ca, cb);
        Item x;
        x.a = *(const C*)(row + ca);
        x.b = ONE ? x.a : *(const C*)(row + cb);
        return x;
    }
    static __device__ __forceinline__ void clear(const Rotation& r, T* row, int item) {
        int ca, cb;
        columns(r, item, ca, cb);
        *(C*)(row + ca) = C{};
        if (!ONE) *(C*)(row + cb) = C{};
    }
    // cs: cosines and sines of the row's token
    static __device__ __forceinline__ void store(const Rotation& r, T* row, int item, const Item& x, const float2* cs) {
        int ca, cb;
        columns(r, item, ca, cb);
        if (item >= r.R / 2 / PAIRS) {
            *(C*)(row + ca) = x.a;
            return;
        }
        union U {
            C c;
            T t[W];
        } a, b;
        a.c = x.a;
        b.c = x.b;
        cs += item * PAIRS;
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
    const double turns = (double)position * (r.freq[pair] * kTurn);
    float s, c;
    sincospif((float)(2.0 * (turns - __builtin_rint(turns))), &s, &c);
    return float2{c * r.magnitude, (r.transpose ? -s : s) * r.magnitude};
}

// Items of a row.
inline __host__ __device__ int row_items(const Rotation& r, int D, int W) {
    const int pairs = r.interleaved && W > 1 ? W / 2 : W;
    return r.R / 2 / pairs + (D - r.R) / W;
}

template <typename T, int W, bool INTERLEAVED, int TOKENS>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs a) {
    using X = Row<T, W, INTERLEAVED>;
    __shared__ float2 cs[TOKENS * (kRotaryMaxDim / 2)];
    const int64_t first = (int64_t)blockIdx.x * TOKENS;
    const int tokens = (int)min((int64_t)TOKENS, (int64_t)a.B * a.T - first);
    const unsigned per_row = row_items(a.r, a.D, W), per_token = per_row * (unsigned)a.H, items = per_token * tokens;
    for (unsigned at = threadIdx.x; at - threadIdx.x < items; at += kRotaryThreads * kInFlight) {
        typename X::Item x[kInFlight];
        int64_t to[kInFlight];
        unsigned tok[kInFlight], item[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const unsigned n = at + i * kRotaryThreads;
            if (n >= items) continue;
            tok[i] = n / per_token;
            const unsigned rest = n - tok[i] * per_token, h = rest / per_row;
            item[i] = rest - h * per_row;
            const unsigned bt = (unsigned)first + tok[i], b = bt / (unsigned)a.T, t = bt - b * (unsigned)a.T;
            to[i] = b * a.o_sb + h * a.o_sh + t * a.o_st;
            x[i] = X::load(a.r, (const T*)a.x + b * a.x_sb + h * a.x_sh + t * a.x_st, (int)item[i]);
        }
        if (at == threadIdx.x) {
            const int pairs = a.r.R / 2;
            for (int n = threadIdx.x; n < tokens * pairs; n += kRotaryThreads) {
                const int j = n / pairs, pair = n - j * pairs;
                const unsigned bt = (unsigned)first + j, b = bt / (unsigned)a.T, t = bt - b * (unsigned)a.T;
                const int64_t position = a.positions != nullptr ? (int64_t)a.positions[b * a.pos_sb + t]
                                         : a.lengths != nullptr ? (int64_t)a.lengths[b] - a.T + t
                                                                : a.offset + t;
                cs[n] = turn(a.r, pair, position);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i)
            if (at + i * kRotaryThreads < items)
                X::store(a.r, (T*)a.o + to[i], (int)item[i], x[i], cs + tok[i] * (a.r.R / 2));
    }
}

// Where the rows of a new token go.
struct Place {
    bool padding;      // not a token of its sequence
    int64_t position;
    int64_t k, v;      // elements from the pools' start; -1: no place
};
__device__ __forceinline__ Place place(const CacheWriteArgs& w, unsigned b, unsigned t) {
    Place p;
    const int count = w.counts != nullptr ? max(0, min(w.counts[b], w.T)) : w.T;
    p.padding = (int)t >= count;
    p.position = (int64_t)w.lengths[b] - count + t;
    p.k = p.v = -1;
    const int64_t slot = p.position >> w.page_shift;
    if (p.padding || p.position < 0 || slot >= w.max_pages) return p;
    const int page = w.table[b * w.table_stride + slot];
    if ((unsigned)page >= (unsigned)w.num_pages) return p;
    const int64_t row = p.position & (((int64_t)1 << w.page_shift) - 1);
    p.k = page * w.kp_sp + row * w.kp_st;
    p.v = page * w.vp_sp + row * w.vp_st;
    return p;
}

// Items of a token: those of its K rows, then its Q rows, then the words of its V rows.
template <typename T, int W, bool INTERLEAVED, int TOKENS>
__global__ __launch_bounds__(kRotaryThreads) void cache_append_kernel(CacheAppendArgs a) {
    using X = Row<T, W, INTERLEAVED>;
    __shared__ float2 cs[TOKENS * (kRotaryMaxDim / 2)];
    __shared__ Place places[TOKENS];
    const CacheWriteArgs& w = a.w;
    const int64_t first = (int64_t)blockIdx.x * TOKENS;
    const int tokens = (int)min((int64_t)TOKENS, (int64_t)w.B * w.T - first);
    const unsigned per_row = row_items(a.r, a.D, W), v_row = (unsigned)a.Dv / W;
    const unsigned kq = per_row * (unsigned)(w.Hkv + a.H), per_token = kq + v_row * (unsigned)w.Hkv;
    const unsigned items = per_token * tokens;
    for (unsigned at = threadIdx.x; at - threadIdx.x < items; at += kRotaryThreads * kInFlight) {
        typename X::Item x[kInFlight];
        unsigned tok[kInFlight], row[kInFlight], item[kInFlight];  // rows: K, then Q, then V
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const unsigned n = at + i * kRotaryThreads;
            if (n >= items) continue;
            tok[i] = n / per_token;
            const unsigned rest = n - tok[i] * per_token;
            const bool is_v = rest >= kq;
            const unsigned r = is_v ? (rest - kq) / v_row : rest / per_row;
            item[i] = is_v ? rest - kq - r * v_row : rest - r * per_row;
            row[i] = is_v ? r + w.Hkv + a.H : r;
            const unsigned bt = (unsigned)first + tok[i], b = bt / (unsigned)w.T, t = bt - b * (unsigned)w.T;
            if (w.counts != nullptr && (int)t >= w.counts[b]) continue;  // padding is not read
            if (is_v)
                x[i].a = *(const typename X::C*)((const T*)w.v + b * w.v_sb + r * w.v_sh + t * w.v_st + item[i] * W);
            else if (r < (unsigned)w.Hkv)
                x[i] = X::load(a.r, (const T*)w.k + b * w.k_sb + r * w.k_sh + t * w.k_st, (int)item[i]);
            else
                x[i] = X::load(a.r, (const T*)a.q + b * a.q_sb + (r - w.Hkv) * a.q_sh + t * a.q_st, (int)item[i]);
        }
        if (at == threadIdx.x) {
            const int pairs = a.r.R / 2;
            for (int n = threadIdx.x; n < tokens * pairs; n += kRotaryThreads) {
                const int j = n / pairs, pair = n - j * pairs;
                const unsigned bt = (unsigned)first + j, b = bt / (unsigned)w.T, t = bt - b * (unsigned)w.T;
                const Place p = place(w, b, t);
                if (pair == 0) places[j] = p;
                cs[n] = turn(a.r, pair, p.position);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            if (at + i * kRotaryThreads >= items) continue;
            const Place& p = places[tok[i]];
            const float2* c = cs + tok[i] * (a.r.R / 2);
            const unsigned bt = (unsigned)first + tok[i], b = bt / (unsigned)w.T, t = bt - b * (unsigned)w.T;
            if (row[i] < (unsigned)w.Hkv) {
                if (p.k >= 0) X::store(a.r, (T*)w.k_pages + p.k + row[i] * w.kp_sh, (int)item[i], x[i], c);
            } else if (row[i] < (unsigned)(w.Hkv + a.H)) {
                T* to = (T*)a.q_out + b * a.o_sb + (row[i] - w.Hkv) * a.o_sh + t * a.o_st;
                if (p.padding) X::clear(a.r, to, (int)item[i]);
                else X::store(a.r, to, (int)item[i], x[i], c);
            } else if (p.v >= 0) {
                *(typename X::C*)((T*)w.v_pages + p.v + (row[i] - w.Hkv - a.H) * w.vp_sh + item[i] * W) = x[i].a;
            }
        }
    }
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

int elem_of(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// Four tokens per workgroup once that leaves enough workgroups to fill the GPU.
bool four_tokens(int64_t tokens) { return tokens >= 16 * (int64_t)kComputeUnits; }

// Items of a workgroup and tokens are 32-bit in the kernels.
bool fits(int64_t tokens, int64_t per_token) {
    return tokens < ((int64_t)1 << 31) && per_token < ((int64_t)1 << 28) &&
           grid_fits(four_tokens(tokens) ? (tokens + 3) / 4 : tokens, kRotaryThreads);
}

#define OFH_ROTARY_LAUNCH(KERNEL, T, W, INTER)                                                                      \
    do {                                                                                                            \
        if (four_tokens(tokens))                                                                                    \
            hipLaunchKernelGGL((KERNEL<T, W, INTER, 4>), dim3((unsigned)((tokens + 3) / 4)), dim3(kRotaryThreads), 0, s, a); \
        else                                                                                                        \
            hipLaunchKernelGGL((KERNEL<T, W, INTER, 1>), dim3((unsigned)tokens), dim3(kRotaryThreads), 0, s, a);     \
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

bool rotary_fits(const RotaryArgs& a, int dtype) {
    const int elem = elem_of(dtype), w = rotary_in_words(a, elem) ? 16 / elem : 1;
    return fits((int64_t)a.B * a.T, (int64_t)a.H * row_items(a.r, a.D, w));
}
bool cache_append_fits(const CacheAppendArgs& a, int dtype) {
    const int elem = elem_of(dtype), w = append_in_words(a, elem) ? 16 / elem : 1;
    return fits((int64_t)a.w.B * a.w.T,
                ((int64_t)a.w.Hkv + a.H) * row_items(a.r, a.D, w) + (int64_t)a.w.Hkv * (a.Dv / w));
}

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
