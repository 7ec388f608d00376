// Attention of new tokens over a cached sequence: every wavefront streams keys
// of its own straight into the operand registers of the matrix instructions.
//
// What bounds it: reading K and V once (2 bytes of K and V per product of a
// row's tile, far below what the matrix cores need). So nothing goes through
// LDS: with S^T = K Q^T and O^T = V^T P^T
//  * a K fragment (16 keys x 32 columns in 16 bits, 16 x 16 in fp32) is one
//    16-byte load per lane from the key's row;
//  * a V row is read 16 bytes per lane with 16 lanes on a row's 128 columns
//    (64 in fp32). Lane c of a row then holds columns 8c .. 8c + 7 of eight
//    keys, and v_perm turns that 8 x 8 block in place into the operands of
//    eight products, product i covering columns 8m + i for its 16 rows m: the
//    transposition that V needs crosses no lanes;
//  * the accumulator layout (lane n + 16 g holds keys 4g .. 4g + 3 of query row
//    n) is the operand layout of P^T when a product's eight keys per lane group
//    are 4g .. 4g + 3 of two 16-key blocks, so P stays where it is formed.
// The next step's K and V are requested before this step's products. Blocks of
// 16 keys never cross a page (page sizes are multiples of 16), so a block's
// page is one scalar load, made two steps ahead.
//
// A tile has 16 (or 32) rows of one (sequence, key-value head): the heads of a
// group and the new tokens share what is read. The wavefronts of a workgroup
// take the steps in turn and fold their (m, l, O) in LDS; `splits` workgroups
// share a tile's steps evenly, by the sequence's own visible keys, and are
// joined with O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
//
// The running max that probabilities are taken against is raised only when a
// score exceeds it by more than 2^8, so a step without a raise (nearly all)
// exchanges nothing between lanes. Sums and O are fp32; P is rounded to the
// input type for the product (the same rounding for numerator and sum), fp32 P
// not at all.
//
// A key that no row of the tile sees has its V zeroed, so whatever a page holds
// past a sequence's end does not reach the result. Where rows differ in what
// they see (several new tokens), a NaN or an infinity in the V of a key leaves a
// NaN in the O of rows that do not see it: a wavefront that ends with a NaN runs
// again and forms the products of such steps once per token.

#include "flash_wave32.h"
#include "serving_kernels.h"

namespace ofh {
namespace {

constexpr int kWaves = kStreamThreads / 64;

// Registers and products of a kernel: NB blocks of 16 keys per step, KF 16-byte
// K fragments per block, V as VC chunks of 16 lanes with VW columns each.
template <typename T, int DK>
struct StreamTile {
    static constexpr int ES = 2, NB = 2;
    static constexpr int KF = DK / 32, KW = 8;  // K columns per lane and fragment
    static constexpr int VC = DK >= 128 ? DK / 128 : 1, VW = DK >= 128 ? 8 : 4;
    static constexpr int NO = VC * VW;
    using P = typename Mfma16<T>::v8;
    template <typename V>
    struct Operands {
        u32x4 v[NO];
        __device__ __forceinline__ void apply(const unsigned (&keep)[4]) {
#pragma unroll
            for (int j = 0; j < NO; ++j) v[j] &= u32x4{keep[0], keep[1], keep[2], keep[3]};
        }
    };
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        if constexpr (__is_same(T, __bf16))
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                           c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b),
                                                          c, 0, 0, 0);
    }
};
template <int DK>
struct StreamTile<float, DK> {
    static constexpr int ES = 4, NB = DK <= 64 ? 2 : 1;
    static constexpr int KF = DK / 16, KW = 4;
    static constexpr int VC = DK / 64, VW = 4;
    static constexpr int NO = VC * VW;
    template <typename V>
    struct Operands {
        V v[NB * 4][VC];
        __device__ __forceinline__ void apply(const unsigned (&keep)[NB * 4]) {
#pragma unroll
            for (int t = 0; t < NB * 4; ++t)
#pragma unroll
                for (int c = 0; c < VC; ++c) v[t][c] &= V{keep[t], keep[t], keep[t], keep[t]};
        }
    };
};

__device__ __forceinline__ float max4(float x) {  // over the four lane groups of a row
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum4(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a row tile reads: 16-key blocks [0, sink_blocks) and, from first_block
// on, the window's; numbered in one row (block()).
struct StreamRange {
    int length;                     // keys of the sequence
    int64_t first_pos;              // position of token 0
    int t0, t1;                     // tokens of the tile
    int sink_blocks, first_block, blocks;
    __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : i - sink_blocks + first_block; }
};

__device__ __forceinline__ StreamRange stream_range(const StreamArgs& a, int b, int rt, int rows) {
    StreamRange r;
    r.length = a.capacity;
    if (a.lengths != nullptr) r.length = max(0, min(a.lengths[b], a.capacity));
    r.first_pos = a.positions_from_end ? (int64_t)r.length - a.T : a.query_offset;
    r.t0 = rt * rows / a.G;
    r.t1 = min(a.T - 1, (rt * rows + rows - 1) / a.G);
    // keys below `end` can be seen, and with a window those from `begin` on
    int64_t last = r.first_pos + r.t1;
    if (!a.positions_from_end && a.lengths != nullptr) last = min(last, (int64_t)r.length - 1);  // padding rows see none
    const int end = (int)max((int64_t)0, min((int64_t)r.length, last + 1));
    const int begin = a.window > 0 ? (int)min((int64_t)end, max((int64_t)0, r.first_pos + r.t0 + 1 - a.window)) : 0;
    const int nb = (end + kStreamKeys - 1) / kStreamKeys;
    r.first_block = begin / kStreamKeys;
    r.sink_blocks = 0;
    if (a.window > 0) {
        r.sink_blocks = min((min(a.sinks, end) + kStreamKeys - 1) / kStreamKeys, nb);
        r.first_block = max(r.first_block, r.sink_blocks);
    }
    r.blocks = r.sink_blocks + max(0, nb - r.first_block);
    return r;
}

// Steps per split and splits that have any, of a tile of `steps` steps.
__device__ __forceinline__ int stream_split(const StreamArgs& a, int steps, int& per) {
    const int n = max(1, min(a.splits, steps / max(1, a.min_steps)));
    per = max(1, (steps + n - 1) / n);
    return max(1, (steps + per - 1) / per);
}

// Workgroup -> (sequence and key-value head, row tile, split). Workgroups go to
// the 8 XCDs in turn; where they can be dealt out evenly, the tiles and splits
// of one key-value head run on one XCD and share its L2. Late tokens, whose
// keys are most, run first.
__device__ __forceinline__ void stream_work(const StreamArgs& a, int id, int& bh, int& rt, int& split) {
    const int n = a.B * a.Hkv, per = a.row_tiles * a.splits;
    int rest;
    if ((n & 7) == 0) {
        const int j = id >> 3;
        bh = j / per * 8 + (id & 7);
        rest = j % per;
    } else {
        bh = id / per;
        rest = id % per;
    }
    split = rest % a.splits;
    rt = a.row_tiles - 1 - rest / a.splits;
}

// O of a row, columns [c, c + W): normalised, in the output's type.
template <typename T, int W>
__device__ __forceinline__ void put_out(const StreamArgs& a, int64_t off, const float* x, float inv) {
    if (sizeof(T) == 4 || a.out_f32) {
#pragma unroll
        for (int i = 0; i < W; i += 4)
            *(f32x4*)((float*)a.o + off + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]} * inv;
    } else {
        typedef T vec __attribute__((ext_vector_type(W)));
        vec val;
#pragma unroll
        for (int i = 0; i < W; ++i) val[i] = (T)(x[i] * inv);
        *(vec*)((T*)a.o + off) = val;
    }
}

template <typename T, int DK, int RT, bool PAGED>
struct StreamWave {
    using S = StreamTile<T, DK>;
    static constexpr int ROWS = 16 * RT;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int VB = S::VW * S::ES;  // bytes of a lane's V chunk: 16 or 8
    static constexpr int VD = VB / 4;         // dwords
    typedef unsigned int vraw __attribute__((ext_vector_type(VD)));

    struct Step {  // K and V of a step as loaded
        u32x4 k[S::NB][S::KF];
        vraw v[S::NB * 4][S::VC];
    };
    struct Pages {  // pages of a step's blocks (contiguous K and V: unused)
        int id[S::NB];
    };

    const StreamArgs& a;
    const StreamRange& r;
    int b, hk, n, g;  // n: row of a 16-row tile, or a lane's place in a V row; g: lane group
    u32x4 q[RT][S::KF];
    f32x4 o[RT][S::NO];
    float m[RT], l[RT];
    // per row: keys below hi and from lo on (or below sinks) are seen
    int hi[RT], lo[RT], tok[RT], pos[RT];
    float slope[RT];
    int hi_min, hi_max, lo_min, lo_max;  // over the tile's rows
    const char* kbase;
    const char* vbase;
    unsigned koff, voff[4];

    __device__ __forceinline__ StreamWave(const StreamArgs& args, const StreamRange& range, int bh, int rt)
        : a(args), r(range) {
        const int lane = threadIdx.x & 63;
        n = lane & 15;
        g = lane >> 4;
        b = bh / a.Hkv;
        hk = bh - b * a.Hkv;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = min(rt * ROWS + 16 * i + n, a.T * a.G - 1);
            const int t = row / a.G, h = hk * a.G + row - t * a.G;
            const T* qrow = (const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st;
#pragma unroll
            for (int c = 0; c < S::KF; ++c) {
                const int d = S::KW * (4 * c + g);
                q[i][c] = u32x4{0u, 0u, 0u, 0u};
                if (d < a.D) q[i][c] = *(const u32x4*)(qrow + d);
            }
#pragma unroll
            for (int j = 0; j < S::NO; ++j) o[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            m[i] = kNegInf;
            l[i] = 0.0f;
            tok[i] = t;
            limits(t, hi[i], lo[i]);
            pos[i] = (int)(r.first_pos + t);
            slope[i] = a.alibi != nullptr ? a.alibi[h] : 0.0f;
        }
        limits(r.t0, hi_min, lo_min);
        limits(r.t1, hi_max, lo_max);
        // (with padding rows in the tile the last token sees none: the rows before it set the range)
        if (!a.positions_from_end && a.lengths != nullptr && r.first_pos + r.t1 >= r.length) {
            hi_min = 0;
            hi_max = r.length;
            lo_max = 0x7fffffff;
        }
        kbase = (const char*)a.k + hk * a.k_sh * S::ES;
        vbase = (const char*)a.v + hk * a.v_sh * S::ES;
        if (!PAGED) {
            kbase += b * a.k_sp * S::ES;
            vbase += b * a.v_sp * S::ES;
        }
        koff = (unsigned)(n * (int)a.k_st * S::ES);
#pragma unroll
        for (int j = 0; j < 4; ++j) voff[j] = (unsigned)((4 * g + j) * (int)a.v_st * S::ES);
    }

    // Keys that the row of token t sees: below h, and from w on or below the sinks.
    __device__ __forceinline__ void limits(int t, int& h, int& w) const {
        const int64_t p = r.first_pos + t;
        h = (int)max((int64_t)0, min((int64_t)r.length, p + 1));
        if (!a.positions_from_end && a.lengths != nullptr && p >= r.length) h = 0;  // padding
        w = a.window > 0 ? (int)max((int64_t)-0x7fffffff, min((int64_t)0x7fffffff, p + 1 - a.window)) : -0x7fffffff;
    }

    // First keys of a step's blocks; a step past the row of blocks, or its
    // second block, repeats the last one (its keys are masked where they count).
    __device__ __forceinline__ int first_key(int step, int j) const {
        return uniform(kStreamKeys * r.block(min(step * S::NB + j, r.blocks - 1)));
    }
    __device__ __forceinline__ Pages pages(int step) const {
        Pages p;
#pragma unroll
        for (int j = 0; j < S::NB; ++j)
            p.id[j] = PAGED ? a.table[b * a.table_stride + (first_key(step, j) >> a.page_shift)] : 0;
        return p;
    }
    __device__ __forceinline__ bool page_ok(int id) const { return (unsigned)id < (unsigned)a.num_pages; }

    __device__ __forceinline__ void load(Step& s, int step, const Pages& p) const {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            const int key = first_key(step, j);
            const char* kb = kbase;
            const char* vb = vbase;
            unsigned ko = koff, vo[4] = {voff[0], voff[1], voff[2], voff[3]};
            if (PAGED) {
                // an entry outside the pool reads page 0, masked
                const int64_t page = page_ok(p.id[j]) ? uniform(p.id[j]) : 0;
                const int64_t row = key & ((1 << a.page_shift) - 1);
                kb += (page * a.k_sp + row * a.k_st) * S::ES;
                vb += (page * a.v_sp + row * a.v_st) * S::ES;
            } else {
                kb += (int64_t)key * a.k_st * S::ES;
                vb += (int64_t)key * a.v_st * S::ES;
                if (key + kStreamKeys > a.capacity) {  // rows past the end repeat the last one
                    const int last = a.capacity - 1 - key;
                    ko = (unsigned)(min(n, last) * (int)a.k_st * S::ES);
#pragma unroll
                    for (int t = 0; t < 4; ++t) vo[t] = (unsigned)(min(4 * g + t, last) * (int)a.v_st * S::ES);
                }
            }
            // columns past the head dim repeat the row's last chunk: K is
            // cleared below, V fills columns that are never stored
#pragma unroll
            for (int c = 0; c < S::KF; ++c)
                s.k[j][c] = *(const u32x4*)(kb + ko + (unsigned)(S::ES * min(S::KW * (4 * c + g), a.D - S::KW)));
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int c = 0; c < S::VC; ++c)
                    s.v[4 * j + t][c] =
                        *(const vraw*)(vb + vo[t] + (unsigned)(S::ES * min(S::VW * (16 * c + n), a.Dv - S::VW)));
        }
    }

    // V operands of a step. 16 bits: product i of chunk c holds eight keys of
    // column 8m + i. fp32: the rows as they are, product (key, chunk, i).
    using Operands = typename S::template Operands<vraw>;
    __device__ __forceinline__ void v_operands(const Step& s, Operands& vt) const {
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < S::NB * 4; ++t)
#pragma unroll
                for (int c = 0; c < S::VC; ++c) vt.v[t][c] = s.v[t][c];
        } else {
#pragma unroll
            for (int c = 0; c < S::VC; ++c)
#pragma unroll
                for (int i = 0; i < S::VW; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        vt.v[c * S::VW + i][j] = __builtin_amdgcn_perm(s.v[2 * j + 1][c][i / 2], s.v[2 * j][c][i / 2],
                                                                       i & 1 ? 0x07060302u : 0x05040100u);
        }
    }

    // Bits of the operands' keys that `h` and `w` let through (16 bits: two keys a word).
    static constexpr int MASKS = F32 ? S::NB * 4 : 4;
    __device__ __forceinline__ void key_masks(const int (&key0)[S::NB], int h, int w, unsigned (&keep)[MASKS]) const {
#pragma unroll
        for (int k = 0; k < MASKS; ++k) {
            if constexpr (F32) {
                keep[k] = key0[k / 4] >= 0 && seen(key0[k / 4] + 4 * g + k % 4, h, w) ? ~0u : 0u;
            } else {
                const int key = key0[k / 2] + 4 * g + 2 * (k & 1);
                keep[k] = key0[k / 2] < 0 ? 0u : (seen(key, h, w) ? 0xffffu : 0u) | (seen(key + 1, h, w) ? ~0xffffu : 0u);
            }
        }
    }
    __device__ __forceinline__ bool seen(int key, int h, int w) const { return key < h && (key >= w || key < a.sinks); }

    // acc += the step's products of accumulator j, with V & keep.
    template <bool MASKED>
    __device__ __forceinline__ f32x4 pv(int j, const Operands& vt, const float (&p)[S::NB * 4], u32x4 pb,
                                        const unsigned (&keep)[MASKS], f32x4 acc) const {
        if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < S::NB * 4; ++t) {
                unsigned x = vt.v[t][j / S::VW][j % S::VW];
                if (MASKED) x &= keep[t];
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), p[t], acc, 0, 0, 0);
            }
        } else {
            u32x4 x = vt.v[j];
            if (MASKED) x &= u32x4{keep[0], keep[1], keep[2], keep[3]};
            acc = S::mma(x, pb, acc);
        }
        return acc;
    }

    // SEEN: steps in which rows differ in what they see form their products once per token.
    template <bool SEEN>
    __device__ __forceinline__ void compute(Step& s, int step, const Pages& pg) {
        int key0[S::NB];  // -1: the block's keys count for nothing
        bool mask = false;
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            key0[j] = first_key(step, j);
            if (step * S::NB + j >= r.blocks || (PAGED && !page_ok(uniform(pg.id[j])))) key0[j] = -1;
            mask = mask || key0[j] < 0 || key0[j] + kStreamKeys > hi_min ||
                   (key0[j] < lo_max && key0[j] + kStreamKeys > a.sinks);
        }
        if (S::KW * 4 * S::KF > a.D) {  // K columns past the head dim
#pragma unroll
            for (int c = 0; c < S::KF; ++c)
                if (S::KW * (4 * c + g) >= a.D) {
#pragma unroll
                    for (int j = 0; j < S::NB; ++j) s.k[j][c] = u32x4{0u, 0u, 0u, 0u};
                }
        }
        Operands vt;
        v_operands(s, vt);
        unsigned keep[MASKS] = {};
        if (mask) {
            key_masks(key0, hi_max, lo_min, keep);
            vt.apply(keep);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            f32x4 sc[S::NB];
#pragma unroll
            for (int j = 0; j < S::NB; ++j) {
                sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < S::KF; ++c) {
                    if constexpr (F32) {
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __builtin_bit_cast(float, (unsigned)s.k[j][c][t]),
                                __builtin_bit_cast(float, (unsigned)q[i][c][t]), sc[j], 0, 0, 0);
                    } else {
                        sc[j] = S::mma(s.k[j][c], q[i][c], sc[j]);
                    }
                }
            }
            // scores in log2 units
            float x[S::NB * 4];
            const float to_log2 = a.scale * kLog2e;
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) x[4 * j + t] = sc[j][t] * to_log2;
            if (a.alibi != nullptr || a.softcap > 0.0f) {
#pragma unroll
                for (int j = 0; j < S::NB; ++j)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        float y = sc[j][t] * a.scale;
                        if (a.alibi != nullptr) y = __builtin_fmaf(slope[i], (float)(key0[j] + 4 * g + t - pos[i]), y);
                        if (a.softcap > 0.0f) {
                            // cap tanh(y / cap) = cap (1 - 2 / (2^u + 1)), u = 2 log2(e) y / cap
                            const float u = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e / a.softcap));
                            y = __builtin_fmaf(-2.0f * a.softcap, __builtin_amdgcn_rcpf(u + 1.0f), a.softcap);
                        }
                        x[4 * j + t] = y * kLog2e;
                    }
            }
            if (mask) {
#pragma unroll
                for (int j = 0; j < S::NB; ++j)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        if (!(key0[j] >= 0 && seen(key0[j] + 4 * g + t, hi[i], lo[i]))) x[4 * j + t] = kNegInf;
            }
            float top = x[0];
#pragma unroll
            for (int t = 1; t < S::NB * 4; ++t) top = fmaxf(top, x[t]);
            if (__builtin_amdgcn_ballot_w64(top > m[i] + kRescaleSlack) != 0) {
                top = max4(top);
                const bool raise = top > m[i] + kRescaleSlack;
                const float alpha = raise ? __builtin_amdgcn_exp2f(m[i] - top) : 1.0f;
                m[i] = raise ? top : m[i];
                l[i] *= alpha;
#pragma unroll
                for (int c = 0; c < S::NO; ++c) o[i][c] *= alpha;
            }
            const float mu = m[i] == kNegInf ? 0.0f : m[i];
            float p[S::NB * 4];
            u32x4 pb = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int t = 0; t < S::NB * 4; ++t) p[t] = __builtin_amdgcn_exp2f(x[t] - mu);
            if constexpr (F32) {
#pragma unroll
                for (int t = 0; t < S::NB * 4; ++t) l[i] += p[t];
            } else {
                typename S::P pk;
#pragma unroll
                for (int t = 0; t < 8; ++t) pk[t] = (T)p[t];
#pragma unroll
                for (int t = 0; t < 8; t += 2) l[i] = Dot2<T>::sum2(typename Dot2<T>::v2{pk[t], pk[t + 1]}, l[i]);
                pb = __builtin_bit_cast(u32x4, pk);
            }
            if (!SEEN || !mask) {
#pragma unroll
                for (int j = 0; j < S::NO; ++j) o[i][j] = pv<false>(j, vt, p, pb, keep, o[i][j]);
            } else {
                for (int t = r.t0; t <= r.t1; ++t) {
                    int h, w;
                    limits(t, h, w);
                    key_masks(key0, h, w, keep);
#pragma unroll
                    for (int j = 0; j < S::NO; ++j) {
                        const f32x4 acc = pv<true>(j, vt, p, pb, keep, o[i][j]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][j][e] = tok[i] == t ? acc[e] : o[i][j][e];
                    }
                }
            }
        }
    }

    __device__ __forceinline__ bool nan_in_o() const {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < S::NO; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad = bad || o[i][c][e] != o[i][c][e];
        return __builtin_amdgcn_ballot_w64(bad) != 0;
    }

    // This wavefront's steps: begin, begin + kWaves, ... below end.
    __device__ __forceinline__ void run(int begin, int end) {
        if (begin >= end) return;
        // loads past the last step repeat it: a branch around them would make
        // every wait one for all loads in flight
        auto clamp = [&](int step) { return min(step, end - 1); };
        if constexpr (DK <= 128) {
            Step s0, s1;
            Pages p0 = pages(begin), p1 = pages(clamp(begin + kWaves));
            load(s0, begin, p0);
            for (int step = begin; step < end; step += 2 * kWaves) {
                load(s1, clamp(step + kWaves), p1);
                const Pages p2 = pages(clamp(step + 2 * kWaves));
                compute<false>(s0, step, p0);
                if (step + kWaves >= end) break;
                load(s0, clamp(step + 2 * kWaves), p2);
                const Pages p3 = pages(clamp(step + 3 * kWaves));
                compute<false>(s1, step + kWaves, p1);
                p0 = p2;
                p1 = p3;
            }
        } else {
            run_plain<false>(begin, end);  // (two steps' K and V do not fit the registers)
        }
        if (r.t0 != r.t1 && nan_in_o()) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int c = 0; c < S::NO; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                m[i] = kNegInf;
                l[i] = 0.0f;
            }
            run_plain<true>(begin, end);
        }
    }
    template <bool SEEN>
    __device__ __forceinline__ void run_plain(int begin, int end) {
        Step s;
        Pages p0 = pages(begin);
        for (int step = begin; step < end; step += kWaves) {
            load(s, step, p0);
            const Pages p1 = pages(min(step + kWaves, end - 1));
            compute<SEEN>(s, step, p0);
            p0 = p1;
        }
    }
};

template <typename T, int DK, int RT, bool PAGED>
__global__ __launch_bounds__(kStreamThreads, 1) void stream_fwd_kernel(StreamArgs a) {
    using W = StreamWave<T, DK, RT, PAGED>;
    using S = typename W::S;
    constexpr int STATE = 64 * (4 * S::NO * RT + 2 * RT);  // floats of a wavefront's state
    __shared__ __attribute__((aligned(16))) float lds[(kWaves - 1) * STATE];
    int bh, rt, split;
    stream_work(a, blockIdx.x, bh, rt, split);
    const StreamRange r = stream_range(a, bh / a.Hkv, rt, W::ROWS);
    const int steps = (r.blocks + S::NB - 1) / S::NB;
    int per;
    const int active = stream_split(a, steps, per);
    if (split >= active) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    W w(a, r, bh, rt);
    w.run(split * per + wave, min(steps, (split + 1) * per));

    // fold the wavefronts' states into wavefront 0's
#pragma unroll
    for (int i = 0; i < RT; ++i) w.l[i] = sum4(w.l[i]);
    if (wave > 0) {
        float* st = lds + (wave - 1) * STATE;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
#pragma unroll
            for (int c = 0; c < S::NO; ++c) *(f32x4*)(st + 4 * (64 * (i * S::NO + c) + lane)) = w.o[i][c];
            st[64 * 4 * S::NO * RT + 64 * (2 * i) + lane] = w.m[i];
            st[64 * 4 * S::NO * RT + 64 * (2 * i + 1) + lane] = w.l[i];
        }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        float ms[kWaves], ls[kWaves];
        ms[0] = w.m[i];
        ls[0] = w.l[i];
        float top = w.m[i];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) {
            const float* st = lds + (k - 1) * STATE + 64 * 4 * S::NO * RT;
            ms[k] = st[64 * (2 * i) + lane];
            ls[k] = st[64 * (2 * i + 1) + lane];
            top = fmaxf(top, ms[k]);
        }
        const float mu = top == kNegInf ? 0.0f : top;
        const float keep = __builtin_amdgcn_exp2f(w.m[i] - mu);
        float sum = ls[0] * keep;
#pragma unroll
        for (int c = 0; c < S::NO; ++c) w.o[i][c] *= keep;
#pragma unroll
        for (int k = 1; k < kWaves; ++k) {
            const float f = __builtin_amdgcn_exp2f(ms[k] - mu);
            sum += f * ls[k];
#pragma unroll
            for (int c = 0; c < S::NO; ++c) {
                const f32x4 v = *(const f32x4*)(lds + (k - 1) * STATE + 4 * (64 * (i * S::NO + c) + lane));
                w.o[i][c] += f * v;
            }
        }
        // row n, columns 16 VW c + VW (4 g + e) + 0 .. VW - 1
        const int row = rt * W::ROWS + 16 * i + w.n;
        if (row >= a.T * a.G) continue;
        const int t = row / a.G, h = w.hk * a.G + row - t * a.G;
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        const int64_t off = w.b * a.o_sb + h * a.o_sh + t * a.o_st;
        const int64_t prow = (((int64_t)bh * a.row_tiles + rt) * a.splits + split) * W::ROWS + 16 * i + w.n;
#pragma unroll
        for (int c = 0; c < S::VC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * S::VW * c + S::VW * (4 * w.g + e);
                if (col >= a.Dv) continue;
                float x[S::VW];
#pragma unroll
                for (int k = 0; k < S::VW; ++k) x[k] = w.o[i][c * S::VW + k][e];
                if (active == 1) {
                    put_out<T, S::VW>(a, off + col, x, inv);
                } else {
#pragma unroll
                    for (int k = 0; k < S::VW; k += 4)
                        *(f32x4*)(a.part_o + prow * a.Dv + col + k) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
                }
            }
        if (active > 1 && w.g == 0) {
            a.part_ml[2 * prow] = top;
            a.part_ml[2 * prow + 1] = sum;
        }
    }
}

// Joins the splits of a row: a workgroup per row, groups of Dv / 4 threads
// taking the splits in turn.
template <typename T>
__global__ __launch_bounds__(kStreamThreads) void stream_join_kernel(StreamArgs a, int rows, int step_keys) {
    __shared__ float red[6 * kStreamThreads];
    const int per_head = a.T * a.G;
    const int bh = (int)(blockIdx.x / per_head), row = (int)(blockIdx.x % per_head);
    const int rt = row / rows;
    const StreamRange r = stream_range(a, bh / a.Hkv, rt, rows);
    const int steps = (r.blocks * kStreamKeys + step_keys - 1) / step_keys;
    int per;
    const int active = stream_split(a, steps, per);
    if (active == 1) return;  // written by its workgroup
    const int chunks = a.Dv / 4, c = (int)threadIdx.x % chunks, grp = (int)threadIdx.x / chunks;
    const int groups = min(active, kStreamThreads / chunks);
    const int64_t first = ((int64_t)bh * a.row_tiles + rt) * a.splits * rows + row - rt * rows;
    float m = kNegInf, l = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (grp < groups)
        for (int s = grp; s < active; s += groups) {
            const int64_t p = first + (int64_t)s * rows;
            lse_fold(m, l, acc, a.part_ml[2 * p], a.part_ml[2 * p + 1], *(const f32x4*)(a.part_o + p * a.Dv + 4 * c));
        }
    if (grp > 0 && grp < groups) {
        float* e = red + 6 * threadIdx.x;
        e[0] = m;
        e[1] = l;
#pragma unroll
        for (int j = 0; j < 4; ++j) e[2 + j] = acc[j];
    }
    __syncthreads();
    if (grp != 0) return;
    for (int k = 1; k < groups; ++k) {
        const float* e = red + 6 * (k * chunks + c);
        lse_fold(m, l, acc, e[0], e[1], f32x4{e[2], e[3], e[4], e[5]});
    }
    const int t = row / a.G, h = bh % a.Hkv * a.G + row - t * a.G;
    const float x[4] = {acc[0], acc[1], acc[2], acc[3]};
    put_out<T, 4>(a, bh / a.Hkv * a.o_sb + h * a.o_sh + t * a.o_st + 4 * c, x, l > 0.0f ? 1.0f / l : 0.0f);
}

template <typename T, int DK, int RT>
hipError_t launch_stream_rt(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * a.row_tiles * a.splits)), block(kStreamThreads);
    if (a.paged) hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, false>), grid, block, 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL((stream_join_kernel<T>), dim3((unsigned)((int64_t)a.B * a.Hkv * a.T * a.G)), block, 0, s, a,
                       16 * RT, kStreamKeys * StreamTile<T, DK>::NB);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_stream_type(const StreamArgs& a, hipStream_t s) {
    const int dk = stream_kernel_dim(a.D, a.Dv);
    const bool wide = stream_tile_rows(dk, a.T * a.G) == 32;
    switch (dk) {
        case 64: return wide ? launch_stream_rt<T, 64, 2>(a, s) : launch_stream_rt<T, 64, 1>(a, s);
        case 128: return wide ? launch_stream_rt<T, 128, 2>(a, s) : launch_stream_rt<T, 128, 1>(a, s);
        case 256: return launch_stream_rt<T, 256, 1>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

int stream_kernel_dim(int D, int Dv) {
    const int d = D > Dv ? D : Dv;
    return d <= 64 ? 64 : d <= 128 ? 128 : d <= 256 ? 256 : 0;
}

// 32 rows halve the reads of a tile; at kernel dim 256 their accumulators and
// two steps of K and V exceed the registers.
int stream_tile_rows(int kernel_dim, int rows) { return kernel_dim <= 128 && rows > 16 ? 32 : 16; }

int stream_step_keys(int dtype, int kernel_dim) { return dtype == DT_F32 && kernel_dim > 64 ? kStreamKeys : 2 * kStreamKeys; }

hipError_t launch_stream(const StreamArgs& a, int dtype, hipStream_t s) {
    switch (dtype) {
        case DT_F32: return launch_stream_type<float>(a, s);
        case DT_BF16: return launch_stream_type<__bf16>(a, s);
        case DT_F16: return launch_stream_type<_Float16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ofh
