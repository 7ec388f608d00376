// Attention of new tokens over a cached sequence: every wavefront streams keys
// of its own straight into the operand registers of the matrix instructions.
//
// What bounds it: reading K and V once (2 bytes of K and V per product of a
// row's tile, far below what the matrix cores need). So nothing goes through
// LDS. Measured: f16 B1 H32/8 of 131,000 keys D128 95 us, 5.7 TB/s, and 5 us of
// the join; bf16 B64 H32/8 of 65-4096 keys 119 us, 4.7 TB/s (the longest run on
// alone); fp32 prompts, bound by the matrix cores instead, B2 H8 N1000-2047 D64
// window 512 56 us.
// With S^T = K Q^T and O^T = V^T P^T
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
// Blocks of 16 keys never cross a page (page sizes are multiples of 16), so a
// block's page is one scalar load, made a step ahead.
//
// A tile has 16 (or 32) rows of one (sequence, key-value head): the heads of a
// group and the new tokens share what is read. The wavefronts of a workgroup
// take the steps in turn and fold their (m, l, O) in LDS. Where tiles are few,
// `splits` workgroups share a tile's steps evenly and are joined with
// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. (On ragged batches finer
// parts cost what their better balance gains, a start of 3-4 us each; shares
// of the whole work, longest sequence first, were slower still.)
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

#include <algorithm>

#include "flash_wave32.h"
#include "serving_kernels.h"
#include "serving_softcap.h"

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
    // A tile of padding rows alone takes no step. Its probabilities would be 0, and 0
    // times a NaN or an infinity in V is a NaN; and it would read and multiply for
    // nothing (fp32 B8 H8 N275-2048 D64 355 us, this 210; window 512 145, 126).
    const bool padding = !a.positions_from_end && a.lengths != nullptr && r.first_pos + r.t0 >= r.length;
    r.blocks = padding ? 0 : r.sink_blocks + max(0, nb - r.first_block);
    return r;
}

// A workgroup's share: part `part` of a tile.
struct StreamPart {
    int b, hk, rt, part;
};

// Workgroups go to the 8 XCDs in turn; where they can be dealt out evenly, the
// tiles and parts of a key-value head run on one XCD and share its L2. Late
// tokens, whose keys are most, run first.
__device__ __forceinline__ StreamPart stream_part(const StreamArgs& a, int id, int row_tiles) {
    const int n = a.B * a.Hkv, per = row_tiles * a.splits;
    StreamPart p;
    int rest, bh;
    if ((n & 7) == 0) {
        const int j = id >> 3;
        bh = j / per * 8 + (id & 7);
        rest = j % per;
    } else {
        bh = id / per;
        rest = id % per;
    }
    p.b = bh / a.Hkv;
    p.hk = bh - p.b * a.Hkv;
    p.part = rest % a.splits;
    p.rt = row_tiles - 1 - rest / a.splits;
    return p;
}

// Parts of a tile of `steps` steps, and the steps of each.
__device__ __forceinline__ int stream_parts(const StreamArgs& a, int steps, int& per) {
    const int n = max(1, min(a.splits, steps / a.min_steps));
    per = max(1, (steps + n - 1) / n);
    return max(1, (steps + per - 1) / per);
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

// How the wavefronts of a workgroup share: a tile's steps among them (kTile), of
// which the workgroup has a part (kPart), or a tile each (kOwn).
enum StreamMode { kTile, kPart, kOwn };

template <typename T, int DK, int RT, bool PAGED, int STRIDE>
struct StreamWave {
    using S = StreamTile<T, DK>;
    static constexpr int ROWS = 16 * RT;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int VB = S::VW * S::ES;  // bytes of a lane's V chunk: 16 or 8
    static constexpr int VD = VB / 4;         // dwords
    typedef unsigned int vraw __attribute__((ext_vector_type(VD)));

    struct StepK {  // K and V of a step as loaded
        u32x4 k[S::NB][S::KF];
    };
    struct StepV {
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

    __device__ __forceinline__ StreamWave(const StreamArgs& args, const StreamRange& range, const StreamPart& at)
        : a(args), r(range), b(at.b), hk(at.hk) {
        const int rt = at.rt;
        const int lane = threadIdx.x & 63;
        n = lane & 15;
        g = lane >> 4;
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

    // Address of the first row of a block, rows `stride` elements apart and pages
    // `page_stride`; an entry outside the pool reads page 0, masked.
    __device__ __forceinline__ const char* block_at(const char* base, int key, int page, int64_t page_stride,
                                                    int64_t stride) const {
        if (!PAGED) return base + (int64_t)key * stride * S::ES;
        const int64_t id = page_ok(page) ? uniform(page) : 0;
        return base + (id * page_stride + (int64_t)(key & ((1 << a.page_shift) - 1)) * stride) * S::ES;
    }
    // Contiguous rows past the end repeat the last one: the rows of the block.
    __device__ __forceinline__ int last_row(int key) const {
        return PAGED ? kStreamKeys - 1 : min(kStreamKeys - 1, a.capacity - 1 - key);
    }
    // (Columns past the head dim repeat the row's last chunk: K is cleared before
    // its product, V fills columns that are never stored.)
    __device__ __forceinline__ void load_k(StepK& s, int step, const Pages& p) const {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            const int key = first_key(step, j), last = last_row(key);
            const char* kb = block_at(kbase, key, p.id[j], a.k_sp, a.k_st);
            const unsigned ko = last == kStreamKeys - 1 ? koff : (unsigned)(min(n, last) * (int)a.k_st * S::ES);
#pragma unroll
            for (int c = 0; c < S::KF; ++c)
                s.k[j][c] = *(const u32x4*)(kb + ko + (unsigned)(S::ES * min(S::KW * (4 * c + g), a.D - S::KW)));
        }
    }
    __device__ __forceinline__ void load_v(StepV& s, int step, const Pages& p) const {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            const int key = first_key(step, j), last = last_row(key);
            const char* vb = block_at(vbase, key, p.id[j], a.v_sp, a.v_st);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const unsigned vo =
                    last == kStreamKeys - 1 ? voff[t] : (unsigned)(min(4 * g + t, last) * (int)a.v_st * S::ES);
#pragma unroll
                for (int c = 0; c < S::VC; ++c)
                    s.v[4 * j + t][c] = *(const vraw*)(vb + vo + (unsigned)(S::ES * min(S::VW * (16 * c + n), a.Dv - S::VW)));
            }
        }
    }

    // V operands of a step. 16 bits: product i of chunk c holds eight keys of
    // column 8m + i. fp32: the rows as they are, product (key, chunk, i).
    using Operands = typename S::template Operands<vraw>;
    __device__ __forceinline__ void v_operands(const StepV& s, Operands& vt) const {
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

    // S^T = K Q^T of row tile i.
    __device__ __forceinline__ void scores(const StepK& s, int i, f32x4 (&sc)[S::NB]) const {
#pragma unroll
        for (int j = 0; j < S::NB; ++j) {
            sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < S::KF; ++c) {
                if constexpr (F32) {
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (unsigned)s.k[j][c][t]),
                                                                     __builtin_bit_cast(float, (unsigned)q[i][c][t]),
                                                                     sc[j], 0, 0, 0);
                } else {
                    sc[j] = S::mma(s.k[j][c], q[i][c], sc[j]);
                }
            }
        }
    }

    // Scores of row tile i -> probabilities against the running max: p, and in 16
    // bits their operand pb; m, l and O are brought to that max.
    __device__ __forceinline__ void softmax(int i, const f32x4 (&sc)[S::NB], const int (&key0)[S::NB], bool mask,
                                            float (&p)[S::NB * 4], u32x4& pb) {
        // scores in log2 units
        float x[S::NB * 4];
        const float to_log2 = a.scale * kLog2e;
#pragma unroll
        for (int j = 0; j < S::NB; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) x[4 * j + t] = sc[j][t] * to_log2;
        if (!F32 && a.softcap > kCapExp) {
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float y = sc[j][t] * a.scale;
                    if (a.alibi != nullptr) y = __builtin_fmaf(slope[i], (float)(key0[j] + 4 * g + t - pos[i]), y);
                    x[4 * j + t] = cap_tanh_wide(y, a.softcap) * kLog2e;
                }
        } else if (a.alibi != nullptr || a.softcap > 0.0f) {
#pragma unroll
            for (int j = 0; j < S::NB; ++j)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float y = sc[j][t] * a.scale;
                    if (a.alibi != nullptr) y = __builtin_fmaf(slope[i], (float)(key0[j] + 4 * g + t - pos[i]), y);
                    if (a.softcap > 0.0f) y = F32 ? cap_tanh(y, a.softcap) : cap_tanh16(y, a.softcap);
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
    }

    // The steps begin, begin + STRIDE, ... below end. K's registers take the next
    // step's rows once its products are formed, V's once its operands are: loads
    // are in flight all the time without a second set of registers. Loads past
    // the last step repeat it (a branch around them would make every wait one for
    // all loads in flight).
    // SEEN: steps in which rows differ in what they see form their products once per token.
    template <bool SEEN>
    __device__ __forceinline__ void run_steps(int begin, int end) {
        StepK sk;
        StepV sv;
        Pages pg = pages(begin);
        load_k(sk, begin, pg);
        load_v(sv, begin, pg);
        Pages pn = pages(min(begin + STRIDE, end - 1));
        for (int step = begin; step < end; step += STRIDE) {
            const int next = min(step + STRIDE, end - 1);
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
                        for (int j = 0; j < S::NB; ++j) sk.k[j][c] = u32x4{0u, 0u, 0u, 0u};
                    }
            }
            f32x4 sc[RT][S::NB];
#pragma unroll
            for (int i = 0; i < RT; ++i) scores(sk, i, sc[i]);
            load_k(sk, next, pn);
            float p[RT][S::NB * 4];
            u32x4 pb[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) softmax(i, sc[i], key0, mask, p[i], pb[i]);
            Operands vt;
            v_operands(sv, vt);
            load_v(sv, next, pn);
            pg = pn;
            pn = pages(min(step + 2 * STRIDE, end - 1));
            unsigned keep[MASKS] = {};
            if (mask) {
                key_masks(key0, hi_max, lo_min, keep);
                vt.apply(keep);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (!SEEN || !mask) {
#pragma unroll
                    for (int j = 0; j < S::NO; ++j) o[i][j] = pv<false>(j, vt, p[i], pb[i], keep, o[i][j]);
                } else {
                    for (int t = r.t0; t <= r.t1; ++t) {
                        int h, w;
                        limits(t, h, w);
                        key_masks(key0, h, w, keep);
#pragma unroll
                        for (int j = 0; j < S::NO; ++j) {
                            const f32x4 acc = pv<true>(j, vt, p[i], pb[i], keep, o[i][j]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[i][j][e] = tok[i] == t ? acc[e] : o[i][j][e];
                        }
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

    // This wavefront's steps: begin, begin + STRIDE, ... below end.
    __device__ __forceinline__ void run(int begin, int end) {
        if (begin >= end) return;
        run_steps<false>(begin, end);
        if (r.t0 != r.t1 && nan_in_o()) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int c = 0; c < S::NO; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                m[i] = kNegInf;
                l[i] = 0.0f;
            }
            run_steps<true>(begin, end);
        }
    }
};

// Joins the parts of every row: O = sum_s w_s O_s / sum_s w_s l_s with w_s =
// 2^(m_s - max m). A wavefront takes 32 columns of a row: lane c + 8 g has four
// columns of parts g, g + 8, ..., four of them in flight, and the eight lane
// groups are folded with lane exchanges, so the order of the sums depends on
// the number of parts alone. It reads every slot, without the lengths that say
// which were used (a part without steps leaves max -inf and sum 0): one memory
// round trip instead of two. (Joining in the workgroup that ends last, with
// coherent stores and loads, took 3 us longer than this launch.)
template <typename T>
__global__ __launch_bounds__(kStreamThreads) void stream_join_kernel(StreamArgs a, int tile_rows) {
    constexpr int G = 4;
    const int lane = threadIdx.x & 63, grp = lane >> 3;
    const int chunks = a.Dv / 4, blocks = (chunks + 7) / 8, rows = a.T * a.G;
    const int64_t item = (int64_t)blockIdx.x * (kStreamThreads / 64) + uniform(threadIdx.x >> 6);
    const int64_t at = item / blocks;  // row of all heads
    const int bh = (int)(at / rows), row = (int)(at - (int64_t)bh * rows);
    if (bh >= a.B * a.Hkv) return;
    const int c = 8 * (int)(item - at * blocks) + (lane & 7), cc = min(c, chunks - 1);
    const int rt = row / tile_rows;
    const int64_t first = ((int64_t)bh * a.row_tiles + rt) * a.splits * tile_rows + row - rt * tile_rows;
    float m = kNegInf, l = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = grp; s < a.splits; s += 8 * G) {
        float ms[G], ls[G];
        f32x4 os[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int64_t p = first + (int64_t)(s + 8 * j < a.splits ? s + 8 * j : s) * tile_rows;
            ms[j] = a.part_ml[2 * p];
            ls[j] = a.part_ml[2 * p + 1];
            os[j] = *(const f32x4*)(a.part_o + p * a.Dv + 4 * cc);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
            if (s + 8 * j >= a.splits) ms[j] = kNegInf;
            // (O of a part without steps was not written; a NaN sum stays)
            const bool none = ms[j] == kNegInf && !(ls[j] != ls[j]);
            lse_fold(m, l, acc, ms[j], none ? 0.0f : ls[j], none ? f32x4{0.f, 0.f, 0.f, 0.f} : os[j]);
        }
    }
#pragma unroll
    for (int d = 8; d < 64; d *= 2) {
        const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d);
        f32x4 o2;
#pragma unroll
        for (int j = 0; j < 4; ++j) o2[j] = __shfl_xor(acc[j], d);
        lse_fold(m, l, acc, m2, l2, o2);
    }
    if (grp == 0 && c < chunks) {
        const int t = row / a.G, h = bh % a.Hkv * a.G + row - t * a.G;
        const float x[4] = {acc[0], acc[1], acc[2], acc[3]};
        put_out<T, 4>(a, bh / a.Hkv * a.o_sb + h * a.o_sh + t * a.o_st + 4 * c, x, l > 0.0f ? 1.0f / l : 0.0f);
    }
}

template <typename T, int DK, int RT, bool PAGED, int MODE>
__global__
__launch_bounds__(kStreamThreads, DK > 128 || (RT == 2 && DK * sizeof(T) >= 256) ? 1 : 2)
void stream_fwd_kernel(StreamArgs a) {
    using W = StreamWave<T, DK, RT, PAGED, MODE == kOwn ? 1 : kWaves>;
    constexpr bool SPLIT = MODE == kPart;
    using S = typename W::S;
    constexpr int STATE = 64 * (4 * S::NO * RT + 2 * RT);  // floats of a wavefront's state
    __shared__ __attribute__((aligned(16))) float lds[MODE == kOwn ? 1 : (kWaves - 1) * STATE];
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    StreamPart at = stream_part(a, blockIdx.x, MODE == kOwn ? (a.row_tiles + kWaves - 1) / kWaves : a.row_tiles);
    if (MODE == kOwn) {
        at.rt = at.rt * kWaves + wave;
        if (at.rt >= a.row_tiles) return;
    }
    const StreamRange r = stream_range(a, at.b, at.rt, W::ROWS);
    const int steps = (r.blocks + S::NB - 1) / S::NB;
    const int64_t slot = (((int64_t)at.b * a.Hkv + at.hk) * a.row_tiles + at.rt) * a.splits + at.part;
    int per = steps;
    if (SPLIT && at.part >= stream_parts(a, steps, per)) {
        // no steps: what the join reads of this part
        if ((int)threadIdx.x < W::ROWS) {
            a.part_ml[2 * (slot * W::ROWS + threadIdx.x)] = kNegInf;
            a.part_ml[2 * (slot * W::ROWS + threadIdx.x) + 1] = 0.0f;
        }
        return;
    }
    W w(a, r, at);
    w.run(at.part * per + (MODE == kOwn ? 0 : wave), min(steps, (at.part + 1) * per));

    // fold the wavefronts' states into wavefront 0's
#pragma unroll
    for (int i = 0; i < RT; ++i) w.l[i] = sum4(w.l[i]);
    if (MODE != kOwn && wave > 0) {
        float* st = lds + (wave - 1) * STATE;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
#pragma unroll
            for (int c = 0; c < S::NO; ++c) *(f32x4*)(st + 4 * (64 * (i * S::NO + c) + lane)) = w.o[i][c];
            st[64 * 4 * S::NO * RT + 64 * (2 * i) + lane] = w.m[i];
            st[64 * 4 * S::NO * RT + 64 * (2 * i + 1) + lane] = w.l[i];
        }
    }
    if (MODE != kOwn) {
        __syncthreads();
        if (wave != 0) return;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        float top = w.m[i], sum = w.l[i];
        if constexpr (MODE != kOwn) {
            float ms[kWaves], ls[kWaves];
            ms[0] = w.m[i];
            ls[0] = w.l[i];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) {
                const float* st = lds + (k - 1) * STATE + 64 * 4 * S::NO * RT;
                ms[k] = st[64 * (2 * i) + lane];
                ls[k] = st[64 * (2 * i + 1) + lane];
                top = fmaxf(top, ms[k]);
            }
            const float mu = top == kNegInf ? 0.0f : top;
            const float keep = __builtin_amdgcn_exp2f(w.m[i] - mu);
            sum = ls[0] * keep;
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
        }
        // row n, columns 16 VW c + VW (4 g + e) + 0 .. VW - 1
        const int row = at.rt * W::ROWS + 16 * i + w.n;
        if (row >= a.T * a.G) continue;
        const int t = row / a.G, h = w.hk * a.G + row - t * a.G;
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        const int64_t off = w.b * a.o_sb + h * a.o_sh + t * a.o_st;
        const int64_t prow = slot * W::ROWS + 16 * i + w.n;
#pragma unroll
        for (int c = 0; c < S::VC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = 16 * S::VW * c + S::VW * (4 * w.g + e);
                if (col >= a.Dv) continue;
                float x[S::VW];
#pragma unroll
                for (int k = 0; k < S::VW; ++k) x[k] = w.o[i][c * S::VW + k][e];
                if (!SPLIT) {
                    put_out<T, S::VW>(a, off + col, x, inv);
                } else {
#pragma unroll
                    for (int k = 0; k < S::VW; k += 4)
                        *(f32x4*)(a.part_o + prow * a.Dv + col + k) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
                }
            }
        if (SPLIT && w.g == 0) {
            a.part_ml[2 * prow] = top;
            a.part_ml[2 * prow + 1] = sum;
        }
    }
}
template <typename T, int DK, int RT, int MODE>
hipError_t launch_stream_mode(const StreamArgs& a, hipStream_t s) {
    const int per_head = MODE == kOwn ? (a.row_tiles + kWaves - 1) / kWaves : a.row_tiles * a.splits;
    const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * per_head)), block(kStreamThreads);
    if (a.paged) hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, true, MODE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, false, MODE>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <typename T, int DK, int RT>
hipError_t launch_stream_rt(const StreamArgs& a, hipStream_t s) {
    if (a.splits == 1) {
        // Enough tiles for every SIMD's wavefront to have one: nothing to fold.
        // Without a window the last tiles, whose keys are most, would end alone
        // (us, a workgroup per tile / a wavefront per tile: f32 D64 B2 H8 N2047
        // window 512 69 / 59, B4 H16 N4096 window 1024 737 / 673; causal B2 H8 N2048
        // 110 / 177; 1024 tiles, B1 H8 N2047 window 512, 37 / 32; 500 tiles, N1000
        // window 256, 16 / 20, D128 B1 H4 N2000 26 / 37. A padded batch
        // has fewer tiles with work, which is not known here: B2 H8 N1000-2047
        // window 512 51 / 56, B8 N275-2048 148 / 126).
        if constexpr (RT == 2 || DK == 256 || sizeof(T) == 4)
            if (a.window > 0 && a.row_tiles >= kWaves && (int64_t)a.B * a.Hkv * a.row_tiles >= 4 * kComputeUnits)
                return launch_stream_mode<T, DK, RT, kOwn>(a, s);
        return launch_stream_mode<T, DK, RT, kTile>(a, s);
    }
    hipError_t e = launch_stream_mode<T, DK, RT, kPart>(a, s);
    if (e != hipSuccess) return e;
    const int64_t items = (int64_t)a.B * a.Hkv * a.T * a.G * ((a.Dv + 31) / 32);
    hipLaunchKernelGGL((stream_join_kernel<T>), dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(kStreamThreads), 0,
                       s, a, 16 * RT);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_stream_type(const StreamArgs& a, hipStream_t s) {
    const int dk = stream_kernel_dim(a.D, a.Dv);
    const bool wide = stream_tile_rows(sizeof(T) == 4 ? DT_F32 : DT_BF16, dk, a.T * a.G) == 32;
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

// 32 rows halve what tiles read: bf16 B16 H64/8 D128, 4 tokens, N500-8000 86 us
// against 109 with 16; f32 187 against 219. At kernel dim 256 their accumulators
// exceed the registers, and many fp32 rows (prompts) are bound by the products,
// which two wavefronts of 16 rows per SIMD overlap better: D64 B4 H16 N4096 window
// 1024 707 us, with 16 rows 673.
int stream_tile_rows(int dtype, int kernel_dim, int rows) {
    return kernel_dim > 128 || rows <= 16 || (dtype == DT_F32 && rows > 256) ? 16 : 32;
}

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
