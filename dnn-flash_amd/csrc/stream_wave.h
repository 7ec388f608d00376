// Device code of the streaming attention kernels (stream_fwd.hip has the
// design): one wavefront's rows against keys that it loads itself, and the join of
// a tile's parts. Shared by the kernels that differ in which keys their rows
// read. Internal header, included by the HIP translation units.
#pragma once

#include <algorithm>
#include <type_traits>

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

// What a row tile reads: 16-key blocks [sink_first, sink_first + sink_blocks) and,
// from first_block on, the window's; numbered in one row (block()).
struct StreamRange {
    int length;                     // keys of the sequence
    int64_t first_pos;              // position of token 0
    int t0, t1;                     // tokens of the tile
    int sink_blocks, first_block, blocks;
    int sink_first;
    // kPrefix: rows of the group, its first sequence, and what its rows see together
    int rows, start, hi_min, hi_max, lo_min, lo_max;
    template <int SRC>
    __device__ __forceinline__ int block(int i) const {
        if (SRC == kTail) return i < sink_blocks ? i + sink_first : i - sink_blocks + first_block;
        return i < sink_blocks ? i : i - sink_blocks + first_block;
    }
};

// Keys that every sequence of b's group reads from the group's pages.
__device__ __forceinline__ int stream_shared(const StreamArgs& a, int b) {
    return max(0, min(a.shared[b], a.capacity)) >> a.page_shift << a.page_shift;
}

template <int SRC>
__device__ __forceinline__ StreamRange stream_range(const StreamArgs& a, int b, int rt, int rows) {
    StreamRange r;
    r.length = a.capacity;
    if (SRC == kSelected) {
        // the keys up to the token, of which it sees the selected pages'
        const int seq = b / a.tokens;
        r.length = max(0, max(0, min(a.lengths[seq], a.capacity)) - a.tokens + b - seq * a.tokens + 1);
        r.first_pos = (int64_t)r.length - 1;
        r.t0 = r.t1 = 0;
        r.sink_blocks = r.first_block = r.sink_first = 0;
        r.blocks = min(a.num_selected, (r.length + (1 << a.page_shift) - 1) >> a.page_shift) << (a.page_shift - 4);
        return r;
    }
    if (a.lengths != nullptr) r.length = max(0, min(a.lengths[b], a.capacity));
    r.first_pos = a.positions_from_end ? (int64_t)r.length - a.T : a.query_offset;
    r.t0 = rt * rows / a.G;
    r.t1 = min(a.T - 1, (rt * rows + rows - 1) / a.G);
    // keys below `end` can be seen, and with a window those from `begin` on
    int64_t last = r.first_pos + r.t1;
    if (!a.positions_from_end && a.lengths != nullptr) last = min(last, (int64_t)r.length - 1);  // padding rows see none
    const int end = (int)max((int64_t)0, min((int64_t)r.length, last + 1));
    int begin = a.window > 0 ? (int)min((int64_t)end, max((int64_t)0, r.first_pos + r.t0 + 1 - a.window)) : 0;
    r.sink_first = 0;
    if (SRC == kTail) {
        const int shared = stream_shared(a, b);
        begin = max(begin, shared);
        r.sink_first = shared / kStreamKeys;
    }
    const int nb = (end + kStreamKeys - 1) / kStreamKeys;
    r.first_block = begin / kStreamKeys;
    r.sink_blocks = 0;
    if (a.window > 0) {
        if (SRC == kTail) {
            r.sink_blocks = max(0, min((min(a.sinks, end) + kStreamKeys - 1) / kStreamKeys, nb) - r.sink_first);
            r.first_block = max(r.first_block, r.sink_first + r.sink_blocks);
        } else {
            r.sink_blocks = min((min(a.sinks, end) + kStreamKeys - 1) / kStreamKeys, nb);
            r.first_block = max(r.first_block, r.sink_blocks);
        }
    }
    // A tile of padding rows alone takes no step. Its probabilities would be 0, and 0
    // times a NaN or an infinity in V is a NaN; and it would read and multiply for
    // nothing (fp32 B8 H8 N275-2048 D64 355 us, this 210; window 512 145, 126).
    const bool padding = !a.positions_from_end && a.lengths != nullptr && r.first_pos + r.t0 >= r.length;
    r.blocks = padding ? 0 : r.sink_blocks + max(0, nb - r.first_block);
    return r;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x = min(x, __shfl_xor(x, d));
    return uniform(x);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// Group of a prefix tile: tiles are counted group by group, of which those that
// share nothing have none. False past the last tile.
struct PrefixTile {
    int start, count, shared, rt;  // sequences of the group, its shared keys, the tile's number in it
};
__device__ __forceinline__ bool prefix_tile(const StreamArgs& a, int tile, int rows, PrefixTile& p) {
    const int lane = threadIdx.x & 63;
    if (a.groups == 1) {
        p = PrefixTile{0, a.B, stream_shared(a, 0), tile};
        return p.shared > 0 && (int64_t)tile * rows < (int64_t)a.B * a.T * a.G;
    }
    for (int base = 0; base < a.groups; base += 64) {
        const int g = base + lane;
        int start = 0, end = 0, shared = 0;
        if (g < a.groups) {
            start = g == 0 ? 0 : max(0, min(a.group_starts[g], a.B));
            end = g == a.groups - 1 ? a.B : max(0, min(a.group_starts[g + 1], a.B));
            if (start < end) shared = stream_shared(a, start);
        }
        const int count = shared > 0 ? end - start : 0;
        const int tiles = (int)(((int64_t)count * a.T * a.G + rows - 1) / rows);
        int upto = tiles;  // of the groups so far
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > tile);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            p.start = uniform(__shfl(start, at));
            p.count = uniform(__shfl(count, at));
            p.shared = uniform(__shfl(shared, at));
            p.rt = tile - uniform(__shfl(upto - tiles, at));
            return true;
        }
        tile -= uniform(__shfl(upto, 63));
    }
    return false;
}
// Row `row` of a group's rows: sequence, token, head of the key-value head's group.
struct PrefixRow {
    int b, t, g;
};
__device__ __forceinline__ PrefixRow prefix_row(const StreamArgs& a, const PrefixTile& p, int row) {
    const int per = a.T * a.G, s = row / per, rest = row - s * per, t = rest / a.G;
    return PrefixRow{p.start + s, t, rest - t * a.G};
}
// What a row sees of the shared keys: below hi, and from lo on or below the sinks.
__device__ __forceinline__ int prefix_limits(const StreamArgs& a, const PrefixTile& p, const PrefixRow& x, int& hi, int& lo) {
    const int pos = max(0, min(a.lengths[x.b], a.capacity)) - a.T + x.t;
    hi = max(0, min(p.shared, pos + 1));
    lo = a.window > 0 ? max(pos, -1) + 1 - a.window : -0x7fffffff;  // (before -1 none is seen: hi)
    return pos;
}
// Row of all heads, in which the prefix's partial rows are kept.
__device__ __forceinline__ int64_t row_of_all(const StreamArgs& a, int b, int hk, int t, int g) {
    return (((int64_t)b * a.Hkv + hk) * a.T + t) * a.G + g;
}

// Blocks that a tile of rows reads, from what its rows see.
__device__ __forceinline__ StreamRange prefix_range(const StreamArgs& a, const PrefixTile& p, int rows) {
    StreamRange r;
    const int lane = threadIdx.x & 63;
    r.length = p.shared;
    r.first_pos = 0;
    r.t0 = r.t1 = 0;
    r.start = p.start;
    r.rows = p.count * a.T * a.G;
    int hi, lo;
    prefix_limits(a, p, prefix_row(a, p, min(p.rt * rows + min(lane, rows - 1), r.rows - 1)), hi, lo);
    r.hi_min = wave_min(hi);
    r.hi_max = wave_max(hi);
    r.lo_min = wave_min(lo);
    r.lo_max = wave_max(lo);
    const int nb = (r.hi_max + kStreamKeys - 1) / kStreamKeys;
    r.sink_first = r.sink_blocks = 0;
    r.first_block = max(0, min(r.lo_min, r.hi_max)) / kStreamKeys;
    if (a.window > 0) {
        r.sink_blocks = min((min(a.sinks, r.hi_max) + kStreamKeys - 1) / kStreamKeys, nb);
        r.first_block = max(r.first_block, r.sink_blocks);
    }
    r.blocks = r.sink_blocks + max(0, nb - r.first_block);
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

// Prefix tiles: the tiles of all groups (rt) of a key-value head, and their parts.
// The tiles that read the same keys, those of a part of a head, run on one XCD, side
// by side: what one reads the others find in its cache. Parts and heads are dealt
// out to the eight XCDs in turn (the grid is filled up to eights: false past the last).
__device__ __forceinline__ bool prefix_part(const StreamArgs& a, int id, StreamPart& p) {
    const int j = id >> 3, round = j / a.prefix_tiles, unit = 8 * round + (id & 7);
    p.b = 0;
    p.rt = j - round * a.prefix_tiles;
    p.part = unit / a.Hkv;
    p.hk = unit - p.part * a.Hkv;
    return p.part < a.prefix_splits;
}

// One launch of prefix workgroups and of the sequences' own (kTail): by turns one of
// each per CU while both last, since the ones compute and the others read. (Eight and
// eight, one per XCD, puts each kind on every other CU.) True for a prefix workgroup;
// id is its number, or the other's.
__device__ __forceinline__ bool shared_workgroup(const StreamArgs& a, int block, int& id) {
    const int prefix = (int)prefix_grid(a), tail = (int)((tail_grid(a) + 7) / 8 * 8);
    const int turns = min(prefix, tail) / kComputeUnits, turn = block / (2 * kComputeUnits);
    const int rest = block - turn * 2 * kComputeUnits;
    if (turn < turns) {
        id = turn * kComputeUnits + rest % kComputeUnits;
        return rest < kComputeUnits;
    }
    // what is left: the prefix's, then the others
    const int left = block - turns * 2 * kComputeUnits, prefix_left = prefix - turns * kComputeUnits;
    id = turns * kComputeUnits + (left < prefix_left ? left : left - prefix_left);
    return left < prefix_left;
}

// Parts of a tile of `steps` steps (at most `splits`, of min_steps each), and the steps of each.
__device__ __forceinline__ int stream_parts(int splits, int min_steps, int steps, int& per) {
    const int n = max(1, min(splits, steps / min_steps));
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

template <typename T, int DK, int RT, int SRC, int STRIDE>
struct StreamWave {
    using S = StreamTile<T, DK>;
    static constexpr bool PAGED = SRC != kContiguous;
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
        int key[SRC == kSelected ? S::NB : 1];  // selected pages: the blocks' first keys
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
    // kSelected: entries listed + lane of the row's list: the entry's first key, and its
    // page (-1: selects nothing). 64 lanes look them up at once; one after the other,
    // list and table were two memory round trips for every step.
    int listed, listed_key, listed_page;

    __device__ __forceinline__ StreamWave(const StreamArgs& args, const StreamRange& range, const StreamPart& at,
                                          const PrefixTile& pt)
        : a(args), r(range), b(at.b), hk(at.hk) {
        const int rt = at.rt;
        const int lane = threadIdx.x & 63;
        n = lane & 15;
        g = lane >> 4;
        if constexpr (SRC == kPrefix) {
            b = pt.start;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const PrefixRow x = prefix_row(a, pt, min(pt.rt * ROWS + 16 * i + n, r.rows - 1));
                const int h = hk * a.G + x.g;
                load_q(i, (const T*)a.q + x.b * a.q_sb + h * a.q_sh + x.t * a.q_st);
                pos[i] = prefix_limits(a, pt, x, hi[i], lo[i]);
                slope[i] = a.alibi != nullptr ? a.alibi[h] : 0.0f;
                tok[i] = 0;
            }
            hi_min = r.hi_min;
            hi_max = r.hi_max;
            lo_min = r.lo_min;
            lo_max = r.lo_max;
            start_pointers();
            return;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = min(rt * ROWS + 16 * i + n, a.T * a.G - 1);
            const int t = row / a.G, h = hk * a.G + row - t * a.G;
            const T* qrow = (const T*)a.q + b * a.q_sb + h * a.q_sh + t * a.q_st;
            if constexpr (SRC == kSelected) {
                const int seq = b / a.tokens;
                load_q(i, (const T*)a.q + seq * a.q_sb + h * a.q_sh + (b - seq * a.tokens) * a.q_st);
            } else if constexpr (PAGED) {
                load_q(i, qrow);
            } else {
                // (load_q written out: the call moves the registers of the kernels that
                // spill; f32 B2 H16/4 N1500 D256 710 us, 755 with it. Written out for
                // pages too, those spill 95 times instead of 71.)
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
            }
            tok[i] = t;
            limits(t, hi[i], lo[i]);
            pos[i] = (int)(r.first_pos + t);
            slope[i] = a.alibi != nullptr ? a.alibi[h] : 0.0f;
        }
        if constexpr (SRC == kSelected) look_up(0);
        limits(r.t0, hi_min, lo_min);
        limits(r.t1, hi_max, lo_max);
        // (with padding rows in the tile the last token sees none: the rows before it set the range)
        if (!a.positions_from_end && a.lengths != nullptr && r.first_pos + r.t1 >= r.length) {
            hi_min = 0;
            hi_max = r.length;
            lo_max = 0x7fffffff;
        }
        start_pointers();
    }

    __device__ __forceinline__ void load_q(int i, const T* qrow) {
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
    }
    __device__ __forceinline__ void start_pointers() {
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
    __device__ __forceinline__ int first_key(int step, int j, const Pages& p) const {
        if (SRC == kSelected) return p.key[j];
        return uniform(kStreamKeys * r.template block<SRC>(min(step * S::NB + j, r.blocks - 1)));
    }
    // An entry outside the table's row, or not above the one before it, selects nothing.
    __device__ __forceinline__ void look_up(int first) {
        listed = first;
        const int e = min(first + (int)(threadIdx.x & 63), a.num_selected - 1), seq = b / a.tokens;
        const int32_t* list = a.selected + (((int64_t)seq * a.Hkv + hk) * a.tokens + b - seq * a.tokens) * a.num_selected;
        const int page = list[e], before = e > 0 ? list[e - 1] : -1;
        const bool ok = page > before && page < a.capacity >> a.page_shift;
        listed_key = ok ? page << a.page_shift : 0;
        const int id = a.table[seq * a.table_stride + (listed_key >> a.page_shift)];
        listed_page = ok ? id : -1;
    }
    __device__ __forceinline__ Pages pages(int step) {
        Pages p;
        if constexpr (SRC == kSelected) {
            const int shift = a.page_shift - 4;
#pragma unroll
            for (int j = 0; j < S::NB; ++j) {
                const int i = uniform(min(step * S::NB + j, r.blocks - 1)), e = i >> shift;
                if (e < listed || e >= listed + 64) look_up(e);
                p.key[j] = __builtin_amdgcn_readlane(listed_key, e - listed) + kStreamKeys * (i - (e << shift));
                p.id[j] = __builtin_amdgcn_readlane(listed_page, e - listed);
            }
            return p;
        }
#pragma unroll
        for (int j = 0; j < S::NB; ++j)
            p.id[j] = PAGED ? a.table[b * a.table_stride + (first_key(step, j, p) >> a.page_shift)] : 0;
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
            const int key = first_key(step, j, p), last = last_row(key);
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
            const int key = first_key(step, j, p), last = last_row(key);
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
                key0[j] = first_key(step, j, pg);
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
                } else if constexpr (SRC == kPrefix) {
                    for (int row = 0; row < 16; ++row) {
                        key_masks(key0, __shfl(hi[i], row), __shfl(lo[i], row), keep);
#pragma unroll
                        for (int j = 0; j < S::NO; ++j) {
                            const f32x4 acc = pv<true>(j, vt, p[i], pb[i], keep, o[i][j]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[i][j][e] = n == row ? acc[e] : o[i][j][e];
                        }
                    }
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
        if ((SRC == kPrefix ? hi_min != hi_max || lo_min != lo_max : r.t0 != r.t1) && nan_in_o()) {
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
//
// kTail: the parts of what the row's group shares stand before its own.
template <typename T, int SRC>
__global__ __launch_bounds__(kStreamThreads) void stream_join_kernel(StreamArgs a, int tile_rows) {
    constexpr int G = 4;
    const int lane = threadIdx.x & 63, grp = lane >> 3;
    const int chunks = a.Dv / 4, blocks = (chunks + 7) / 8, rows = a.T * a.G;
    // (below 2^26 by the launch's limit; the older two keep their code)
    using Item = typename std::conditional<SRC == kTail || SRC == kSelected, unsigned, int64_t>::type;
    const Item item = (Item)blockIdx.x * (kStreamThreads / 64) + uniform(threadIdx.x >> 6);
    const Item at = item / blocks;  // row of all heads
    const int bh = (int)(at / rows), row = (int)(at - (int64_t)bh * rows);
    if (bh >= a.B * a.Hkv) return;
    const int c = 8 * (int)(item - at * blocks) + (lane & 7), cc = min(c, chunks - 1);
    const int rt = row / tile_rows;
    const int64_t first = ((int64_t)bh * a.row_tiles + rt) * a.splits * tile_rows + row - rt * tile_rows;
    float m = kNegInf, l = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if constexpr (SRC == kTail || SRC == kSelected) {
        // one list of parts, whose loads do not wait for each other or for the group's keys
        const int before = SRC == kTail ? a.prefix_splits : 0;
        const int64_t total = (int64_t)a.B * a.Hkv * rows;
        const int n = before + a.splits;
        const bool shares = SRC == kTail && stream_shared(a, bh / a.Hkv) > 0;
        auto take = [&](int s0, auto count) {
            constexpr int C = decltype(count)::value;
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            f32x2 ml[C];
            f32x4 os[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int s = min(s0 + 8 * j + grp, n - 1), own = s - before;
                const int64_t p = own < 0 ? s * total + at : first + (int64_t)own * tile_rows;
                ml[j] = *(const f32x2*)((own < 0 ? a.prefix_ml : a.part_ml) + 2 * p);
                os[j] = *(const f32x4*)((own < 0 ? a.prefix_o : a.part_o) + p * a.Dv + 4 * cc);
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int s = s0 + 8 * j + grp;
                const bool skip = s >= n || (s < before && !shares);
                const float mj = skip ? kNegInf : ml[j][0];
                const bool none = skip || (mj == kNegInf && !(ml[j][1] != ml[j][1]));
                lse_fold(m, l, acc, mj, none ? 0.0f : ml[j][1], none ? f32x4{0.f, 0.f, 0.f, 0.f} : os[j]);
            }
        };
        for (int s0 = 0; s0 < n; s0 += 32) {
            if (n - s0 <= 8) take(s0, std::integral_constant<int, 1>{});
            else if (n - s0 <= 16) take(s0, std::integral_constant<int, 2>{});
            else if (n - s0 <= 24) take(s0, std::integral_constant<int, 3>{});
            else take(s0, std::integral_constant<int, 4>{});
        }
    }
    if constexpr (SRC != kTail && SRC != kSelected)
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
        int64_t off = bh / a.Hkv * a.o_sb + t * a.o_st;
        if constexpr (SRC == kSelected) off = bh / a.Hkv / a.tokens * a.o_sb + bh / a.Hkv % a.tokens * a.o_st;
        put_out<T, 4>(a, off + h * a.o_sh + 4 * c, x, l > 0.0f ? 1.0f / l : 0.0f);
    }
}

// Workgroups of a CU that the registers leave room for.
template <typename T, int DK, int RT>
constexpr int stream_per_cu() {
    return DK > 128 || (RT == 2 && DK * sizeof(T) >= 256) ? 1 : 2;
}
// Floats of a wavefront's state.
template <typename T, int DK, int RT>
constexpr int stream_state() {
    return 64 * (4 * StreamTile<T, DK>::NO * RT + 2 * RT);
}

template <typename T, int DK, int RT, int SRC, int MODE>
__device__ __forceinline__ void stream_workgroup(const StreamArgs& a, int id, float* lds) {
#include "stream_workgroup.inc"
}

template <typename T, int DK, int RT, int SRC, int MODE>
__global__ __launch_bounds__(kStreamThreads, (stream_per_cu<T, DK, RT>()))
void stream_fwd_kernel(StreamArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[MODE == kOwn ? 1 : (kWaves - 1) * stream_state<T, DK, RT>()];
    const int id = blockIdx.x;
#include "stream_workgroup.inc"
}

}  // namespace
}  // namespace ofh
