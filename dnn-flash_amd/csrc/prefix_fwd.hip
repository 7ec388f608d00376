// The shared part of a batch's keys on the matrix cores, in 16 bits: rows of all
// sequences of a group, 128 or 64 per workgroup, against the group's pages staged
// through LDS, with the wavefronts of window_wave.h. Rows are numbered sequence by
// sequence, so that a tile goes on from one to the next, and leave partial rows (max,
// sum, unnormalised O) that the join folds with each sequence's own keys.
//
// A copy of a wavefront stays within 16 keys, which are one page's: its base is a
// scalar, read from the lane that holds the place of these keys.
//
// One workgroup of a CU is a prefix's while another reads a sequence's own keys, so
// a workgroup by itself has to keep enough loads in flight: K and V of a step are
// halves of their own in a ring of 80 KB, each waited for by count, and a barrier
// before a half is used frees the one used before it. (With two stages of K and V
// together, 64 KB, a step waited for its memory.)
//
// Probabilities are rounded to the inputs' type for their product with V, and alike in
// the row's sum, as in all of the library's 16-bit attention: half a step each, averaged
// over the keys, is about what the rounding of the result is (rms of normal rows: bf16
// 1.6e-3 and 1.7e-3, both 2.3e-3; fp16 2.0e-4, 2.1e-4, both 2.9e-4). In 32 bits each
// product with V would be two, of P's upper and lower half.
//
// Measured with the sequences' own keys beside it: bf16 B64 H32/8 D128, 16384 shared
// keys in pages of 16, 33-1024 of each sequence's own, 65.4 us: this launch 58.6, the
// join 8.6. (The parts one after the other, in launches of their own: 85.) What
// bounds it: 67 MB of shared and 138 MB of own keys are 36 us of reading; a step of 64
// keys takes 1.3-1.8 us, its products, softmax and LDS reads one after the other in a
// wavefront (matrix cores 18 % of the SIMD time, VALU 30 %, no LDS conflicts), and what
// overlaps is the other workgroup of the CU.

#include "stream_wave.h"
#include "window_wave.h"

namespace ofh {
namespace {

// dma16s of COUNT copies that are `step` bytes of LDS apart, M0 saved once.
template <int COUNT>
__device__ __forceinline__ void dma16s_row(const char* const (&base)[COUNT], unsigned off, unsigned lds, unsigned step);
template <>
__device__ __forceinline__ void dma16s_row<2>(const char* const (&base)[2], unsigned off, unsigned lds, unsigned step) {
    unsigned save;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
        "s_add_u32 m0, m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
        : "=&s"(save) : "v"(off), "s"(base[0]), "s"(base[1]), "s"(lds), "s"(step) : "memory", "scc");
}
template <>
__device__ __forceinline__ void dma16s_row<4>(const char* const (&base)[4], unsigned off, unsigned lds, unsigned step) {
    unsigned save;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
        "s_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
        "s_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %4\n\t"
        "s_add_u32 m0, m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\ts_mov_b32 m0, %0"
        : "=&s"(save)
        : "v"(off), "s"(base[0]), "s"(base[1]), "s"(base[2]), "s"(base[3]), "s"(lds), "s"(step)
        : "memory", "scc");
}

// Steps of SN keys, which KS groups of wavefronts share in BN, and a ring of HALVES.
template <int D, int KS>
struct PrefixTiles {
    static constexpr int THREADS = 256, WAVES = THREADS / 64;
    static constexpr int R = WAVES / KS;
    static constexpr int BN = D == 256 || KS == 2 ? 32 : 64;
    static constexpr int SN = D == 256 ? 32 : 64;
    static constexpr int SB = SN / BN;
    static constexpr int WAVES_PER_SIMD = D <= 128 ? 2 : 1;
    static constexpr int HALVES = D == 128 ? 5 : 9;
    static_assert(SB % KS == 0, "the groups share a step");
};

template <typename T, int D, int KS>
struct PrefixWave : WindowWave<T, D, KS, PrefixTiles<D, KS>> {
    using Base = WindowWave<T, D, KS, PrefixTiles<D, KS>>;
    using Tiles = typename Base::Tiles;
    using typename Base::L;
    using typename Base::v8;
    using Base::a;
    using Base::dma_row0;
    using Base::g;
    using Base::smem;
    using Base::wave;
    static constexpr int SN = Base::SN, BLOCKS = SN / kStreamKeys, NW = Tiles::THREADS / 64;
    // Where the 16-key blocks of some steps stand, a block per lane.
    struct Places {
        uint64_t k, v;     // addresses of the first rows; of page 0's where there is no page
        uint64_t missing;  // a bit for each block without one
    };
    static constexpr int KEPT = 64 / BLOCKS;  // steps

    const StreamArgs& sa;
    PrefixRow at;
    bool in;  // a row of the group
    int hk;
    unsigned koff, voff;

    __device__ __forceinline__ PrefixWave(const FwdArgs& args, const StreamArgs& s, unsigned char* sm, const PrefixTile& pt,
                                          int head, int wv, int slice)
        : Base(args, sm, wv), sa(s), hk(head) {
        const int lane = threadIdx.x & 63, rows = pt.count * sa.T * sa.G;
        const int row = pt.rt * Tiles::R * kQueriesPerWave + slice * kQueriesPerWave + (lane & 31);
        in = row < rows;
        at = prefix_row(sa, pt, min(row, rows - 1));
        const int h = hk * sa.G + at.g;
        const T* q = (const T*)sa.q + at.b * sa.q_sb + h * sa.q_sh + at.t * sa.q_st + 8 * g;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            u32x4 u = {0u, 0u, 0u, 0u};
            if (16 * c + 8 * g < a.D) u = *(const u32x4*)(q + 16 * c);
            this->qf[c] = __builtin_bit_cast(v8, u);
        }
        this->pos = prefix_limits(sa, pt, at, this->hi, this->lo);
        this->sinks = sa.sinks;
        this->slope = sa.alibi != nullptr ? sa.alibi[h] : 0.0f;
        this->hi_min = wave_min(this->hi);
        this->hi_max = wave_max(this->hi);
        this->lo_min = wave_min(this->lo);
        this->lo_max = wave_max(this->lo);
        if (pt.rt * Tiles::R * kQueriesPerWave + slice * kQueriesPerWave >= rows) this->hi_max = 0;  // no rows of its own
        const int place = (64 * wave + lane) % L::CPR;
        koff = 2u * (unsigned)((dma_row0 & 15) * (int)sa.k_st + 8 * Base::src_chunk(place ^ L::kswz(dma_row0), a.D));
        voff = 2u * (unsigned)((dma_row0 & 15) * (int)sa.v_st + 8 * Base::src_chunk(place ^ L::vswz(dma_row0), a.Dv));
    }

    // Places of a lane's block: of step tile number `tile`, block j of it (blocks past the
    // keys repeat the last). Formed by 64 lanes at once: as scalars, four of a step's
    // blocks took 250 instructions of each step's time.
    __device__ __forceinline__ Places places(int first, int tile, int j) const {
        const int key = min(tile * BLOCKS + j, a.N / kStreamKeys - 1) * kStreamKeys;
        const int id = sa.table[first * sa.table_stride + (key >> sa.page_shift)];
        const bool ok = (unsigned)id < (unsigned)sa.num_pages;
        const int64_t page = ok ? id : 0, row = key & ((1 << sa.page_shift) - 1);
        Places p;
        p.k = (uint64_t)sa.k + 2 * (page * sa.k_sp + hk * sa.k_sh + row * sa.k_st);
        p.v = (uint64_t)sa.v + 2 * (page * sa.v_sp + hk * sa.v_sh + row * sa.v_st);
        p.missing = __builtin_amdgcn_ballot_w64(!ok);
        return p;
    }
    static __device__ __forceinline__ uint64_t of_lane(uint64_t x, int lane) {
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, lane);
        const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), lane);
        return (uint64_t)hi << 32 | lo;
    }
    // Global -> LDS copies of a step's K or V (asynchronous) to `to`.
    // x: K or V of the blocks; `lane` holds the step's first.
    __device__ __forceinline__ void copy_half(uint64_t x, int lane, int64_t row_stride, unsigned off, int to) const {
        constexpr int COPY_ROWS = 64 / L::CPR;  // of a wavefront's copy: 8, 4 or 2
        constexpr int PER = Base::DSTEP;        // of the workgroup's: 32, 16 or 8
        const char* base[Base::CPT];
#pragma unroll
        for (int u = 0; u < Base::CPT; ++u) {
            const int block = PER >= 32 ? 2 * u + uniform(wave * COPY_ROWS >> 4) : PER * u >> 4;
            base[u] = (const char*)(of_lane(x, lane + block) + (PER < 16 ? (PER * u & 15) * 2 * row_stride : 0));
        }
        dma16s_row<Base::CPT>(base, off, (unsigned)(uintptr_t)smem + to + 1024 * wave, 1024 * NW);
    }
    // V rows of a landed step that count for nothing -> 0: past the keys, or without a page.
    __device__ __forceinline__ void clear_rows(int tile, int at_lds, unsigned missing) const {
        if (missing == 0 && tile * SN + SN <= a.N) return;
#pragma unroll
        for (int u = 0; u < Base::CPT; ++u) {
            const int row = dma_row0 + u * Base::DSTEP;
            if (tile * SN + row >= a.N || (missing >> (row >> 4) & 1))
                *(u32x4*)(smem + at_lds + 1024 * wave + 1024 * NW * u + 16 * (threadIdx.x & 63)) =
                    u32x4{0u, 0u, 0u, 0u};
        }
    }

    __device__ __forceinline__ void store_part(int64_t prow) {
        const float l_tot = this->l_run + __shfl_xor(this->l_run, 32);
        if (!in) return;
        float* po = sa.prefix_o + prow * a.Dv + 8 * g;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
                if (32 * db + 16 * cc + 8 * g >= a.Dv) continue;
                f32x4 lo, hi;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    lo[t] = this->o[db][8 * cc + t];
                    hi[t] = this->o[db][8 * cc + 4 + t];
                }
                *(f32x4*)(po + 32 * db + 16 * cc) = lo;
                *(f32x4*)(po + 32 * db + 16 * cc + 4) = hi;
            }
        if (g == 0) {
            sa.prefix_ml[2 * prow] = this->m_run;
            sa.prefix_ml[2 * prow + 1] = l_tot;
        }
    }
};

// LDS of a workgroup: the ring, or the states that key groups fold.
template <typename T, int D, int KS>
constexpr int prefix_lds() {
    using W = PrefixWave<T, D, KS>;
    constexpr int FOLD = KS > 1 ? (KS - 1) * W::Tiles::R * group_state_bytes(D) : 0, RING = W::Tiles::HALVES * W::L::KTILE;
    return FOLD > RING ? FOLD : RING;
}

// Workgroup `id` of the prefix's.
template <typename T, int D, int KS, WindowScores SCORES>
__device__ __forceinline__ void prefix_workgroup(const StreamArgs& sa, int id, unsigned char* smem) {
    using W = PrefixWave<T, D, KS>;
    constexpr int R = W::Tiles::R, ROWS = R * kQueriesPerWave, SN = W::SN, SB = SN / W::BN;
    constexpr int HALF = W::L::KTILE, HALVES = W::Tiles::HALVES;
    StreamPart part;
    PrefixTile pt;
    if (!prefix_part(sa, id, part) || !prefix_tile(sa, part.rt, ROWS, pt)) return;
    FwdArgs a{};
    a.q = sa.q;
    a.k = sa.k;
    a.v = sa.v;
    a.H = a.M = 1;
    a.N = pt.shared;
    a.D = sa.D;
    a.Dv = sa.Dv;
    a.scale = sa.scale;
    a.scale_log2 = sa.scale * kLog2e;
    a.softcap = sa.softcap;
    a.inv_softcap = sa.softcap > 0.0f ? 1.0f / sa.softcap : 0.0f;
    const int wave = uniform(threadIdx.x >> 6), slice = wave % R, kg = wave / R;
    W w(a, sa, smem, pt, part.hk, wave, slice);
    // The tiles that some row of the workgroup sees: [0, sink_tiles) and [first, end).
    // (Without a window all shared ones: where sequences end within them, masked; the
    // lengths, a memory round trip, are then on their way beside the first keys.)
    int* seen = (int*)smem;
    int hi_max = pt.shared, lo_min = 0;
    if (sa.window > 0) {
        if ((threadIdx.x & 63) == 0) {
            seen[wave] = w.hi_max;
            seen[4 + wave] = w.lo_min;
        }
        __syncthreads();
        hi_max = 0;
        lo_min = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi_max = max(hi_max, uniform(seen[i]));
            lo_min = min(lo_min, uniform(seen[4 + i]));
        }
        __syncthreads();  // (the ring takes its place)
    }
    const int end = (hi_max + SN - 1) / SN;
    int sink_tiles = 0, first = 0;
    if (sa.window > 0) {
        sink_tiles = min((min(sa.sinks, hi_max) + SN - 1) / SN, end);
        first = max(sink_tiles, min(end, max(0, lo_min) / SN));
    }
    const int steps = sink_tiles + end - first;
    int per = steps;
    const int parts = stream_parts(sa.prefix_splits, sa.prefix_min_steps, steps, per);
    const int begin = part.part < parts ? min(steps, part.part * per) : steps, stop = min(steps, begin + per);
    auto tile = [&](int st) { return st < sink_tiles ? st : st - sink_tiles + first; };
    auto run = [&](auto redo) {
        constexpr bool REDO = decltype(redo)::value;
        // Half h is K (even) or V (odd) of step begin + h / 2, at place h % HALVES of the
        // ring; HALVES - 1 of them, of AHEAD steps, are on their way or in use.
        constexpr int AHEAD = (HALVES - 1) / 2;
        static_assert(HALVES % 2 == 1, "a step's halves are copied where those of an earlier one are used");
        const int halves = 2 * (stop - begin);
        auto forward = [](int x) { return x == (HALVES - 1) * HALF ? 0 : x + HALF; };
        int to = 0, at = 0;     // places to copy to, and in use
        uint64_t missing = 0;   // of the steps copied, four bits each, the last lowest
        typename W::Places p;
        int lane0 = 0;          // of the step copied last
        auto copy_k = [&](int st) {
            const int n = st - begin, lane = threadIdx.x & 63;
            if (n % W::KEPT == 0)
                p = w.places(pt.start, tile(min(st + lane / W::BLOCKS, stop - 1)), lane % W::BLOCKS);
            lane0 = n % W::KEPT * W::BLOCKS;
            missing = missing << 4 | (p.missing >> lane0 & ((1u << W::BLOCKS) - 1));
            w.copy_half(p.k, lane0, sa.k_st, w.koff, to);
            to = forward(to);
        };
        auto copy_v = [&] {
            w.copy_half(p.v, lane0, sa.v_st, w.voff, to);
            to = forward(to);
        };
        // Half h has landed for every wavefront, and the one before it is used up.
        auto await = [&](int h) {
            if (h + HALVES - 1 <= halves) wait_vm<W::CPT * (HALVES - 2)>();
            else wait_vm_loads();
        };
        for (int i = 0; i < AHEAD; ++i)
            if (begin + i < stop) {
                copy_k(begin + i);
                copy_v();
            }
        for (int st = begin; st < stop; ++st) {
            const int h = 2 * (st - begin), t = tile(st), ahead = min(AHEAD, stop - st);  // steps copied from this one on
            const unsigned gone = (unsigned)(missing >> 4 * (ahead - 1)) & 15u;
            await(h);
            if (a.D < D) w.zero_pad(at);
            __syncthreads();
            if (st + AHEAD < stop) copy_k(st + AHEAD);
            const int sub = kg, k0 = t * SN + sub * W::BN;
            const unsigned no = gone >> (sub * W::BN / kStreamKeys) & ((1u << W::BN / kStreamKeys) - 1);
            const bool some = w.sees(k0), partly = w.partly(k0) || no != 0;
            if (some) {
                __builtin_amdgcn_s_setprio(1);
                w.qk(at, sub);
                __builtin_amdgcn_s_setprio(0);
                w.template softmax_window<SCORES>(k0, partly, no);
            }
            at = forward(at);
            await(h + 1);
            w.clear_rows(t, at, gone);
            __syncthreads();
            if (st + AHEAD < stop) copy_v();
            const int stage = at - HALF;  // (V stands behind K there)
            if (some && REDO && partly) {
                w.pv_seen(stage, sub, k0);
            } else if (some) {
                __builtin_amdgcn_s_setprio(1);
                w.pv(stage, sub);
                __builtin_amdgcn_s_setprio(0);
            }
            at = forward(at);
        }
        __syncthreads();
    };
    static_assert(SB == KS, "a group has one step's scores at a time");
    if (begin < stop) {
        run(Bool<false>{});
        // (by hand: __syncthreads_or has LDS of its own, and two rings fill the CU's)
        const uint64_t mine = __builtin_amdgcn_ballot_w64(w.nan_in_o());
        if ((threadIdx.x & 63) == 0) seen[wave] = mine != 0;
        __syncthreads();
        const bool bad = seen[0] | seen[1] | seen[2] | seen[3];
        __syncthreads();
        if (uniform(bad)) {
            w.restart();
            run(Bool<true>{});
        }
    }
    if constexpr (KS > 1) fold_groups<W, KS, R>(w, smem, wave, slice, kg);
    if (kg == 0)
        w.store_part((int64_t)part.part * sa.B * sa.Hkv * sa.T * sa.G + row_of_all(sa, w.at.b, part.hk, w.at.t, w.at.g));
}

template <typename T, int D, int KS, WindowScores SCORES>
__global__ __launch_bounds__((PrefixTiles<D, KS>::THREADS), (PrefixTiles<D, KS>::WAVES_PER_SIMD))
void prefix_fwd_kernel(StreamArgs a) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[prefix_lds<T, D, KS>()];
    prefix_workgroup<T, D, KS, SCORES>(a, blockIdx.x, smem);
}

// With the plain scale, beside the sequences' own keys in one launch: the matrix cores
// are busy with the ones while the others wait for memory.
template <typename T, int D, int KS, int RT>
__global__ __launch_bounds__(kStreamThreads, (PrefixTiles<D, KS>::WAVES_PER_SIMD))
void prefix_shared_kernel(StreamArgs a) {
    constexpr int TAIL = (kWaves - 1) * stream_state<T, D, RT>() * 4, PREFIX = prefix_lds<T, D, KS>();
    __shared__ __attribute__((aligned(16))) unsigned char smem[PREFIX > TAIL ? PREFIX : TAIL];
    int id;
    if (shared_workgroup(a, blockIdx.x, id)) prefix_workgroup<T, D, KS, kScoresPlain>(a, id, smem);
    else if (id < tail_grid(a)) stream_workgroup<T, D, RT, kTail, kPart>(a, id, (float*)smem);
}

template <typename T, int D, int KS>
hipError_t launch_prefix_groups(const StreamArgs& a, int dtype, hipStream_t s) {
    const dim3 block(kStreamThreads);
    static_assert(PrefixTiles<D, KS>::THREADS == kStreamThreads, "both parts of a launch have its workgroup");
    const bool plain = a.alibi == nullptr && a.softcap <= 0.0f;
    const bool wide = D <= 128 && stream_tile_rows(dtype, D, a.T * a.G) == 32;
    // (at D = 128 the registers of 32-row tiles leave room for one workgroup per CU: with
    // two, 115 would spill)
    if (plain && !(wide && D == 128)) {
        const dim3 grid((unsigned)shared_grid(a));
        if constexpr (D == 64)
            if (wide) hipLaunchKernelGGL((prefix_shared_kernel<T, D, KS, 2>), grid, block, 0, s, a);
        if (!wide) hipLaunchKernelGGL((prefix_shared_kernel<T, D, KS, 1>), grid, block, 0, s, a);
        if (hipError_t e = hipGetLastError()) return e;
        return launch_stream_join(a, dtype, s);
    }
    const dim3 grid((unsigned)prefix_grid(a));
    if (a.softcap > kCapExp) hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresWideCap>), grid, block, 0, s, a);
    else if (!plain) hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresMod>), grid, block, 0, s, a);
    else if constexpr (D == 128) hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresPlain>), grid, block, 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_stream_tail(a, dtype, s);
}
template <typename T>
hipError_t launch_prefix_type(const StreamArgs& a, int dtype, int key_splits, hipStream_t s) {
    const bool two = key_splits == 2;
    switch (stream_kernel_dim(a.D, a.Dv)) {
        case 64: return two ? launch_prefix_groups<T, 64, 2>(a, dtype, s) : launch_prefix_groups<T, 64, 1>(a, dtype, s);
        case 128: return two ? launch_prefix_groups<T, 128, 2>(a, dtype, s) : launch_prefix_groups<T, 128, 1>(a, dtype, s);
        case 256: return launch_prefix_groups<T, 256, 1>(a, dtype, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_prefix_shared(const StreamArgs& a, int dtype, int key_splits, hipStream_t s) {
    switch (dtype) {
        case DT_BF16: return launch_prefix_type<__bf16>(a, dtype, key_splits, s);
        case DT_F16: return launch_prefix_type<_Float16>(a, dtype, key_splits, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ofh
