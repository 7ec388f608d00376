// The shared part of a batch's keys on the matrix cores, in 16 bits: rows of all
// sequences of a group, 128 or 64 per workgroup, against the group's pages staged
// through LDS, with the wavefronts of window_wave.h. Rows are numbered sequence by
// sequence, so that a tile goes on from one to the next, and leave partial rows (max,
// sum, unnormalised O) that the join folds with each sequence's own keys.
//
// A page's 16 rows are 16 KB or less of consecutive copies with one scalar base, so
// pages cost a table entry per 16 keys (loaded a tile ahead) and nothing per lane.

#include "stream_wave.h"
#include "window_wave.h"

namespace ofh {
namespace {

template <typename T, int D, int KS>
struct PrefixWave : WindowWave<T, D, KS> {
    using Base = WindowWave<T, D, KS>;
    using Tiles = typename Base::Tiles;
    using typename Base::L;
    using typename Base::v8;
    using Base::a;
    using Base::dma_row0;
    using Base::g;
    using Base::smem;
    using Base::wave;
    static constexpr int SN = Base::SN, BLOCKS = SN / kStreamKeys, NW = Tiles::THREADS / 64;
    struct Pages {
        int id[BLOCKS];    // of each 16 keys; 0 where there is none
        unsigned missing;  // one bit each
    };

    const StreamArgs& sa;
    const int32_t* table;
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
        table = sa.table + pt.start * sa.table_stride;
        const int place = (64 * wave + lane) % L::CPR;
        koff = 2u * (unsigned)((dma_row0 & 15) * (int)sa.k_st + 8 * Base::src_chunk(place ^ L::kswz(dma_row0), a.D));
        voff = 2u * (unsigned)((dma_row0 & 15) * (int)sa.v_st + 8 * Base::src_chunk(place ^ L::vswz(dma_row0), a.Dv));
    }

    // Pages of a staged tile; blocks past the last repeat it.
    __device__ __forceinline__ Pages pages(int tile) const {
        Pages p;
        p.missing = 0;
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            const int key = min(tile * BLOCKS + j, a.N / kStreamKeys - 1) * kStreamKeys;
            const int id = uniform(table[key >> sa.page_shift]);
            const bool ok = (unsigned)id < (unsigned)sa.num_pages;
            p.id[j] = ok ? id : 0;
            p.missing |= ok ? 0u : 1u << j;
        }
        return p;
    }

    // Global -> LDS copies of a staged tile (asynchronous): copy u of a wavefront covers
    // rows of one block.
    static constexpr int COPY_ROWS = 64 / L::CPR;  // of a wavefront's copy: 8, 4 or 2
    __device__ __forceinline__ void copy_pages(int tile, int stage, const Pages& p) const {
        const unsigned lds0 = (unsigned)(uintptr_t)smem + stage + 1024 * wave;
#pragma unroll
        for (int u = 0; u < Base::CPT; ++u) {
            constexpr int PER = Base::DSTEP;  // rows of the workgroup's copy
            const int block = PER >= 32 ? 2 * u + (wave * COPY_ROWS >> 4) : PER * u >> 4;
            const int id = PER >= 32 ? (wave * COPY_ROWS >> 4 ? p.id[(2 * u + 1) % BLOCKS] : p.id[2 * u % BLOCKS]) : p.id[block];
            const int key = min(tile * BLOCKS + block, a.N / kStreamKeys - 1) * kStreamKeys;
            const int row = (key & ((1 << sa.page_shift) - 1)) + (PER < 16 ? PER * u & 15 : 0);
            const T* k = (const T*)sa.k + id * sa.k_sp + hk * sa.k_sh + row * sa.k_st;
            const T* v = (const T*)sa.v + id * sa.v_sp + hk * sa.v_sh + row * sa.v_st;
            dma16s(k, koff, lds0 + 1024 * NW * u);
            dma16s(v, voff, lds0 + L::KTILE + 1024 * NW * u);
        }
    }
    // V rows of a landed tile that count for nothing -> 0: past the keys, or without a page.
    __device__ __forceinline__ void clear_rows(int tile, int stage, unsigned missing) const {
        if (missing == 0 && tile * SN + SN <= a.N) return;
#pragma unroll
        for (int u = 0; u < Base::CPT; ++u) {
            const int row = dma_row0 + u * Base::DSTEP;
            if (tile * SN + row >= a.N || (missing >> (row >> 4) & 1))
                *(u32x4*)(smem + stage + L::KTILE + 1024 * wave + 1024 * NW * u + 16 * (threadIdx.x & 63)) =
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

template <typename T, int D, int KS, WindowScores SCORES>
__global__ __launch_bounds__((WindowTiles<D, KS>::THREADS), (WindowTiles<D, KS>::WAVES_PER_SIMD))
void prefix_fwd_kernel(StreamArgs sa) {
    using W = PrefixWave<T, D, KS>;
    using L = typename W::L;
    constexpr int R = W::Tiles::R, ROWS = R * kQueriesPerWave, SN = W::SN, SB = SN / W::BN;
    constexpr int FOLD = KS > 1 ? (KS - 1) * R * group_state_bytes(D) : 0;
    __shared__ __attribute__((aligned(16))) unsigned char smem[FOLD > 2 * L::STAGE ? FOLD : 2 * L::STAGE];
    StreamPart part;
    PrefixTile pt;
    if (!prefix_part(sa, (int)blockIdx.x, part) || !prefix_tile(sa, part.rt, ROWS, pt)) return;
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
    // the tiles that some row of the workgroup sees: [0, sink_tiles) and [first, end)
    __shared__ int seen[2][4];
    if ((threadIdx.x & 63) == 0) {
        seen[0][wave] = w.hi_max;
        seen[1][wave] = w.lo_min;
    }
    __syncthreads();
    int hi_max = 0, lo_min = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi_max = max(hi_max, uniform(seen[0][i]));
        lo_min = min(lo_min, uniform(seen[1][i]));
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
        auto p = w.pages(tile(begin));
        w.copy_pages(tile(begin), 0, p);
        auto next = w.pages(tile(min(begin + 1, stop - 1)));
        wait_vm_loads();
        w.clear_rows(tile(begin), 0, p.missing);
        if (a.D < D) w.zero_pad(0);
        __syncthreads();
        for (int st = begin; st < stop; ++st) {
            const int stage = (st - begin & 1) * L::STAGE, other = L::STAGE - stage;
            if (st + 1 < stop) w.copy_pages(tile(st + 1), other, next);
            const auto after = w.pages(tile(min(st + 2, stop - 1)));
#pragma unroll
            for (int i = 0; i < SB / KS; ++i) {
                const int sub = i * KS + kg, k0 = tile(st) * SN + sub * W::BN;
                if (w.sees(k0))
                    w.template step<SCORES, decltype(redo)::value>(stage, sub, k0,
                                                                   p.missing >> (sub * W::BN / kStreamKeys) & ((1u << W::BN / kStreamKeys) - 1));
            }
            wait_vm_loads();
            if (st + 1 < stop) {
                w.clear_rows(tile(st + 1), other, next.missing);
                if (a.D < D) w.zero_pad(other);
            }
            p = next;
            next = after;
            __syncthreads();
        }
    };
    if (begin < stop) {
        run(Bool<false>{});
        if (__syncthreads_or(w.nan_in_o())) {
            w.restart();
            run(Bool<true>{});
        }
    }
    if constexpr (KS > 1) fold_groups<W, KS, R>(w, smem, wave, slice, kg);
    if (kg == 0)
        w.store_part((int64_t)part.part * sa.B * sa.Hkv * sa.T * sa.G + row_of_all(sa, w.at.b, part.hk, w.at.t, w.at.g));
}

template <typename T, int D, int KS>
hipError_t launch_prefix_groups(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)prefix_grid(a)), block(WindowTiles<D, KS>::THREADS);
    if (a.softcap > kCapExp) hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresWideCap>), grid, block, 0, s, a);
    else if (a.alibi != nullptr || a.softcap > 0.0f)
        hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresMod>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((prefix_fwd_kernel<T, D, KS, kScoresPlain>), grid, block, 0, s, a);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_prefix_type(const StreamArgs& a, int key_splits, hipStream_t s) {
    switch (stream_kernel_dim(a.D, a.Dv)) {
        case 64: return key_splits == 2 ? launch_prefix_groups<T, 64, 2>(a, s) : launch_prefix_groups<T, 64, 1>(a, s);
        case 128: return key_splits == 2 ? launch_prefix_groups<T, 128, 2>(a, s) : launch_prefix_groups<T, 128, 1>(a, s);
        case 256: return launch_prefix_groups<T, 256, 1>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_prefix(const StreamArgs& a, int dtype, int key_splits, hipStream_t s) {
    switch (dtype) {
        case DT_BF16: return launch_prefix_type<__bf16>(a, key_splits, s);
        case DT_F16: return launch_prefix_type<_Float16>(a, key_splits, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ofh
