// Windowed attention of prompts in 16 bits on the matrix cores: 32-row
// wavefronts (flash_wave32.h) against K and V tiles staged through LDS.
//
// A workgroup's rows see the first tokens' tiles and then the tiles from the
// oldest row's window to the youngest row's diagonal; no other tile is loaded.
// A wavefront skips the tiles that none of its 32 rows sees and masks element
// by element only in those that some of its rows see partly. Four wavefronts
// take 128 rows, or share the keys of 64 rows between two groups (fold_groups):
// a workgroup reads its window and its rows' own span, so small windows waste
// least with few rows, and small calls fill the GPU.
//
// What bounds it: the products and the softmax of a wavefront one after the
// other (bf16 D128 B4 H32/8 N2048 window 1024, 4 first tokens: 139-157 us by
// card, 746-658 TFLOP/s; N300-2048 in one batch 104 us, matrix cores 34 % and
// vector ALUs 40 % of the busy CUs' time, no LDS conflicts). K and V of a window
// are read once per 128 rows, mostly from L2.
//
// Masked tiles: a key that a row does not see has probability 0, which does
// not hide a NaN or an infinity in its V row from the product: O then holds a
// NaN. A workgroup that ends with one in any of its rows runs again and adds
// its partly masked tiles key by key, to the rows that see the key. (With that
// loop, or a test, inside the one loop the compiler moved the accumulators
// about on every step: bf16 B4 H32 N4096 D128 773 us against 663.)

#include "window_wave.h"

namespace ofh {
namespace {

// Workgroup -> (sequence, query head, query tile). The 8 XCDs take workgroups in
// turn: where they can be dealt out evenly, each takes every eighth key-value
// head, so that sequences of a padded batch, whose lengths differ, are spread over
// all of them (in blocks of neighbouring heads: bf16 B4 H32/8 N300-2048 D128 window
// 1024 139 us, this 104), and runs its query heads side by side: they share K and V
// in its L2. Late tiles, whose keys are most without a window, run first.
__device__ __forceinline__ void window_work(const WindowArgs& wa, int id, int& b, int& h, int& qt) {
    const int n = wa.f.B * wa.f.H, nqt = wa.f.num_q_tiles;
    int bh, t;
    if ((n & 7) == 0) {
        const int side = (n / wa.G & 7) == 0 ? wa.G : 1, j = id >> 3;
        const int unit = j / (nqt * side), rest = j - unit * (nqt * side);
        t = rest / side;
        bh = (8 * unit + (id & 7)) * side + rest - t * side;
    } else {
        bh = id % n;
        t = id / n;
    }
    b = bh / wa.f.H;
    h = bh - b * wa.f.H;
    qt = nqt - 1 - t;
}

template <typename T, int D, int KS, WindowScores SCORES>
__global__ __launch_bounds__((WindowTiles<D, KS>::THREADS), (WindowTiles<D, KS>::WAVES_PER_SIMD))
void window_fwd_kernel(WindowArgs wa) {
    using W = WindowWave<T, D, KS>;
    using L = typename W::L;
    constexpr int R = W::Tiles::R, ROWS = R * kQueriesPerWave, SN = W::SN, SB = SN / W::BN;
    constexpr int FOLD = KS > 1 ? (KS - 1) * R * group_state_bytes(D) : 0;
    __shared__ __attribute__((aligned(16))) unsigned char smem[FOLD > 2 * L::STAGE ? FOLD : 2 * L::STAGE];
    int b, h, qt;
    window_work(wa, (int)blockIdx.x, b, h, qt);
    FwdArgs a = wa.f;
    if (wa.lengths != nullptr) a.N = max(0, min(wa.lengths[b], a.N));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = wave % R, kg = wave / R;
    const int q0 = qt * ROWS;
    // staged tiles [0, sink_tiles) and [first, end)
    const int p0 = q0 + wa.query_offset, p1 = min(q0 + ROWS, a.M) - 1 + wa.query_offset;
    const int kend = wa.lengths != nullptr && p0 >= a.N ? 0 : min(a.N, p1 + 1);
    const int end = (kend + SN - 1) / SN;
    int sink_tiles = 0, first = 0;
    if (wa.window > 0) {
        sink_tiles = min((min(wa.sinks, kend) + SN - 1) / SN, end);
        first = max(sink_tiles, min(end, max(0, p0 + 1 - wa.window) / SN));
    }
    const int steps = sink_tiles + end - first;
    auto tile = [&](int st) { return st < sink_tiles ? st : st - sink_tiles + first; };
    W w(a, wa, smem, b, h, q0 + (slice - wave) * kQueriesPerWave, wave);  // rows q0 + 32 slice ..
    auto run = [&](auto seen) {
        w.copy_tile(tile(0), 0);
        wait_vm_loads();
        w.zero_tail(tile(0), 0);
        if (a.D < D) w.zero_pad(0);
        __syncthreads();
        for (int st = 0; st < steps; ++st) {
            const int stage = (st & 1) * L::STAGE, next = ((st + 1) & 1) * L::STAGE;
            if (st + 1 < steps) w.copy_tile(tile(st + 1), next);
#pragma unroll
            for (int i = 0; i < SB / KS; ++i) {
                const int sub = i * KS + kg, k0 = tile(st) * SN + sub * W::BN;
                if (w.sees(k0)) w.template step<SCORES, decltype(seen)::value>(stage, sub, k0);
            }
            wait_vm_loads();
            if (st + 1 < steps) {
                w.zero_tail(tile(st + 1), next);
                if (a.D < D) w.zero_pad(next);
            }
            __syncthreads();
        }
    };
    if (steps > 0) {
        run(Bool<false>{});
        if (__syncthreads_or(w.nan_in_o())) {
            w.restart();
            run(Bool<true>{});
        }
    }
    if constexpr (KS > 1) fold_groups<W, KS, R>(w, smem, wave, slice, kg);
    if (kg == 0) w.store_output();
}

template <typename T, int D, int KS>
hipError_t launch_window_groups(const WindowArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.f.B * a.f.H * a.f.num_q_tiles)), block(WindowTiles<D, KS>::THREADS);
    if (a.f.softcap > kCapExp)
        hipLaunchKernelGGL((window_fwd_kernel<T, D, KS, kScoresWideCap>), grid, block, 0, s, a);
    else if (a.f.alibi != nullptr || a.f.softcap > 0.0f)
        hipLaunchKernelGGL((window_fwd_kernel<T, D, KS, kScoresMod>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((window_fwd_kernel<T, D, KS, kScoresPlain>), grid, block, 0, s, a);
    return hipGetLastError();
}
template <typename T, int D>
hipError_t launch_window_dim(const WindowArgs& a, hipStream_t s) {
    if (a.key_splits == 1) return launch_window_groups<T, D, 1>(a, s);
    if constexpr (D <= 128)
        if (a.key_splits == 2) return launch_window_groups<T, D, 2>(a, s);
    return hipErrorInvalidValue;
}
template <typename T>
hipError_t launch_window_type(const WindowArgs& a, hipStream_t s) {
    switch (stream_kernel_dim(a.f.D, a.f.Dv)) {
        case 64: return launch_window_dim<T, 64>(a, s);
        case 128: return launch_window_dim<T, 128>(a, s);
        case 256: return launch_window_dim<T, 256>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_window(const WindowArgs& a, int dtype, hipStream_t s) {
    const int rows = window_rows(a.key_splits);
    if (a.f.num_q_tiles != (a.f.M + rows - 1) / rows) return hipErrorInvalidValue;
    switch (dtype) {
        case DT_BF16: return launch_window_type<__bf16>(a, s);
        case DT_F16: return launch_window_type<_Float16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ofh
