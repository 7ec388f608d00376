// Attention of new tokens over a paged cache where not every sequence reads all
// of its own pages by itself, with the wavefronts of stream_wave.h:
//  * a batch in groups that share their first pages. Tiles of 16 or 32 rows of all
//    sequences of a group read those pages once per tile (kPrefix; many rows in
//    16 bits run in prefix_fwd.hip instead); each sequence's own tiles read the rest
//    (kTail); the join folds both.
//  * selected pages (kSelected): a tile per token and key-value head, whose
//    16-key blocks are those of the pages on its list.

#include "stream_wave.h"

namespace ofh {
namespace {

template <typename T, int DK, int RT>
hipError_t launch_prefix_rt(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)prefix_grid(a)), block(kStreamThreads);
    hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kPrefix, kPart>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <typename T, int SRC>
hipError_t launch_join(const StreamArgs& a, int tile_rows, hipStream_t s) {
    const int64_t items = (int64_t)a.B * a.Hkv * a.T * a.G * ((a.Dv + 31) / 32);
    hipLaunchKernelGGL((stream_join_kernel<T, SRC>), dim3((unsigned)((items + kWaves - 1) / kWaves)),
                       dim3(kStreamThreads), 0, s, a, tile_rows);
    return hipGetLastError();
}

template <typename T, int DK, int RT>
hipError_t launch_tail_rt(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * a.row_tiles * a.splits)), block(kStreamThreads);
    hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kTail, kPart>), grid, block, 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<T, kTail>(a, 16 * RT, s);
}

template <typename T, int DK, int RT>
hipError_t launch_selected_rt(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * a.row_tiles * a.splits)), block(kStreamThreads);
    if (a.splits == 1) {
        hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kSelected, kTile>), grid, block, 0, s, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kSelected, kPart>), grid, block, 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<T, kSelected>(a, 16 * RT, s);
}

// What to launch: a call's dtype, kernel head dim and rows of a tile.
enum What { kLaunchPrefix, kLaunchTail, kLaunchSelected };

template <What W, typename T, int DK, int RT>
hipError_t launch_rt(const StreamArgs& a, hipStream_t s) {
    if constexpr (W == kLaunchPrefix) return launch_prefix_rt<T, DK, RT>(a, s);
    else if constexpr (W == kLaunchTail) return launch_tail_rt<T, DK, RT>(a, s);
    else return launch_selected_rt<T, DK, RT>(a, s);
}
template <What W, typename T>
hipError_t launch_type(const StreamArgs& a, int rows, hipStream_t s) {
    const int dk = stream_kernel_dim(a.D, a.Dv);
    const bool wide = stream_tile_rows(sizeof(T) == 4 ? DT_F32 : DT_BF16, dk, rows) == 32;
    switch (dk) {
        case 64: return wide ? launch_rt<W, T, 64, 2>(a, s) : launch_rt<W, T, 64, 1>(a, s);
        case 128: return wide ? launch_rt<W, T, 128, 2>(a, s) : launch_rt<W, T, 128, 1>(a, s);
        case 256: return launch_rt<W, T, 256, 1>(a, s);
        default: return hipErrorInvalidValue;
    }
}
template <What W>
hipError_t launch(const StreamArgs& a, int dtype, int rows, hipStream_t s) {
    switch (dtype) {
        case DT_F32: return launch_type<W, float>(a, rows, s);
        case DT_BF16: return launch_type<W, __bf16>(a, rows, s);
        case DT_F16: return launch_type<W, _Float16>(a, rows, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

// Groups of different sizes have one kernel: that of their average rows.
PrefixKernel prefix_kernel(const StreamArgs& a, int dtype) {
    const int dk = stream_kernel_dim(a.D, a.Dv), rows = a.B / a.groups * a.T * a.G;
    // (a lane of prefix_fwd.hip adds the bytes of up to 16 rows in 32 bits, as here)
    if (dtype != DT_F32 && rows > 32) {
        const int key_splits = dk <= 128 && rows <= window_rows(2) ? 2 : 1;
        return PrefixKernel{window_rows(key_splits), 64, key_splits};
    }
    return PrefixKernel{stream_tile_rows(dtype, dk, rows), stream_step_keys(dtype, dk), 0};
}
hipError_t launch_stream_prefix(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchPrefix>(a, dtype, a.B / a.groups * a.T * a.G, s);
}
hipError_t launch_stream_tail(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchTail>(a, dtype, a.T * a.G, s);
}
hipError_t launch_stream_selected(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchSelected>(a, dtype, a.G, s);
}

}  // namespace ofh
