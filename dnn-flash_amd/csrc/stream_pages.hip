// Attention of new tokens over a paged cache where not every sequence reads all
// of its own pages by itself, with the wavefronts of stream_wave.h:
//  * a batch in groups that share their first pages. Tiles of 16 or 32 rows of all
//    sequences of a group read those pages once per tile (kPrefix; many rows in
//    16 bits run in prefix_fwd.hip instead); each sequence's own tiles read the rest
//    (kTail); the join folds both.
//  * selected pages (kSelected): a tile per token and key-value head, whose
//    16-key blocks are those of the pages on its list.
//
// Probabilities are rounded to the inputs' type for their product with V, and alike in
// the row's sum, as in all of the library's 16-bit attention: half a step each, averaged
// over the keys, is about what the rounding of the result is (rms of normal rows: bf16
// 1.6e-3 and 1.7e-3, both 2.3e-3; fp16 2.0e-4, 2.1e-4, both 2.9e-4). In 32 bits each
// product with V would be two, of P's upper and lower half. fp32 keeps its own.
//
// Measured (us) and what bounds it: few rows are latency, launch, table, K, V and the
// join's launch in turn (bf16 4 sequences, H32/8 D128, 1024 shared 12.6, of which the
// join 4.2; fp32 D64 3 groups of 5 with 3 tokens, H8, 4000 shared 24.5, 60 MB, matrix
// cores 20 %); selected pages are read at 5.2 TB/s (bf16 B32 H32/8 D128, 64 pages of
// 32 each, 268 MB in 51.6).

#include "stream_wave.h"

namespace ofh {
namespace {

template <typename T, int SRC>
hipError_t launch_join(const StreamArgs& a, int tile_rows, hipStream_t s) {
    const int64_t items = (int64_t)a.B * a.Hkv * a.T * a.G * ((a.Dv + 31) / 32);
    hipLaunchKernelGGL((stream_join_kernel<T, SRC>), dim3((unsigned)((items + kWaves - 1) / kWaves)),
                       dim3(kStreamThreads), 0, s, a, tile_rows);
    return hipGetLastError();
}

// The shared part and the sequences' own in one launch (RTP: of the prefix's tiles).
template <typename T, int DK, int RTP, int RT>
__global__ __launch_bounds__(kStreamThreads, (RTP > RT ? stream_per_cu<T, DK, RTP>() : stream_per_cu<T, DK, RT>()))
void stream_shared_kernel(StreamArgs a) {
    __shared__ __attribute__((aligned(16))) float lds[(kWaves - 1) * stream_state<T, DK, (RTP > RT ? RTP : RT)>()];
    int id;
    if (shared_workgroup(a, blockIdx.x, id)) stream_workgroup<T, DK, RTP, kPrefix, kPart>(a, id, lds);
    else if (id < tail_grid(a)) stream_workgroup<T, DK, RT, kTail, kPart>(a, id, lds);
}
template <typename T, int DK, int RTP, int RT>
hipError_t launch_shared_rt(const StreamArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((stream_shared_kernel<T, DK, RTP, RT>), dim3((unsigned)shared_grid(a)), dim3(kStreamThreads), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<T, kTail>(a, 16 * RT, s);
}
template <typename T, int DK, int RT>
hipError_t launch_shared(const StreamArgs& a, int prefix_rows, hipStream_t s) {
    if (prefix_rows == 16) {
        // (a tile of 16 rows for a group of which each sequence has more: fp32 alone)
        if constexpr (RT == 1 || sizeof(T) == 4) return launch_shared_rt<T, DK, 1, RT>(a, s);
    } else if constexpr (DK <= 128) {
        return launch_shared_rt<T, DK, 2, RT>(a, s);
    }
    return hipErrorInvalidValue;
}

template <typename T, int DK, int RT>
hipError_t launch_tail_rt(const StreamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)tail_grid(a)), block(kStreamThreads);
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
enum What { kLaunchShared, kLaunchTail, kLaunchJoin, kLaunchSelected };

template <What W, typename T, int DK, int RT>
hipError_t launch_rt(const StreamArgs& a, int prefix_rows, hipStream_t s) {
    if constexpr (W == kLaunchShared) return launch_shared<T, DK, RT>(a, prefix_rows, s);
    else if constexpr (W == kLaunchTail) return launch_tail_rt<T, DK, RT>(a, s);
    else if constexpr (W == kLaunchJoin) return launch_join<T, kTail>(a, 16 * RT, s);
    else return launch_selected_rt<T, DK, RT>(a, s);
}
template <What W, typename T>
hipError_t launch_type(const StreamArgs& a, int rows, int prefix_rows, hipStream_t s) {
    const int dk = stream_kernel_dim(a.D, a.Dv);
    const bool wide = stream_tile_rows(sizeof(T) == 4 ? DT_F32 : DT_BF16, dk, rows) == 32;
    switch (dk) {
        case 64: return wide ? launch_rt<W, T, 64, 2>(a, prefix_rows, s) : launch_rt<W, T, 64, 1>(a, prefix_rows, s);
        case 128: return wide ? launch_rt<W, T, 128, 2>(a, prefix_rows, s) : launch_rt<W, T, 128, 1>(a, prefix_rows, s);
        case 256: return launch_rt<W, T, 256, 1>(a, prefix_rows, s);
        default: return hipErrorInvalidValue;
    }
}
template <What W>
hipError_t launch(const StreamArgs& a, int dtype, int rows, int prefix_rows, hipStream_t s) {
    switch (dtype) {
        case DT_F32: return launch_type<W, float>(a, rows, prefix_rows, s);
        case DT_BF16: return launch_type<W, __bf16>(a, rows, prefix_rows, s);
        case DT_F16: return launch_type<W, _Float16>(a, rows, prefix_rows, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

// Groups of different sizes have one kernel: the largest one's.
//
// Through LDS (16 bits, more than 32 rows) or streaming.
PrefixKernel prefix_kernel(const StreamArgs& a, int dtype, int rows) {
    const int dk = stream_kernel_dim(a.D, a.Dv);
    if (dtype != DT_F32 && rows > 32) {
        const int key_splits = dk <= 128 && rows <= window_rows(2) ? 2 : 1;
        return PrefixKernel{window_rows(key_splits), dk == 256 ? 32 : 64, key_splits, 1};
    }
    const int tile = stream_tile_rows(dtype, dk, rows);
    const bool one = dk == 256 || (dk == 128 && tile == 32);
    return PrefixKernel{tile, stream_step_keys(dtype, dk), 0, one ? 1 : 2};
}

// Through LDS: a workgroup per CU, whose other place the sequences' own keys have (us,
// bf16 H32/8 D128, 16384 shared keys, 33-1024 of each sequence's own, 256 / 512
// workgroups: 64 sequences 66 / 76, 32 49 / 58, 16 31 / 40).
//
// Streaming: shared and own together no more than run at once, since what waits for a
// place then costs a whole pass (us, 512 / 624 workgroups at two per CU: f32 D64, 3 groups
// of 5 sequences with 3 tokens, H8, 4000 shared 24.9 / 29.9; f16 D64, 4 groups of 4,
// H16/8, 8192 shared 23.0 / 28.2; 256 / 324 at one: f16 D256, one group of 5, H16/4,
// 6000 shared 21.5 / 29.5). A second one of a CU only up to 16 parts (16 against 6 of those
// f32 groups 24.9 / 26.9, 12 against 4 of the f16 ones 23.0 / 29.3; but 24 against 56 of
// one group of 8, f32 D64 H8, 16000 shared 24.7 / 33.9), where the parts of an own
// tile, mostly short, count as one (f32 D128, one group of 4, H32/8, 16000 shared, 28
// parts 37.9, 16 44.8).
int64_t prefix_parts(const PrefixKernel& k, int64_t units, int64_t own, int64_t own_parts) {
    constexpr int64_t kCus = kComputeUnits, kFew = 16;
    if (k.key_splits > 0) return (kCus + units - 1) / units;
    const int64_t at_once = std::max(k.per_cu * kCus - own_parts, kCus / 2) / units;
    const int64_t first = (kCus - own) / units;
    return std::min(at_once, std::max(first, kFew));
}
hipError_t launch_stream_shared(const StreamArgs& a, int dtype, int prefix_rows, hipStream_t s) {
    return launch<kLaunchShared>(a, dtype, a.T * a.G, prefix_rows, s);
}
hipError_t launch_stream_tail(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchTail>(a, dtype, a.T * a.G, 0, s);
}
hipError_t launch_stream_join(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchJoin>(a, dtype, a.T * a.G, 0, s);
}
hipError_t launch_stream_selected(const StreamArgs& a, int dtype, hipStream_t s) {
    return launch<kLaunchSelected>(a, dtype, a.G, 0, s);
}

}  // namespace ofh
