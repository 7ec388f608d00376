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

#include "stream_wave.h"

namespace ofh {
namespace {

template <typename T, int DK, int RT, int MODE>
hipError_t launch_stream_mode(const StreamArgs& a, hipStream_t s) {
    const int per_head = MODE == kOwn ? (a.row_tiles + kWaves - 1) / kWaves : a.row_tiles * a.splits;
    const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * per_head)), block(kStreamThreads);
    if (a.paged) hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kPaged, MODE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((stream_fwd_kernel<T, DK, RT, kContiguous, MODE>), grid, block, 0, s, a);
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
    hipLaunchKernelGGL((stream_join_kernel<T, kPaged>), dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(kStreamThreads), 0,
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
