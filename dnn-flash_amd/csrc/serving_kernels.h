// Argument blocks and launchers of the serving operators: attention over a
// paged key-value cache, windowed attention of prompts, and the writing and
// copying of cache pages. Internal header: not installed.
#pragma once

#include "ofh_kernels.h"

namespace ofh {

// Visibility of both attentions. The query at position p of a sequence of
// `length` keys sees key j iff j < length, j <= p and, with a window,
// p - j < window or j < sinks.
//
// Query head h reads key-value head h / G, G = H / Hkv. Rows of one (sequence,
// key-value head) are numbered r = t G + g: token t, head g of the group, so a
// tile of rows shares the K and V that it reads.
struct StreamArgs {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    int64_t q_sb, q_sh, q_st;
    int64_t o_sb, o_sh, o_st;
    // elements between pages (contiguous K and V: sequences), heads, tokens
    int64_t k_sp, k_sh, k_st;
    int64_t v_sp, v_sh, v_st;
    // paged: keys [i S, (i + 1) S) of sequence b stand in page table[b table_stride + i], S = 1 << page_shift
    const int32_t* table;
    int64_t table_stride;
    int num_pages, page_shift;
    const int32_t* lengths;  // [B], or null: every sequence has `capacity` keys
    int capacity;            // keys of K and V (paged: entries of a table row times S)
    int paged;
    int B, H, Hkv, G, T, D, Dv;
    // Position of token 0: length - T (positions_from_end), or query_offset.
    // With lengths and query_offset, tokens at or past the length are padding:
    // their rows are zero.
    int positions_from_end;
    int64_t query_offset;
    int window, sinks;  // window 0: none
    float scale, softcap;
    const float* alibi;  // [H] or null
    int out_f32;
    int row_tiles;  // per (sequence, key-value head)
    // Workgroups per tile. A tile shares its own steps among as many of them as
    // get min_steps each; the others have nothing to do.
    int splits, min_steps;
    float* part_o;   // [tiles][splits][rows of a tile][Dv]
    float* part_ml;  // [tiles][splits][rows of a tile][2]: max (log2 units), sum
};

constexpr int kStreamThreads = 256;
constexpr int kStreamKeys = 16;  // keys of a block, the unit in which K and V are read

// Head dim that a stream kernel is built for: 64, 128 or 256 (0: none).
int stream_kernel_dim(int D, int Dv);
// Rows of a tile: 16 or 32.
int stream_tile_rows(int dtype, int kernel_dim, int rows);
// Keys of a wavefront's step.
int stream_step_keys(int dtype, int kernel_dim);
hipError_t launch_stream(const StreamArgs& a, int dtype, hipStream_t s);

// Prompts on the matrix cores with K and V staged through LDS (window_fwd.hip).
struct WindowArgs {
    FwdArgs f;  // B, H (query heads), M, N, D, Dv, strides, scale, score_mod, out_f32, num_q_tiles
    int G;      // query heads per key-value head
    int window, sinks;
    int query_offset;
    const int32_t* lengths;
    int key_splits;  // wavefronts that share the keys of 32 rows: 1, or 2 up to kernel dim 128
};
// Query rows of a workgroup.
inline int window_rows(int key_splits) { return 4 * kQueriesPerWave / key_splits; }
hipError_t launch_window(const WindowArgs& a, int dtype, hipStream_t s);

// New rows into pages.
struct CacheWriteArgs {
    const void* k;
    const void* v;
    void* k_pages;
    void* v_pages;
    int64_t k_sb, k_sh, k_st;  // batch, head, token
    int64_t v_sb, v_sh, v_st;
    int64_t kp_sp, kp_sh, kp_st;  // page, head, token
    int64_t vp_sp, vp_sh, vp_st;
    const int32_t* table;
    int64_t table_stride;
    int num_pages, page_shift, max_pages;
    const int32_t* lengths;  // [B] tokens of each sequence with the new ones
    const int32_t* counts;   // [B] new tokens, or null: T
    int B, Hkv, T;
    int k_bytes, v_bytes;  // bytes of a K and a V row
    int elem;              // bytes of an element
};
bool cache_write_fits(const CacheWriteArgs& a);  // in one launch
hipError_t launch_cache_write(const CacheWriteArgs& a, hipStream_t s);

// Whole pages src -> dst in several pools of one geometry. The words of a
// launch (its arguments hold 4 KB) are the pools' addresses, low word first, then
// the pairs: a word each, dst above src, or with `wide` (pages past 2^16) two.
constexpr int kCopyWords = 976;
struct CopyPagesArgs {
    uint32_t words[kCopyWords];
    int64_t page_stride;  // bytes
    int64_t page_bytes;
    int num_pools, num_pairs, wide;
};
hipError_t launch_copy_pages(const CopyPagesArgs& a, hipStream_t s);

}  // namespace ofh
