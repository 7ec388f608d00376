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

    // A batch in groups whose sequences share their first keys. Those are read by
    // tiles of all rows of a group (kPrefix), the rest by each sequence's own
    // (kTail). Group g has the sequences [group_starts[g], group_starts[g + 1]), of
    // which each shares its first shared[b] keys, whole pages, in the pages of the
    // group's first sequence.
    const int32_t* group_starts;
    const int32_t* shared;
    int groups;
    int prefix_tiles, prefix_splits, prefix_min_steps;
    float* prefix_o;   // [prefix_splits][B Hkv T G][Dv]
    float* prefix_ml;  // [prefix_splits][B Hkv T G][2]

    // Selected pages (kSelected): row (b, hk, t) of `selected` lists the pages,
    // by their places in b's table row, whose keys the token sees. B counts tokens
    // then (of `tokens` per sequence) and T is 1.
    const int32_t* selected;
    int num_selected, tokens;
};

// Where a tile's rows find their keys.
enum StreamSource {
    kContiguous,
    kPaged,
    kTail,      // paged, behind what the sequence's group shares
    kPrefix,    // the pages that a group shares; rows of all its sequences
    kSelected,  // selected pages
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

// Attention over groups of sequences that share pages, and over selected pages.
// The prefix writes its partial rows (prefix_*); the tail's launch reads the rest
// and joins both.
// How the shared keys are read: rows of a tile, keys of a step, workgroups that a CU
// runs at once.
struct PrefixKernel {
    int rows, step_keys, key_splits;  // key_splits: of prefix_fwd.hip's kernel, 0: the streaming kernel
    int per_cu;
};
// Parts to divide the shared keys of `units` tiles and heads into, beside `own` tiles
// and heads of the sequences' own keys in `own_parts` workgroups.
int64_t prefix_parts(const PrefixKernel& k, int64_t units, int64_t own, int64_t own_parts);
PrefixKernel prefix_kernel(const StreamArgs& a, int dtype, int rows);  // of the largest group
__host__ __device__ inline int64_t prefix_grid(const StreamArgs& a) {  // (filled up to eights)
    return ((int64_t)a.Hkv * a.prefix_splits + 7) / 8 * 8 * a.prefix_tiles;
}
__host__ __device__ inline int64_t tail_grid(const StreamArgs& a) { return (int64_t)a.B * a.Hkv * a.row_tiles * a.splits; }
inline int64_t shared_grid(const StreamArgs& a) { return prefix_grid(a) + (tail_grid(a) + 7) / 8 * 8; }
// All of a call: the streaming kernel, and the other (kernel.key_splits > 0).
hipError_t launch_stream_shared(const StreamArgs& a, int dtype, int prefix_rows, hipStream_t s);
hipError_t launch_prefix_shared(const StreamArgs& a, int dtype, int key_splits, hipStream_t s);
// Parts of it: the sequences' own keys and the join, the join.
hipError_t launch_stream_tail(const StreamArgs& a, int dtype, hipStream_t s);
hipError_t launch_stream_join(const StreamArgs& a, int dtype, hipStream_t s);
hipError_t launch_stream_selected(const StreamArgs& a, int dtype, hipStream_t s);

// Bounds of the keys of pages: the pages that hold the last counts[b] tokens of each
// sequence (`touched` of them at most). bounds [page][head][lo, hi][D].
struct PageBoundsArgs {
    const void* k_pages;
    void* bounds;
    int64_t k_sp, k_sh, k_st;  // page, head, token
    int64_t b_sp, b_sh, b_st;  // page, head, from lo to hi
    const int32_t* table;
    int64_t table_stride;
    int num_pages, page_shift, max_pages;
    const int32_t* lengths;
    const int32_t* counts;  // or null: T
    int B, Hkv, T, D, touched;
};
bool page_bounds_fits(const PageBoundsArgs& a);
hipError_t launch_page_bounds(const PageBoundsArgs& a, int dtype, hipStream_t s);

// `pages` places of the table's row for each (b, hk, t): the first and the recent
// ones of those with keys up to the token, and the others of the highest score.
struct SelectArgs {
    const void* q;
    const void* bounds;
    int32_t* selected;  // [B][Hkv][T][pages], ascending, then -1
    uint32_t* scores;   // [B][Hkv][T][max_pages]
    int64_t q_sb, q_sh, q_st;
    int64_t b_sp, b_sh, b_st;
    const int32_t* table;
    int64_t table_stride;
    int num_pages, page_shift, max_pages;
    const int32_t* lengths;
    int B, Hkv, G, T, D;
    int pages, first_pages, recent_pages;
    int negative;  // scores of -q
};
bool page_select_fits(const SelectArgs& a, int dtype);
hipError_t launch_page_select(const SelectArgs& a, int dtype, hipStream_t s);

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

// Rotary positions. The first R columns of a row are R / 2 pairs, (i, i + R / 2)
// or interleaved (2 i, 2 i + 1); pair i turns by position freq[i] radians.
struct Rotation {
    const double* freq;
    int R, interleaved;
    float magnitude;
    int transpose;  // turn back
};
constexpr int kRotaryMaxDim = 1024;  // of a head

struct RotaryArgs {
    const void* x;
    void* o;
    int64_t x_sb, x_sh, x_st;  // batch, head, token
    int64_t o_sb, o_sh, o_st;
    int B, H, T, D;
    Rotation r;
    // position of token (b, t): positions[b pos_sb + t], or lengths[b] - T + t, or offset + t
    const int32_t* positions;
    int64_t pos_sb;
    const int32_t* lengths;
    int64_t offset;
};
bool rotary_fits(const RotaryArgs& a);  // in one launch
hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s);

// New rows into pages with K turned on the way, and Q turned into q_out (H 0: no Q).
struct CacheAppendArgs {
    CacheWriteArgs w;
    const void* q;
    void* q_out;
    int64_t q_sb, q_sh, q_st;
    int64_t o_sb, o_sh, o_st;
    int H, D, Dv;
    Rotation r;
};
bool cache_append_fits(const CacheAppendArgs& a);
hipError_t launch_cache_append(const CacheAppendArgs& a, int dtype, hipStream_t s);

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
