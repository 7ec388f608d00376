// C ABI of the serving operators (include/onednn_flash_hip.h): windowed and paged
// attention, also over shared prefixes and selected pages, bounds and selection of
// pages, writing and copying of cache pages. Argument checks, layout
// resolution, the split of a call's keys over workgroups, scratch.

#include "onednn_flash_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <string>
#include <vector>

#include "capi_shared.h"
#include "serving_checks.h"
#include "serving_kernels.h"

using ofh::api_error;

namespace {

struct Tensor {
    const char* name;
    const void* ptr;
    const int64_t* strides;
    size_t last;
};

// 16-byte accesses: pointer and strides; token offsets that a lane adds in 32 bits.
int check_tensor(const Tensor& t, int elem, bool check_ptr, int64_t rows) {
    if (check_ptr && t.ptr == nullptr) return invalid(std::string(t.name) + " must be non-null");
    if (check_ptr && ((uintptr_t)t.ptr & 15) != 0) return unsupported(std::string(t.name) + " must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
        if (t.strides[i] < 0) return invalid(std::string(t.name) + " strides must be non-negative");
        if (t.strides[i] * elem % 16 != 0)
            return unsupported(std::string(t.name) + " strides must be multiples of 16 bytes");
    }
    if (t.strides[2] > (kMaxOffset / elem - (int64_t)t.last) / rows)
        return unsupported(std::string(t.name) + " token stride is too large");
    return OFH_SUCCESS;
}

// What both attentions ask.
int check_common(size_t batch, size_t heads, size_t kv_heads, size_t tokens, size_t D, size_t Dv, int dtype,
                 int out_dtype, float scale, float softcap, size_t window, size_t sinks, int max_key_splits) {
    if (batch == 0 || heads == 0 || kv_heads == 0 || tokens == 0 || D == 0 || Dv == 0)
        return invalid("attention dimensions must be non-zero");
    if (heads % kv_heads != 0) return invalid("heads must be a multiple of kv_heads");
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    if (out_dtype != dtype && out_dtype != OFH_DTYPE_F32) return invalid("out_dtype must equal dtype or be f32");
    if (!std::isfinite(scale)) return invalid("scale must be finite");
    if (!(softcap >= 0.0f) || !std::isfinite(softcap)) return invalid("softcap must be finite and >= 0");
    if (max_key_splits < 0) return invalid("max_key_splits must be >= 0");
    if (window == 0 && sinks != 0) return invalid("sink_tokens need a window");
    const size_t step = dtype == OFH_DTYPE_F32 ? 4 : 8;
    if (D % step != 0 || Dv % step != 0 || D > 256 || Dv > 256)
        return unsupported("head_dim and value_dim must be multiples of " + std::to_string(step) + " up to 256");
    if (batch > (size_t)kMaxTokens || heads > (size_t)kMaxTokens || tokens > (size_t)kMaxTokens ||
        window > (size_t)kMaxTokens || sinks > (size_t)kMaxTokens || heads * tokens > (size_t)kMaxTokens ||
        batch * heads > (size_t)kMaxTokens)
        return unsupported("attention dimensions exceed the 32-bit index range");
    return OFH_SUCCESS;
}

// The cap as the kernels take it. Their 2 log2(e) / cap has no value for a cap
// near 2^-126, and scores within 2^-40 of 0 have the same weights in 32 bits.
float kernel_softcap(float softcap) { return softcap > 0.0f ? std::max(softcap, 0x1p-40f) : 0.0f; }

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Split of a row tile's keys over workgroups. The lengths are on the device, so
// the grid is sized for the most keys that a tile can see, and every tile
// shares its own keys among as many of its workgroups as get min_steps steps
// (the rest leave at once).
struct Split {
    int tile_rows, row_tiles, splits, min_steps;
    int64_t units;
    size_t bytes;
};

// Measured (us, bf16 H32/8 D128 unless said, parts per tile): a workgroup per CU
// fills the memory's rate, so more parts only add starts and rows to join: B8
// N4000 4 parts 31.6, 16 36.0; D256 B4 H16/4 N20000 16 parts 65, 32 71; two per CU
// pay off with long parts: f32 D128 B8 H16 N2000-8000 2 parts 140, 4 133, D64 B16
// H16 N2000-8000 1 part 82, 2 75, but B32 N100-600 1 part 15.4, 2 20.1. Parts of a
// step per wavefront (4): one sequence of 1001 keys 12.5, of 8 steps 12.7, of 16
// 16.3; with less than four such parts in all the join costs more than they save:
// B4 N300 split 12.8, unsplit 9.8.
Split plan_split(const ofh::StreamArgs& a, int dtype, int max_key_splits) {
    Split s{};
    const int dk = ofh::stream_kernel_dim(a.D, a.Dv);
    s.tile_rows = ofh::stream_tile_rows(dtype, dk, a.T * a.G);
    s.row_tiles = (int)(((int64_t)a.T * a.G + s.tile_rows - 1) / s.tile_rows);
    s.units = (int64_t)a.B * a.Hkv * s.row_tiles;
    s.splits = 1;
    s.min_steps = ofh::kStreamThreads / 64;
    const int64_t tile_tokens = std::min<int64_t>(a.T, s.tile_rows / a.G + 2);
    int64_t keys = a.capacity;
    if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + a.sinks + tile_tokens + 2 * ofh::kStreamKeys);
    const int step = ofh::stream_step_keys(dtype, dk);
    const int64_t steps = (keys + step - 1) / step;
    if (steps < 4 * s.min_steps) return s;
    const int64_t one = (ofh::kComputeUnits + s.units - 1) / s.units, two = (2 * ofh::kComputeUnits + s.units - 1) / s.units;
    int64_t n = dk <= 128 ? std::max(one, std::min<int64_t>(two, steps / 32)) : one;
    n = std::min<int64_t>({n, steps / s.min_steps, max_key_splits > 0 ? max_key_splits : 128});
    s.splits = (int)std::max<int64_t>(1, n);
    const size_t rows = (size_t)s.units * s.splits * s.tile_rows;
    s.bytes = s.splits > 1 ? round256(rows * a.Dv * 4) + rows * 8 : 0;
    return s;
}

void unsplit(Split& s) {
    s.splits = 1;
    s.bytes = 0;
}

// The call's scratch: the caller's, or the library's of the stream (held by `lease`).
int take_workspace(size_t need, void*& workspace, size_t workspace_bytes, hipStream_t stream, ofh::ScratchLease& lease) {
    const std::string small = "workspace too small: need " + std::to_string(need) + " bytes";
    if (need > 0 && workspace == nullptr) {
        bool fits = true;
        if (int rc = lease.acquire(need, stream, fits)) return rc;
        if (!fits) return api_error(OFH_ERROR_WORKSPACE_TOO_SMALL, small);
        workspace = lease.ptr;
    } else if (need > workspace_bytes) {
        return api_error(OFH_ERROR_WORKSPACE_TOO_SMALL, small);
    }
    if (need > 0 && ((uintptr_t)workspace & 15) != 0) return unsupported("workspace must be 16-byte aligned");
    return OFH_SUCCESS;
}

int run_stream(ofh::StreamArgs& a, int dtype, Split s, void* workspace, size_t workspace_bytes, hipStream_t stream,
               hipError_t (*launch)(const ofh::StreamArgs&, int, hipStream_t) = ofh::launch_stream) {
    if (!ofh::grid_fits(s.units * s.splits, ofh::kStreamThreads) ||
        !ofh::grid_fits((int64_t)a.B * a.Hkv * a.T * a.G * ((a.Dv + 31) / 32), 64))
        return unsupported("attention call exceeds the launch range");
    ofh::ScratchLease lease;
    if (s.bytes > 0 && workspace == nullptr) {
        bool fits = true;
        if (int rc = lease.acquire(s.bytes, stream, fits)) return rc;
        if (fits) workspace = lease.ptr;
        else unsplit(s);
    } else if (s.bytes > workspace_bytes) {
        return api_error(OFH_ERROR_WORKSPACE_TOO_SMALL, "workspace too small: need " + std::to_string(s.bytes) + " bytes");
    }
    if (s.bytes > 0 && ((uintptr_t)workspace & 15) != 0) return unsupported("workspace must be 16-byte aligned");
    a.row_tiles = s.row_tiles;
    a.splits = s.splits;
    a.min_steps = s.min_steps;
    if (s.splits > 1) {
        const size_t rows = (size_t)s.units * s.splits * s.tile_rows;
        a.part_o = static_cast<float*>(workspace);
        a.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(rows * a.Dv * 4));
    }
    OFH_HIP_CHECK(launch(a, dtype, stream));
    return lease.release();
}

void set_rows(ofh::StreamArgs& a, size_t batch, size_t heads, size_t kv_heads, size_t tokens, size_t D, size_t Dv) {
    a.B = (int)batch;
    a.H = (int)heads;
    a.Hkv = (int)kv_heads;
    a.G = (int)(heads / kv_heads);
    a.T = (int)tokens;
    a.D = (int)D;
    a.Dv = (int)Dv;
}

void set_strides(ofh::StreamArgs& a, const int64_t q[3], const int64_t k[3], const int64_t v[3], const int64_t o[3]) {
    a.q_sb = q[0]; a.q_sh = q[1]; a.q_st = q[2];
    a.k_sp = k[0]; a.k_sh = k[1]; a.k_st = k[2];
    a.v_sp = v[0]; a.v_sh = v[1]; a.v_st = v[2];
    a.o_sb = o[0]; a.o_sh = o[1]; a.o_st = o[2];
}

// Checks a windowed call and fills its arguments (pointers may be null when only its plan is asked for).
int window_args(const ofh_window_params* p, bool check_ptrs, const void* q, const void* k, const void* v, void* out,
                ofh::StreamArgs& a) {
    if (p == nullptr) return invalid("params must be non-null");
    if (p->struct_size != sizeof(*p))
        return invalid("ofh_window_params.struct_size mismatch (call ofh_window_params_init)");
    if (int rc = check_common(p->batch, p->heads, p->kv_heads, p->query_tokens, p->head_dim, p->value_dim, p->dtype,
                              p->out_dtype, p->scale, p->softcap, p->window, p->sink_tokens, p->max_key_splits))
        return rc;
    if (p->key_tokens == 0) return invalid("attention dimensions must be non-zero");
    // (positions of whole row tiles are 32-bit)
    if (p->key_tokens > (size_t)kMaxTokens || p->query_offset > (size_t)kMaxTokens ||
        p->query_offset + p->query_tokens > (size_t)kMaxTokens)
        return unsupported("attention dimensions exceed the 32-bit index range");
    int64_t qs[3], ks[3], vs[3], os[3];
    resolve_strides(qs, p->q_strides, p->heads, p->query_tokens, p->head_dim);
    resolve_strides(ks, p->k_strides, p->kv_heads, p->key_tokens, p->head_dim);
    resolve_strides(vs, p->v_strides, p->kv_heads, p->key_tokens, p->value_dim);
    resolve_strides(os, p->o_strides, p->heads, p->query_tokens, p->value_dim);
    const int es = elem_size(p->dtype);
    const Tensor in[] = {{"q", q, qs, p->head_dim}, {"k", k, ks, p->head_dim}, {"v", v, vs, p->value_dim}};
    for (const Tensor& t : in)
        if (int rc = check_tensor(t, es, check_ptrs, ofh::kStreamKeys)) return rc;
    if (int rc = check_tensor({"out", out, os, p->value_dim}, elem_size(p->out_dtype), check_ptrs, 1)) return rc;
    a = ofh::StreamArgs{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.o = out;
    set_rows(a, p->batch, p->heads, p->kv_heads, p->query_tokens, p->head_dim, p->value_dim);
    set_strides(a, qs, ks, vs, os);
    a.lengths = p->lengths;
    a.capacity = (int)p->key_tokens;
    a.query_offset = (int64_t)p->query_offset;
    a.window = (int)p->window;
    a.sinks = (int)p->sink_tokens;
    a.scale = p->scale;
    a.softcap = kernel_softcap(p->softcap);
    a.alibi = p->alibi_slopes;
    a.out_f32 = p->out_dtype == OFH_DTYPE_F32;
    return OFH_SUCCESS;
}

// How a windowed call runs: the streaming kernel (0), or in 16 bits K and V
// staged through LDS with 128 rows per workgroup (1), or 64 (2).
//
// 64 rows, whose keys two wavefront groups share, have half the chain and twice
// the workgroups: faster while 128-row tiles leave CUs idle (us, 128 / 64 rows,
// D128: B1 H32 N512 16.2 / 13.0, B1 H8 N2000 window 512 21.3 / 16.2, B2 H16 N700
// 19.6 / 17.8), slower past that (480 tiles, B1 H40 N1500 window 256: 24.8 /
// 28.6; 768, B2 H32 N1500: 53 / 68).
//
// The streaming kernel splits the keys over workgroups, so few rows against many
// keys are its calls; but each of its tiles of 16 or 32 rows reads all its keys
// itself. Measured (us, streaming / LDS, tiles): D128 N1500 B1 H8 M32 14.9 /
// 26.8 (8), B8 H32/8 M4 23.7 / 28.1 (64), B4 H16 M32 32.1 / 28.0 (64), B8 H32/8
// M16 46.0 / 28.0 (128); N6000 B1 H32/8 M32 38.7 / 88 (32), B4 H16 M63 73 / 86
// (128), B8 H32/8 M32 110 / 89 (256); N300 B1 H32/8 M4 9.2 / 10.1 (8), B4 H16 M63
// 13.1 / 10.8 (128); D256, where the LDS kernel has one workgroup per CU: B4 H16
// M32 N6000 112 / 344 (128), B32 H32/4 M16 N6000 484 / 1317 (1024, four rounds),
// B8 H32/8 M63 N6000 464 / 341 (1024, one round), B8 H32/8 M32 N300 28.5 / 24.0
// (512).
int window_groups(const ofh::StreamArgs& a, int dtype) {
    if (dtype == OFH_DTYPE_F32) return 0;
    // (a lane adds the offsets of up to 128 rows in 32 bits)
    for (int64_t stride : {a.k_st, a.v_st})
        if (stride > (kMaxOffset / 2 - 256) / 256) return 0;
    const int dk = ofh::stream_kernel_dim(a.D, a.Dv);
    const int64_t heads = (int64_t)a.B * a.H;
    const int64_t wide = heads * ((a.T + ofh::window_rows(1) - 1) / ofh::window_rows(1));
    const int groups = dk <= 128 && wide <= ofh::kComputeUnits ? 2 : 1;
    const int64_t wgs = groups == 1 ? wide : heads * ((a.T + ofh::window_rows(2) - 1) / ofh::window_rows(2));
    const int64_t slots = dk <= 128 ? 2 * ofh::kComputeUnits : ofh::kComputeUnits;
    const int64_t rounds = (wgs + slots - 1) / slots;
    const int rows = ofh::stream_tile_rows(dtype, dk, a.T * a.G);
    const int64_t tiles = (int64_t)a.B * a.Hkv * (((int64_t)a.T * a.G + rows - 1) / rows);
    int64_t keys = a.capacity;
    if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + a.sinks + a.T);
    const int64_t few = dk == 256 ? 400 : std::min<int64_t>(keys / 24, 160);
    return tiles <= rounds * few ? 0 : groups;
}

int run_window(const ofh::StreamArgs& a, int dtype, int groups, hipStream_t stream) {
    ofh::WindowArgs w{};
    ofh::FwdArgs& f = w.f;
    f.q = a.q;
    f.k = a.k;
    f.v = a.v;
    f.o = a.o;
    f.q_sb = a.q_sb; f.q_sh = a.q_sh; f.q_sm = a.q_st;
    f.k_sb = a.k_sp; f.k_sh = a.k_sh; f.k_sn = a.k_st;
    f.v_sb = a.v_sp; f.v_sh = a.v_sh; f.v_sn = a.v_st;
    f.o_sb = a.o_sb; f.o_sh = a.o_sh; f.o_sm = a.o_st;
    f.B = a.B;
    f.H = a.H;
    f.M = a.T;
    f.N = a.capacity;
    f.D = a.D;
    f.Dv = a.Dv;
    f.scale = a.scale;
    f.scale_log2 = a.scale * 1.4426950408889634f;
    f.softcap = a.softcap;
    f.inv_softcap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    f.alibi = a.alibi;
    f.out_f32 = a.out_f32;
    const int rows = ofh::window_rows(groups);
    f.num_q_tiles = (a.T + rows - 1) / rows;
    w.G = a.G;
    w.window = a.window;
    w.sinks = a.sinks;
    w.query_offset = (int)a.query_offset;
    w.lengths = a.lengths;
    w.key_splits = groups;
    if (!ofh::grid_fits((int64_t)a.B * a.H * f.num_q_tiles, 256)) return unsupported("attention call exceeds the launch range");
    OFH_HIP_CHECK(ofh::launch_window(w, dtype, stream));
    return OFH_SUCCESS;
}

int paged_args(const ofh_paged_params* p, bool check_ptrs, const void* q, const void* k, const void* v, void* out,
               ofh::StreamArgs& a) {
    if (p == nullptr) return invalid("params must be non-null");
    if (p->struct_size != sizeof(*p))
        return invalid("ofh_paged_params.struct_size mismatch (call ofh_paged_params_init)");
    if (int rc = check_common(p->batch, p->heads, p->kv_heads, p->query_tokens, p->head_dim, p->value_dim, p->dtype,
                              p->out_dtype, p->scale, p->softcap, p->window, p->sink_tokens, p->max_key_splits))
        return rc;
    if (int rc = check_pages(p->num_pages, p->page_size, p->max_pages, p->table_stride, p->page_table, p->lengths,
                             check_ptrs))
        return rc;
    int64_t qs[3], ks[3], vs[3], os[3];
    resolve_strides(qs, p->q_strides, p->heads, p->query_tokens, p->head_dim);
    resolve_strides(ks, p->k_strides, p->kv_heads, p->page_size, p->head_dim);
    resolve_strides(vs, p->v_strides, p->kv_heads, p->page_size, p->value_dim);
    resolve_strides(os, p->o_strides, p->heads, p->query_tokens, p->value_dim);
    const int es = elem_size(p->dtype);
    const Tensor in[] = {{"q", q, qs, p->head_dim}, {"k_pages", k, ks, p->head_dim}, {"v_pages", v, vs, p->value_dim}};
    for (const Tensor& t : in)
        if (int rc = check_tensor(t, es, check_ptrs, ofh::kStreamKeys)) return rc;
    if (int rc = check_tensor({"out", out, os, p->value_dim}, elem_size(p->out_dtype), check_ptrs, 1)) return rc;
    a = ofh::StreamArgs{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.o = out;
    set_rows(a, p->batch, p->heads, p->kv_heads, p->query_tokens, p->head_dim, p->value_dim);
    set_strides(a, qs, ks, vs, os);
    a.paged = 1;
    a.positions_from_end = 1;
    a.table = p->page_table;
    a.table_stride = p->table_stride != 0 ? p->table_stride : (int64_t)p->max_pages;
    a.num_pages = (int)p->num_pages;
    a.page_shift = log2_of(p->page_size);
    a.lengths = p->lengths;
    a.capacity = (int)(p->max_pages * p->page_size);
    a.window = (int)p->window;
    a.sinks = (int)p->sink_tokens;
    a.scale = p->scale;
    a.softcap = kernel_softcap(p->softcap);
    a.alibi = p->alibi_slopes;
    a.out_f32 = p->out_dtype == OFH_DTYPE_F32;
    return OFH_SUCCESS;
}

// The bounds of a pool's pages, [page, kv_head, 2, head_dim].
int check_bounds(size_t batch, size_t kv_heads, size_t D, int dtype, const int64_t in[3], const void* bounds,
                 bool check_ptr, int64_t strides[3]) {
    if (batch == 0 || kv_heads == 0 || D == 0) return invalid("cache dimensions must be non-zero");
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    const size_t step = dtype == OFH_DTYPE_F32 ? 4 : 8;
    if (D % step != 0 || D > 256) return unsupported("head_dim must be a multiple of " + std::to_string(step) + " up to 256");
    if (batch > (size_t)kMaxTokens || kv_heads > (size_t)kMaxTokens)
        return unsupported("cache dimensions exceed the 32-bit index range");
    resolve_strides(strides, in, kv_heads, 2, D);
    return check_tensor({"bounds", bounds, strides, D}, elem_size(dtype), check_ptr, 1);
}

int select_args(const ofh_select_params* p, bool check_ptrs, const void* q, const void* bounds, int32_t* selected,
                ofh::SelectArgs& a) {
    if (p == nullptr) return invalid("params must be non-null");
    if (p->struct_size != sizeof(*p))
        return invalid("ofh_select_params.struct_size mismatch (call ofh_select_params_init)");
    if (p->heads == 0 || p->query_tokens == 0) return invalid("attention dimensions must be non-zero");
    int64_t qs[3], bs[3];
    if (int rc = check_bounds(p->batch, p->kv_heads, p->head_dim, p->dtype, p->bounds_strides, bounds, check_ptrs, bs))
        return rc;
    if (p->heads % p->kv_heads != 0) return invalid("heads must be a multiple of kv_heads");
    if (int rc = check_pages(p->num_pages, p->page_size, p->max_pages, p->table_stride, p->page_table, p->lengths, check_ptrs))
        return rc;
    if (p->pages == 0) return invalid("pages must be non-zero");
    if (p->first_pages > p->pages || p->recent_pages > p->pages - p->first_pages)
        return invalid("first_pages and recent_pages must be at most pages together");
    if (p->heads > (size_t)kMaxTokens || p->query_tokens > (size_t)kMaxTokens || p->pages > (size_t)kMaxTokens ||
        (uint64_t)p->heads * p->query_tokens > (uint64_t)kMaxTokens ||
        (uint64_t)p->batch * p->heads * p->query_tokens > (uint64_t)kMaxTokens)
        return unsupported("attention dimensions exceed the 32-bit index range");
    resolve_strides(qs, p->q_strides, p->heads, p->query_tokens, p->head_dim);
    for (int i = 0; i < 3; ++i)
        if (qs[i] < 0) return invalid("q strides must be non-negative");
    if (check_ptrs && (q == nullptr || selected == nullptr)) return invalid("q and selected must be non-null");
    if (check_ptrs && ((uintptr_t)q % elem_size(p->dtype) != 0 || (uintptr_t)selected % 4 != 0))
        return unsupported("q and selected must be aligned to their elements");
    a = ofh::SelectArgs{};
    a.q = q;
    a.bounds = bounds;
    a.selected = selected;
    a.q_sb = qs[0]; a.q_sh = qs[1]; a.q_st = qs[2];
    a.b_sp = bs[0]; a.b_sh = bs[1]; a.b_st = bs[2];
    a.table = p->page_table;
    a.table_stride = p->table_stride != 0 ? p->table_stride : (int64_t)p->max_pages;
    a.num_pages = (int)p->num_pages;
    a.page_shift = log2_of(p->page_size);
    a.max_pages = (int)p->max_pages;
    a.lengths = p->lengths;
    a.B = (int)p->batch;
    a.Hkv = (int)p->kv_heads;
    a.G = (int)(p->heads / p->kv_heads);
    a.T = (int)p->query_tokens;
    a.D = (int)p->head_dim;
    a.pages = (int)p->pages;
    a.first_pages = (int)p->first_pages;
    a.recent_pages = (int)p->recent_pages;
    a.negative = p->negative != 0;
    return OFH_SUCCESS;
}

// Scores, where a sequence can have more pages than it may take.
size_t select_bytes(const ofh::SelectArgs& a) {
    return a.max_pages > a.pages ? (size_t)a.B * a.Hkv * a.T * a.max_pages * 4 : 0;
}

// A batch in groups that share pages.
struct PrefixPlan {
    Split tail;
    ofh::PrefixKernel kernel;
    int tiles, splits, min_steps;
    size_t tail_o, tail_ml, prefix_o, prefix_ml;  // bytes
    size_t bytes() const { return tail_o + tail_ml + prefix_o + prefix_ml; }
};

int prefix_args(const ofh_paged_params* p, const ofh_prefix_groups* g, bool check_ptrs, const void* q, const void* k,
                const void* v, void* out, ofh::StreamArgs& a) {
    if (int rc = paged_args(p, check_ptrs, q, k, v, out, a)) return rc;
    if (g == nullptr) return invalid("groups must be non-null");
    if (g->struct_size != sizeof(*g))
        return invalid("ofh_prefix_groups.struct_size mismatch (call ofh_prefix_groups_init)");
    if (g->groups == 0 || g->groups > p->batch) return invalid("groups must be 1 to batch");
    if (check_ptrs && (g->starts == nullptr || g->shared_tokens == nullptr))
        return invalid("starts and shared_tokens must be non-null");
    if (g->least_shared > g->most_shared || g->most_shared > p->max_pages * p->page_size)
        return invalid("least_shared and most_shared must be within the table's tokens, in this order");
    if (g->sharing_groups > g->groups || g->sharing_sequences > p->batch || g->most_sequences > p->batch)
        return invalid("sharing groups and sequences must be within the batch's");
    // (rows of all sequences are numbered in 32 bits)
    if ((uint64_t)p->batch * p->heads * p->query_tokens > (uint64_t)kMaxTokens)
        return unsupported("attention dimensions exceed the 32-bit index range");
    a.group_starts = g->starts;
    a.shared = g->shared_tokens;
    a.groups = (int)g->groups;
    return OFH_SUCCESS;
}

PrefixPlan plan_prefix(const ofh::StreamArgs& a, int dtype, const ofh_prefix_groups* g, int max_key_splits) {
    PrefixPlan plan{};
    ofh::StreamArgs own = a;
    own.capacity = std::max(a.capacity - (int)g->least_shared, 1);
    plan.tail = plan_split(own, dtype, max_key_splits);
    const int64_t groups = g->sharing_groups > 0 ? (int64_t)g->sharing_groups : a.groups;
    const int64_t sequences = g->sharing_sequences > 0 ? (int64_t)g->sharing_sequences : a.B;
    const int64_t largest = g->most_sequences > 0 ? (int64_t)g->most_sequences : (sequences + groups - 1) / groups;
    plan.kernel = ofh::prefix_kernel(a, dtype, (int)(largest * a.T * a.G));
    const int rows = plan.kernel.rows, step = plan.kernel.step_keys;
    // (a wavefront of the streaming kernel takes a step, a workgroup of the other)
    plan.min_steps = plan.kernel.key_splits == 0 ? ofh::kStreamThreads / 64 : 2;
    plan.tiles = (int)((sequences * a.T * a.G + groups * (rows - 1)) / rows);
    const int64_t steps = ((int64_t)g->most_shared + step - 1) / step;
    // (groups of a tile each at most have no more tiles than groups)
    const bool one_each = largest * a.T * a.G <= rows;
    const int64_t units = (int64_t)a.Hkv * (one_each ? std::min<int64_t>(plan.tiles, groups) : plan.tiles);
    const int64_t parts =
        ofh::prefix_parts(plan.kernel, units, plan.tail.units, plan.tail.units * plan.tail.splits);
    const int64_t n = std::min<int64_t>({parts, steps / plan.min_steps, max_key_splits > 0 ? max_key_splits : 128});
    plan.splits = (int)std::max<int64_t>(1, n);
    const size_t tail_rows = (size_t)plan.tail.units * plan.tail.splits * plan.tail.tile_rows;
    const size_t prefix_rows = (size_t)a.B * a.Hkv * a.T * a.G * plan.splits;
    plan.tail_o = round256(tail_rows * a.Dv * 4);
    plan.tail_ml = round256(tail_rows * 8);
    plan.prefix_o = round256(prefix_rows * a.Dv * 4);
    plan.prefix_ml = round256(prefix_rows * 8);
    return plan;
}

int run_prefix(ofh::StreamArgs& a, int dtype, const PrefixPlan& plan, void* workspace, size_t workspace_bytes,
               hipStream_t stream) {
    if (!ofh::grid_fits(plan.tail.units * plan.tail.splits, ofh::kStreamThreads) ||
        !ofh::grid_fits(((int64_t)a.Hkv * plan.splits + 8) * plan.tiles + plan.tail.units * plan.tail.splits + 8,
                        ofh::kStreamThreads) ||
        !ofh::grid_fits((int64_t)a.B * a.Hkv * a.T * a.G * ((a.Dv + 31) / 32), 64))
        return unsupported("attention call exceeds the launch range");
    ofh::ScratchLease lease;
    if (int rc = take_workspace(plan.bytes(), workspace, workspace_bytes, stream, lease)) return rc;
    a.row_tiles = plan.tail.row_tiles;
    a.splits = plan.tail.splits;
    a.min_steps = plan.tail.min_steps;
    a.prefix_tiles = plan.tiles;
    a.prefix_splits = plan.splits;
    a.prefix_min_steps = plan.min_steps;
    char* at = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(at);
    a.part_ml = reinterpret_cast<float*>(at += plan.tail_o);
    a.prefix_o = reinterpret_cast<float*>(at += plan.tail_ml);
    a.prefix_ml = reinterpret_cast<float*>(at += plan.prefix_o);
    if (plan.kernel.key_splits > 0) OFH_HIP_CHECK(ofh::launch_prefix_shared(a, dtype, plan.kernel.key_splits, stream));
    else OFH_HIP_CHECK(ofh::launch_stream_shared(a, dtype, plan.kernel.rows, stream));
    return lease.release();
}

// Attention over selected pages: a token is a sequence of the kernels.
int selected_args(const ofh_paged_params* p, size_t pages, bool check_ptrs, const int32_t* selected, const void* q,
                  const void* k, const void* v, void* out, ofh::StreamArgs& a) {
    if (int rc = paged_args(p, check_ptrs, q, k, v, out, a)) return rc;
    if (pages == 0) return invalid("pages must be non-zero");
    if (p->window != 0) return unsupported("selected pages take no window");
    if (check_ptrs && selected == nullptr) return invalid("selected must be non-null");
    if (pages > (size_t)kMaxTokens || (uint64_t)pages * p->page_size > (uint64_t)kMaxTokens)
        return unsupported("selected pages exceed the 32-bit index range");
    if ((uint64_t)p->batch * p->heads * p->query_tokens > (uint64_t)kMaxTokens)
        return unsupported("attention dimensions exceed the 32-bit index range");
    a.selected = selected;
    a.num_selected = (int)pages;
    a.tokens = a.T;
    a.B *= a.T;
    a.T = 1;
    return OFH_SUCCESS;
}

// Tokens take equally many keys, so a workgroup per CU is enough, and parts of eight
// steps, four at kernel dim 256 (us, parts per tile: bf16 B32 H32/8 D128, 64 pages of
// 32, 256 tiles 1 52, 2 59; B8, 64 tiles, 2 22.8, 4 20.2; f16 B1, 64 pages of 64, 8 tiles,
// 8 16.3, 16 13.8, 32 14.7; bf16 D256, 64 pages of 32, 8 tiles, 8 18.7, 16 16.3); with less
// than 32 steps the join costs what they save (f32 B4 H8 3 tokens D64, 20 steps, 96
// tiles 1 15.2, 2 16.4, 3 18.7).
Split plan_selected(const ofh::StreamArgs& a, int dtype, int max_key_splits) {
    ofh::StreamArgs seen = a;
    seen.capacity = (int)std::min<int64_t>(a.capacity, (int64_t)a.num_selected << a.page_shift);
    Split s = plan_split(seen, dtype, 1);
    const int dk = ofh::stream_kernel_dim(a.D, a.Dv), step = ofh::stream_step_keys(dtype, dk);
    const int64_t steps = ((int64_t)seen.capacity + step - 1) / step;
    if (steps < 32) return s;
    const int64_t least = dk == 256 ? 4 : 8;
    const int64_t n =
        std::min<int64_t>({ofh::kComputeUnits / s.units, steps / least, max_key_splits > 0 ? max_key_splits : 128});
    if (n <= 1) return s;
    s.splits = (int)n;
    const size_t rows = (size_t)s.units * s.splits * s.tile_rows;
    s.bytes = round256(rows * a.Dv * 4) + rows * 8;
    return s;
}

}  // namespace

extern "C" {

void ofh_window_params_init(ofh_window_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
    p->scale = 1.0f;
}

int ofh_window_attention_workspace_bytes(const ofh_window_params* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (bytes == nullptr) return invalid("bytes must be non-null");
        ofh::StreamArgs a;
        if (int rc = window_args(p, false, nullptr, nullptr, nullptr, nullptr, a)) return rc;
        *bytes = window_groups(a, p->dtype) > 0 ? 0 : plan_split(a, p->dtype, p->max_key_splits).bytes;
        return OFH_SUCCESS;
    });
}

int ofh_window_attention_fwd(const ofh_window_params* p, const void* q, const void* k, const void* v, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        ofh::StreamArgs a;
        if (int rc = window_args(p, true, q, k, v, out, a)) return rc;
        if (const int groups = window_groups(a, p->dtype))
            return run_window(a, p->dtype, groups, static_cast<hipStream_t>(stream));
        return run_stream(a, p->dtype, plan_split(a, p->dtype, p->max_key_splits), workspace, workspace_bytes,
                          static_cast<hipStream_t>(stream));
    });
}

void ofh_paged_params_init(ofh_paged_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
    p->query_tokens = 1;
    p->scale = 1.0f;
}

int ofh_paged_attention_workspace_bytes(const ofh_paged_params* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (bytes == nullptr) return invalid("bytes must be non-null");
        ofh::StreamArgs a;
        if (int rc = paged_args(p, false, nullptr, nullptr, nullptr, nullptr, a)) return rc;
        *bytes = plan_split(a, p->dtype, p->max_key_splits).bytes;
        return OFH_SUCCESS;
    });
}

int ofh_paged_attention_fwd(const ofh_paged_params* p, const void* q, const void* k_pages, const void* v_pages,
                            void* out, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        ofh::StreamArgs a;
        if (int rc = paged_args(p, true, q, k_pages, v_pages, out, a)) return rc;
        return run_stream(a, p->dtype, plan_split(a, p->dtype, p->max_key_splits), workspace, workspace_bytes,
                          static_cast<hipStream_t>(stream));
    });
}

void ofh_prefix_groups_init(ofh_prefix_groups* g) {
    if (g == nullptr) return;
    std::memset(g, 0, sizeof(*g));
    g->struct_size = sizeof(*g);
}

int ofh_shared_prefix_workspace_bytes(const ofh_paged_params* p, const ofh_prefix_groups* g, size_t* bytes) {
    return guarded([&]() -> int {
        if (bytes == nullptr) return invalid("bytes must be non-null");
        ofh::StreamArgs a;
        if (int rc = prefix_args(p, g, false, nullptr, nullptr, nullptr, nullptr, a)) return rc;
        *bytes = plan_prefix(a, p->dtype, g, p->max_key_splits).bytes();
        return OFH_SUCCESS;
    });
}

int ofh_shared_prefix_attention_fwd(const ofh_paged_params* p, const ofh_prefix_groups* g, const void* q,
                                    const void* k_pages, const void* v_pages, void* out, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        ofh::StreamArgs a;
        if (int rc = prefix_args(p, g, true, q, k_pages, v_pages, out, a)) return rc;
        return run_prefix(a, p->dtype, plan_prefix(a, p->dtype, g, p->max_key_splits), workspace, workspace_bytes,
                          static_cast<hipStream_t>(stream));
    });
}

int ofh_selected_attention_workspace_bytes(const ofh_paged_params* p, size_t pages, size_t* bytes) {
    return guarded([&]() -> int {
        if (bytes == nullptr) return invalid("bytes must be non-null");
        ofh::StreamArgs a;
        if (int rc = selected_args(p, pages, false, nullptr, nullptr, nullptr, nullptr, nullptr, a)) return rc;
        *bytes = plan_selected(a, p->dtype, p->max_key_splits).bytes;
        return OFH_SUCCESS;
    });
}

int ofh_selected_attention_fwd(const ofh_paged_params* p, const int32_t* selected, size_t pages, const void* q,
                               const void* k_pages, const void* v_pages, void* out, void* workspace,
                               size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        ofh::StreamArgs a;
        if (int rc = selected_args(p, pages, true, selected, q, k_pages, v_pages, out, a)) return rc;
        return run_stream(a, p->dtype, plan_selected(a, p->dtype, p->max_key_splits), workspace, workspace_bytes,
                          static_cast<hipStream_t>(stream), ofh::launch_stream_selected);
    });
}

void ofh_page_bounds_params_init(ofh_page_bounds_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
}

int ofh_page_bounds(const ofh_page_bounds_params* p, const void* k_pages, void* bounds, void* stream) {
    return guarded([&]() -> int {
        if (p == nullptr) return invalid("params must be non-null");
        if (p->struct_size != sizeof(*p))
            return invalid("ofh_page_bounds_params.struct_size mismatch (call ofh_page_bounds_params_init)");
        if (p->tokens == 0) return invalid("cache dimensions must be non-zero");
        int64_t ks[3], bs[3];
        if (int rc = check_bounds(p->batch, p->kv_heads, p->head_dim, p->dtype, p->bounds_strides, bounds, true, bs)) return rc;
        if (p->tokens > (size_t)kMaxTokens) return unsupported("cache dimensions exceed the 32-bit index range");
        if (int rc = check_pages(p->num_pages, p->page_size, p->max_pages, p->table_stride, p->page_table, p->lengths, true))
            return rc;
        resolve_strides(ks, p->k_page_strides, p->kv_heads, p->page_size, p->head_dim);
        if (int rc = check_tensor({"k_pages", k_pages, ks, p->head_dim}, elem_size(p->dtype), true, 1)) return rc;
        ofh::PageBoundsArgs a{};
        a.k_pages = k_pages;
        a.bounds = bounds;
        a.k_sp = ks[0]; a.k_sh = ks[1]; a.k_st = ks[2];
        a.b_sp = bs[0]; a.b_sh = bs[1]; a.b_st = bs[2];
        a.table = p->page_table;
        a.table_stride = p->table_stride != 0 ? p->table_stride : (int64_t)p->max_pages;
        a.num_pages = (int)p->num_pages;
        a.page_shift = log2_of(p->page_size);
        a.max_pages = (int)p->max_pages;
        a.lengths = p->lengths;
        a.counts = p->counts;
        a.B = (int)p->batch;
        a.Hkv = (int)p->kv_heads;
        a.T = (int)p->tokens;
        a.D = (int)p->head_dim;
        // a page's last token, and what comes after it
        a.touched = (int)std::min<size_t>((p->tokens + p->page_size - 2) / p->page_size + 1, p->max_pages);
        if (!ofh::page_bounds_fits(a)) return unsupported("page bounds exceed the launch range");
        OFH_HIP_CHECK(ofh::launch_page_bounds(a, p->dtype, static_cast<hipStream_t>(stream)));
        return OFH_SUCCESS;
    });
}

void ofh_select_params_init(ofh_select_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
    p->query_tokens = 1;
}

int ofh_select_pages_workspace_bytes(const ofh_select_params* p, size_t* bytes) {
    return guarded([&]() -> int {
        if (bytes == nullptr) return invalid("bytes must be non-null");
        ofh::SelectArgs a;
        if (int rc = select_args(p, false, nullptr, nullptr, nullptr, a)) return rc;
        *bytes = select_bytes(a);
        return OFH_SUCCESS;
    });
}

int ofh_select_pages(const ofh_select_params* p, const void* q, const void* bounds, int32_t* selected, void* workspace,
                     size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        ofh::SelectArgs a;
        if (int rc = select_args(p, true, q, bounds, selected, a)) return rc;
        if (!ofh::page_select_fits(a, p->dtype)) return unsupported("selection exceeds the launch range");
        ofh::ScratchLease lease;
        if (int rc = take_workspace(select_bytes(a), workspace, workspace_bytes, static_cast<hipStream_t>(stream), lease))
            return rc;
        a.scores = static_cast<uint32_t*>(workspace);
        OFH_HIP_CHECK(ofh::launch_page_select(a, p->dtype, static_cast<hipStream_t>(stream)));
        return lease.release();
    });
}

void ofh_cache_write_params_init(ofh_cache_write_params* p) {
    if (p == nullptr) return;
    std::memset(p, 0, sizeof(*p));
    p->struct_size = sizeof(*p);
}

int ofh_cache_write(const ofh_cache_write_params* p, const void* k, const void* v, void* k_pages, void* v_pages,
                    void* stream) {
    return guarded([&]() -> int {
        ofh::CacheWriteArgs a;
        if (int rc = cache_write_args(p, k, v, k_pages, v_pages, a)) return rc;
        if (!ofh::cache_write_fits(a))
            return unsupported("cache write exceeds the launch range");
        OFH_HIP_CHECK(ofh::launch_cache_write(a, static_cast<hipStream_t>(stream)));
        return OFH_SUCCESS;
    });
}

int ofh_cache_copy_pages(void* const* pools, size_t num_pools, size_t num_pages, size_t page_bytes,
                         size_t page_stride_bytes, const int32_t* src, const int32_t* dst, size_t count,
                         void* stream) {
    return guarded([&]() -> int {
        if (num_pools == 0 || num_pages == 0 || page_bytes == 0) return invalid("pool dimensions must be non-zero");
        if (pools == nullptr || (count > 0 && (src == nullptr || dst == nullptr)))
            return invalid("pools, src and dst must be non-null");
        const size_t stride = page_stride_bytes != 0 ? page_stride_bytes : page_bytes;
        if (stride < page_bytes) return invalid("pages must not overlap");
        if (num_pages > (size_t)kMaxOffset || stride > ((size_t)1 << 34))
            return unsupported("pages exceed the index range");
        if (page_bytes % 2 != 0 || stride % 2 != 0) return unsupported("pages must be whole 2-byte elements");
        for (size_t i = 0; i < num_pools; ++i) {
            if (pools[i] == nullptr) return invalid("pools, src and dst must be non-null");
            if ((uintptr_t)pools[i] % 2 != 0) return unsupported("pools must be 2-byte aligned");
        }
        std::vector<uint8_t> role(count > 0 ? num_pages : 0, 0);  // 1: read, 2: written
        for (size_t i = 0; i < count; ++i) {
            if (src[i] < 0 || dst[i] < 0 || (size_t)src[i] >= num_pages || (size_t)dst[i] >= num_pages)
                return invalid("copied pages must be within the pool");
            role[(size_t)src[i]] |= 1;
        }
        for (size_t i = 0; i < count; ++i) {
            if (role[(size_t)dst[i]] & 2) return invalid("a page is copied to twice");
            role[(size_t)dst[i]] |= 2;
            if (role[(size_t)dst[i]] & 1) return invalid("a page is both copied from and copied to");
        }
        // A launch has at most 2^32 work items of which 2-byte chunks move 8
        // bytes each: fewer pairs and pools of pages past 16 MiB, one of both past 2 GiB.
        const bool wide = num_pages > ((size_t)1 << 16);
        const size_t most_pools = page_bytes > ((size_t)1 << 31) ? 1 : page_bytes > ((size_t)1 << 24) ? 8 : ofh::kCopyWords / 4;
        const size_t most_pairs = page_bytes > ((size_t)1 << 24) ? 1 : (size_t)1 << 31;
        for (size_t j = 0; j < num_pools; j += most_pools) {
            ofh::CopyPagesArgs a{};
            a.num_pools = (int)std::min(most_pools, num_pools - j);
            a.wide = wide ? 1 : 0;
            a.page_stride = (int64_t)stride;
            a.page_bytes = (int64_t)page_bytes;
            for (int t = 0; t < a.num_pools; ++t) {
                const uint64_t at = reinterpret_cast<uintptr_t>(pools[j + t]);
                a.words[2 * t] = (uint32_t)at;
                a.words[2 * t + 1] = (uint32_t)(at >> 32);
            }
            uint32_t* pairs = a.words + 2 * a.num_pools;
            // (a launch of small pages stays within 2^32 work items too)
            const size_t items = (page_bytes / 8 + 256) * (size_t)a.num_pools;
            const size_t fit = std::min(most_pairs, std::max<size_t>(1, (((size_t)1 << 32) - 1) / items));
            const size_t room = std::min(fit, (size_t)(ofh::kCopyWords - 2 * a.num_pools) / (wide ? 2 : 1));
            for (size_t i = 0; i < count; i += room) {
                a.num_pairs = (int)std::min(room, count - i);
                for (int t = 0; t < a.num_pairs; ++t) {
                    const uint32_t from = (uint32_t)src[i + t], to = (uint32_t)dst[i + t];
                    if (wide) {
                        pairs[2 * t] = from;
                        pairs[2 * t + 1] = to;
                    } else {
                        pairs[t] = from | to << 16;
                    }
                }
                OFH_HIP_CHECK(ofh::launch_copy_pages(a, static_cast<hipStream_t>(stream)));
            }
        }
        return OFH_SUCCESS;
    });
}

}  // extern "C"
