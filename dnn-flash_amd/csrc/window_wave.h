// Device code of a wavefront of 32 rows that see a window and first tokens of keys
// staged through LDS (window_fwd.hip has the design), shared by the kernels whose
// rows stand in different places. Internal header, included by the HIP
// translation units.
#pragma once

#include "flash_wave32.h"
#include "serving_kernels.h"
#include "serving_softcap.h"

namespace ofh {
namespace {

// A workgroup of four wavefronts, KS of which share the keys of 32 rows, with
// keys in compute steps of BN and staged tiles of SN: two stages in at most 64
// KB, so that two workgroups share a CU and one's start, barriers and stores run
// beside the other's products (at D = 256 the registers hold one). Measured
// against eight wavefronts on tiles of 128 keys (us, one card): bf16 D128 B4
// H32/8 N2048 window 1024 140 / 151, B2 N4096 window 128 72 / 84, B1 H32 N4096
// without one 148 / 155, N16384 window 4096 983 / 949.
template <int D, int KS>
struct WindowTiles {
    static constexpr int THREADS = 256, WAVES = THREADS / 64;
    static constexpr int R = WAVES / KS;  // row slices of a workgroup
    static constexpr int BN = D == 256 || KS == 2 ? 32 : 64;
    static constexpr int SN = D == 64 && KS == 1 ? 128 : 64;
    static constexpr int SB = SN / BN;  // compute steps of a staged tile, shared by the KS groups
    static constexpr int WAVES_PER_SIMD = D <= 128 ? 2 : 1;
    static_assert(SB % KS == 0, "the groups share a tile's steps");
};

// What happens to a score: the scale alone; ALiBi, a soft-cap of at most kCapExp, or
// both; a wider cap, with or without ALiBi (in one kernel the two forms of the cap
// held more registers: f16 H32 N4096 D64 cap 50 186 us, with a kernel each 182).
enum WindowScores { kScoresPlain, kScoresMod, kScoresWideCap };

template <bool B>
struct Bool {
    static constexpr bool value = B;
};

template <typename T, int D, int KS, typename Tiles_ = WindowTiles<D, KS>>
struct WindowWave : Wave32<T, D, MOD_PLAIN, false, Tiles_::THREADS, Tiles_::BN, Tiles_::SB> {
    using Tiles = Tiles_;
    using Base = Wave32<T, D, MOD_PLAIN, false, Tiles::THREADS, Tiles::BN, Tiles::SB>;
    using typename Base::L;
    using typename Base::M16;
    using typename Base::v8;
    using Base::a;
    using Base::g;
    using Base::l_run;
    using Base::m_run;
    using Base::o;
    using Base::pf;
    using Base::s;
    using Base::smem;
    static constexpr int BN = Tiles::BN;

    // This lane's row sees keys below hi that are at or past lo or below the sinks.
    int hi, lo, sinks, pos;
    float slope;
    int hi_min, hi_max, lo_min, lo_max;  // over the wavefront's rows

    __device__ __forceinline__ WindowWave(const FwdArgs& args, const WindowArgs& wa, unsigned char* sm, int b, int h,
                                          int q0, int wv)
        : Base(args, sm, b * args.H + h, q0, wv) {
        this->Kp = (const T*)a.k + b * a.k_sb + h / wa.G * a.k_sh;
        this->Vp = (const T*)a.v + b * a.v_sb + h / wa.G * a.v_sh;
        sinks = wa.sinks;
        slope = a.alibi != nullptr ? a.alibi[h] : 0.0f;
        pos = this->my_q + wa.query_offset;
        limits(wa, this->my_q, hi, lo);
        const int first = this->qw0, last = min(first + kQueriesPerWave, a.M) - 1;
        int h0, h1;
        limits(wa, first, h0, lo_min);
        limits(wa, last, h1, lo_max);
        hi_min = min(h0, h1);
        hi_max = max(h0, h1);  // (a padding row's is 0: the rows before it see all keys)
        if (h1 < h0) hi_max = a.N;
        if (first >= a.M) hi_max = 0;
    }
    // Rows, keys and limits are set by the class that derives from this.
    __device__ __forceinline__ WindowWave(const FwdArgs& args, unsigned char* sm, int wv) : Base(args, sm, 0, 0, wv) {}
    __device__ __forceinline__ void limits(const WindowArgs& wa, int row, int& h, int& w) const {
        const int p = row + wa.query_offset;
        h = min(a.N, p + 1);
        if (wa.lengths != nullptr && p >= a.N) h = 0;  // padding
        w = wa.window > 0 ? p + 1 - wa.window : 0;
    }

    // K columns of a staged tile past the head dim -> 0: the copies repeat the row's
    // last chunk there, and an infinity in it times Q's zeros would be a NaN.
    __device__ __forceinline__ void zero_pad(int stage) {
        const int lane = threadIdx.x & 63, pos = (64 * this->wave + lane) % L::CPR;
        if (8 * (pos ^ L::kswz(this->dma_row0)) < a.D) return;
        constexpr int NW = Tiles::THREADS / 64;
#pragma unroll
        for (int u = 0; u < Base::CPT; ++u)
            *(u32x4*)(smem + stage + 1024 * (this->wave + NW * u) + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
    }

    __device__ __forceinline__ bool sees(int k0) const { return k0 < hi_max && (k0 + BN > lo_min || k0 < sinks); }
    __device__ __forceinline__ bool partly(int k0) const {
        return k0 + BN > hi_min || (k0 < lo_max && k0 + BN > sinks);
    }
    __device__ __forceinline__ bool seen(int key) const { return key < hi && (key >= lo || key < sinks); }

    // Online softmax of the scores in s (keys k0 ..): as Wave32::softmax. Bit i of
    // `missing`: the i-th 16 keys count for nothing (with mask).
    template <WindowScores SCORES>
    __device__ __forceinline__ void softmax_window(int k0, bool mask, unsigned missing = 0) {
        constexpr bool GENERAL = SCORES != kScoresPlain;
        float mx = kNegInf;
        const bool raw = !GENERAL && !mask && a.scale_log2 >= 0.0f;  // s holds dot products
        // At D = 64 the softmax's arithmetic bounds a step: p is taken against the
        // running max first. A row sum of at most 2^kRescaleSlack proves that the
        // tile's max would have raised nothing; else the tile is redone with it.
        if (D <= 64 && raw && __builtin_amdgcn_ballot_w64(m_run == kNegInf) == 0) {
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < BN / 16; ++c) {
#pragma unroll
                for (int t = 0; t < 8; ++t)
                    pf[c][t] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[c >> 1][8 * (c & 1) + t], a.scale_log2, -m_run));
#pragma unroll
                for (int t = 0; t < 8; t += 2) sum = Dot2<T>::sum2(typename Dot2<T>::v2{pf[c][t], pf[c][t + 1]}, sum);
            }
            if (__builtin_amdgcn_ballot_w64(!(sum <= kSumBound)) == 0) {
                l_run += sum;
                return;
            }
        }
        if (raw) {
#pragma unroll
            for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[sb][e]);
            mx *= a.scale_log2;
        } else {
            if (GENERAL) {
                const bool cap = SCORES == kScoresMod && a.softcap > 0.0f;
                const float c = cap ? 2.0f * kLog2e * a.inv_softcap : kLog2e;
                const float sl = slope * c, base = sl * (float)(k0 + 8 * g - pos), c_s = a.scale * c;
                const float cap_hi = a.softcap * kLog2e;
#pragma unroll
                for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float u = __builtin_fmaf(s[sb][e], c_s, __builtin_fmaf(sl, (float)tile_pos(sb, e), base));
                        // cap tanh(y / cap) = cap - 2 cap / (2^u + 1)
                        if (cap)
                            u = __builtin_fmaf(-2.0f * cap_hi, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u) + 1.0f),
                                               cap_hi);
                        s[sb][e] = u;
                    }
                if (SCORES == kScoresWideCap) {
                    const float cap_log2 = a.softcap * kLog2e;
#pragma unroll
                    for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[sb][e] = cap_tanh_wide(s[sb][e], cap_log2);
                }
            } else {
#pragma unroll
                for (int sb = 0; sb < BN / 32; ++sb) s[sb] *= a.scale_log2;
            }
            // relative to the lane's first key, so that positions are constants
            if (k0 + BN > hi_min) {
                const int h = hi - k0 - 8 * g;
#pragma unroll
                for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (tile_pos(sb, e) >= h) s[sb][e] = kNegInf;
            }
            if (k0 < lo_max && k0 + BN > sinks) {
                // (a tile that holds the last sink: its keys past the sinks, unless the window has them)
                const int w = lo - k0 - 8 * g, f = sinks - k0 - 8 * g;
                if (k0 >= sinks) {
#pragma unroll
                    for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (tile_pos(sb, e) < w) s[sb][e] = kNegInf;
                } else {
#pragma unroll
                    for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (tile_pos(sb, e) < w && tile_pos(sb, e) >= f) s[sb][e] = kNegInf;
                }
            }
            if (missing != 0) {
#pragma unroll
                for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (missing >> (2 * sb + (e >> 3)) & 1) s[sb][e] = kNegInf;
            }
#pragma unroll
            for (int sb = 0; sb < BN / 32; ++sb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[sb][e]);
        }
        mx = half_swap_max(mx);
        const bool raise = mx > m_run + kRescaleSlack;
        if (__builtin_amdgcn_ballot_w64(raise) != 0) {
            const float alpha = raise ? __builtin_amdgcn_exp2f(m_run - mx) : 1.0f;
            m_run = raise ? mx : m_run;
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < D / 32; ++db) o[db] *= alpha;
        }
        const float m_use = m_run == kNegInf ? 0.0f : m_run;
        const float to_log2 = raw ? a.scale_log2 : 1.0f;
#pragma unroll
        for (int c = 0; c < BN / 16; ++c)
#pragma unroll
            for (int t = 0; t < 8; ++t)
                pf[c][t] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[c >> 1][8 * (c & 1) + t], to_log2, -m_use));
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < BN / 16; ++c)
#pragma unroll
            for (int t = 0; t < 8; t += 2) sum = Dot2<T>::sum2(typename Dot2<T>::v2{pf[c][t], pf[c][t + 1]}, sum);
        l_run += sum;
    }

    // O += P V key by key, for the rows that see the key.
    __device__ __forceinline__ void pv_seen(int stage, int sub, int k0) {
        const lds_u8* vbs = (const lds_u8*)smem + stage + L::KTILE + sub * BN * L::VSTR;
        const int lane = threadIdx.x & 63;
#pragma nounroll
        for (int key = 0; key < BN; ++key) {
            // probability of (row, key): lane half (key / 8) % 2, pf[key / 16][key % 8]
            unsigned p2 = 0;
#pragma unroll
            for (int c = 0; c < BN / 16; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    if (key >> 4 == c && (key & 7) >> 1 == w) p2 = __builtin_bit_cast(u32x4, pf[c])[w];
            p2 = __shfl(p2, (lane & 31) + 32 * ((key >> 3) & 1));
            const unsigned short bits = (unsigned short)(key & 1 ? p2 >> 16 : p2);
            const float p = (float)__builtin_bit_cast(T, bits);
            const bool ok = seen(k0 + key);
            const int row = sub * BN + key;  // (the swizzle goes by the row of the staged tile)
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const v8 v = __builtin_bit_cast(
                        v8, *(const lds_u32x4*)(vbs + key * L::VSTR + 16 * ((4 * db + 2 * cc + g) ^ L::vswz(row))));
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        o[db][8 * cc + t] = ok ? __builtin_fmaf(p, (float)v[t], o[db][8 * cc + t]) : o[db][8 * cc + t];
                }
        }
    }

    __device__ __forceinline__ void restart() {
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
        m_run = kNegInf;
        l_run = 0.0f;
    }

    // A NaN in O: of a V that the row sees, or of one that it does not.
    __device__ __forceinline__ bool nan_in_o() const {
        bool bad = false;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) bad = bad || o[db][e] != o[db][e];
        return bad;
    }

    // SEEN: partly masked tiles are added key by key.
    template <WindowScores SCORES, bool SEEN>
    __device__ __forceinline__ void step(int stage, int sub, int k0) {
        const bool mask = partly(k0);
        __builtin_amdgcn_s_setprio(1);
        this->qk(stage, sub);
        __builtin_amdgcn_s_setprio(0);
        softmax_window<SCORES>(k0, mask);
        if (SEEN && mask) {
            pv_seen(stage, sub, k0);
            return;
        }
        __builtin_amdgcn_s_setprio(1);
        this->pv(stage, sub);
        __builtin_amdgcn_s_setprio(0);
    }
};

}  // namespace
}  // namespace ofh
