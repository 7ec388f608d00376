// The tanh soft-cap of the serving kernels. Internal header: not installed.
#pragma once

#include "flash_wave32.h"

namespace ofh {

// cap tanh(y / cap). Through the exponential, cap (1 - 2 / (2^u + 1)) with u =
// 2 log2(e) y / cap, its error is at most 8 2^-24 cap however small y is. In 16
// bits that is less than a quarter of what rounding P costs (fp16 2^-11) up to
// kCapExp, 256; past it, and in fp32, a score keeps its own precision through
// Lambert's continued fraction up to |y| = cap, cut where it is right to 2^-37:
// y (135135 + 17325 z^2 + 378 z^4 + z^6) / (135135 + 62370 z^2 + 3150 z^4 + 28 z^6),
// z = y / cap. (Past |y| = cap the exponential's error is a few 2^-24 of the score.)
// Off 64 bits, relative, rms: fp32 B2 H8 N1000 D64 cap 30 1.2e-6 through the
// exponential, 2.8e-7 so. Through the exponential a cap of 1e6 puts scores off by
// 0.1, and one of 1e9 makes them all 0. The fraction costs prompts more: f16 H32 N4096
// D64 310 us, 183 with a cap of 50; a decode step 1 us of 48.
constexpr float kCapExp = 256.0f;

__device__ __forceinline__ float cap_tanh16(float y, float cap) {
    const float u = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e / cap));
    return __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(u + 1.0f), cap);
}
__device__ __forceinline__ float lambert_num(float w) {
    return __builtin_fmaf(__builtin_fmaf(w + 378.0f, w, 17325.0f), w, 135135.0f);
}
__device__ __forceinline__ float lambert_den(float w) {
    return __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(28.0f, w, 3150.0f), w, 62370.0f), w, 135135.0f);
}
__device__ __forceinline__ float cap_tanh(float y, float cap) {
    const float z = y / cap, w = z * z;
    const float num = y * lambert_num(w), den = lambert_den(w);
    return __builtin_fabsf(z) <= 1.0f ? num / den : cap_tanh16(y, cap);
}
// In 16 bits with a cap past kCapExp: reciprocals of 1 ulp in place of divisions.
__device__ __forceinline__ float cap_tanh_wide(float y, float cap) {
    const float z = y * __builtin_amdgcn_rcpf(cap), w = z * z;
    return __builtin_fabsf(z) <= 1.0f ? y * lambert_num(w) * __builtin_amdgcn_rcpf(lambert_den(w)) : cap_tanh16(y, cap);
}

}  // namespace ofh
