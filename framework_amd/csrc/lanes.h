// Sums and maxima over neighbouring lanes of a wavefront without LDS: the exchanges are DPP moves inside rows of 16
// lanes and row swaps between them, so a reduction over W lanes costs log2(W) vector instructions and no latency of the
// LDS pipe.  Every lane of a group ends with the same bits (both partners of a step add the same two values).
#pragma once
#include <hip/hip_runtime.h>

namespace mni {

template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {  // all lanes active, no bound control needed
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// The values of the lanes 16 (32) apart, as (the lower half's, the upper half's) in every lane.
__device__ __forceinline__ void swap16(float v, float &lo, float &hi) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap32(float v, float &lo, float &hi) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lo = __uint_as_float(r[0]);
    hi = __uint_as_float(r[1]);
}
// Sum over aligned groups of W lanes (W a power of two up to 64).
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
    if (W >= 2) v += lane_move<0xB1>(v);    // lane ^ 1
    if (W >= 4) v += lane_move<0x4E>(v);    // lane ^ 2
    if (W >= 8) v += lane_move<0x141>(v);   // mirrored in eight lanes: the other quad
    if (W >= 16) v += lane_move<0x140>(v);  // mirrored in sixteen lanes: the other eight
    float a, b;
    if (W >= 32) { swap16(v, a, b); v = a + b; }
    if (W >= 64) { swap32(v, a, b); v = a + b; }
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
    if (W >= 2) v = fmaxf(v, lane_move<0xB1>(v));
    if (W >= 4) v = fmaxf(v, lane_move<0x4E>(v));
    if (W >= 8) v = fmaxf(v, lane_move<0x141>(v));
    if (W >= 16) v = fmaxf(v, lane_move<0x140>(v));
    float a, b;
    if (W >= 32) { swap16(v, a, b); v = fmaxf(a, b); }
    if (W >= 64) { swap32(v, a, b); v = fmaxf(a, b); }
    return v;
}
// The same of the bits of floats that are not negative, which order as the floats do, infinity above them and every NaN
// above infinity: a maximum that a NaN does not drop out of.
template <int CTRL>
__device__ __forceinline__ uint32_t bits_move(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
template <int W>
__device__ __forceinline__ uint32_t lanes_max_bits(uint32_t v) {
    if (W >= 2) v = max(v, bits_move<0xB1>(v));
    if (W >= 4) v = max(v, bits_move<0x4E>(v));
    if (W >= 8) v = max(v, bits_move<0x141>(v));
    if (W >= 16) v = max(v, bits_move<0x140>(v));
    if (W >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(r[0], r[1]);
    }
    if (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(r[0], r[1]);
    }
    return v;
}

}  // namespace mni
