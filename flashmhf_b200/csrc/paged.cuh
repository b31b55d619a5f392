// What the kernels of the paged 8-bit key/value cache share: codes and scales, and where a position lies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace fmhf {

// Codes for indices that only the device sees (DeviceCtl::index).
constexpr int kPagedAppendPage = 401, kPagedAppendPosition = 402, kPagedAppendRows = 403;
constexpr int kPagedAttnPage = 501, kPagedAttnLength = 502;
constexpr int kPromptRows = 551;

constexpr int kMinScaleExp = -60;   // the smallest scale, 2^-60: what a page of zeros has

__device__ __forceinline__ void note_index(int *index, int code) { atomicCAS(index, 0, code); }

// The smallest 2^n, n >= -60, with amax <= 448 * 2^n, by the bits of amax >= 0 (finite): 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
    int n = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    n = max(n, kMinScaleExp);
    return __uint_as_float((uint32_t)(n + 127) << 23);
}

// 1 / 2^n of a scale 2^n (n <= 120, the most that scale_for gives).
__device__ __forceinline__ float inverse_scale(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }

// Two codes of (a, b) * inv, rounded to nearest even.  Not ALL_FINITE: NaN and infinities become NaN (x - x is 0 for every finite x).
template <bool ALL_FINITE>
__device__ __forceinline__ uint32_t to_codes2(float a, float b, float inv) {
    const float2 v = ALL_FINITE ? make_float2(a * inv, b * inv) : make_float2(fmaf(a, inv, a - a), fmaf(b, inv, b - b));
    return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
}

// Four codes under another scale: their values times `ratio`, rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * i)), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        r |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3) << (16 * i);
    }
    return r;
}

}  // namespace fmhf
