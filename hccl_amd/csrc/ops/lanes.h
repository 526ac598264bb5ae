// What the operators' kernels share: reductions over a wavefront, 16-byte accesses, the e4m3 conversions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kernels/elem.h"

namespace hcclx {

constexpr float kE4m3Most = 448.0f;   // the largest finite e4m3 value

// v of the lane that DPP control CTRL names; lanes without one get `none`.
template <int CTRL>
__device__ __forceinline__ float dpp_or(float none, float v)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(none), __float_as_uint(v), CTRL, 0xf, 0xf, false));
}

// Sum and maximum over the 64 lanes, the same in all of them: four steps inside rows of 16 lanes, two across rows, all in
// registers (no LDS round trip), then the last lane's value as a scalar.  The order of the additions is fixed.
__device__ __forceinline__ float wave_sum(float v)
{
    v += dpp_or<0x111>(0.0f, v);   // row_shr 1
    v += dpp_or<0x112>(0.0f, v);
    v += dpp_or<0x114>(0.0f, v);
    v += dpp_or<0x118>(0.0f, v);
    v += dpp_or<0x142>(0.0f, v);   // row_bcast 15
    v += dpp_or<0x143>(0.0f, v);   // row_bcast 31
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
// Of magnitudes (0 is the least); a NaN loses against any number.
__device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v, dpp_or<0x111>(0.0f, v));
    v = fmaxf(v, dpp_or<0x112>(0.0f, v));
    v = fmaxf(v, dpp_or<0x114>(0.0f, v));
    v = fmaxf(v, dpp_or<0x118>(0.0f, v));
    v = fmaxf(v, dpp_or<0x142>(0.0f, v));
    v = fmaxf(v, dpp_or<0x143>(0.0f, v));
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// How a magnitude becomes a scale and its block's codes: code = (x * up) * inverse.  up keeps the inverse of tiny scales finite.
struct CodeScale {
    float scale;
    float up;
    float inverse;
    __device__ __forceinline__ explicit CodeScale(float most)
    {
        scale = most / kE4m3Most;
        up = scale < 0x1p-100f ? 0x1p64f : 1.0f;
        inverse = scale > 0.0f ? 1.0f / (scale * up) : 0.0f;
    }
    __device__ __forceinline__ float operator()(float x) const { return (x * up) * inverse; }
};

// Four codes, rounded to nearest even.  The hardware makes NaN of what is nearer to 480 than to 448: magnitudes that the
// scale brought to 448 are off by a rounding or two and stay 448.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d)
{
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void from_e4m3(uint32_t codes, float (&out)[4])
{
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), true);
    out[0] = lo.x;
    out[1] = lo.y;
    out[2] = hi.x;
    out[3] = hi.y;
}

}  // namespace hcclx
