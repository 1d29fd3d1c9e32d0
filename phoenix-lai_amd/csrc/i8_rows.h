// An int8 row and its scale, as phx_quant_i8 defines them.
#pragma once
#include "device_common.h"

namespace phx {

// d = max |v| / 127, q = roundf(v * (1 / d)); a row whose d is under 2^-126 is zeros with d = 0, one that holds a NaN
// or an infinity zeros with d = NaN.  |v| compared as integers: a NaN or an infinity is then above every number.
struct RowScale { float d, inv; };
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits)
{
    if (amax_bits >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
    const float d = __uint_as_float(amax_bits) / 127.0f;
    if (!(d >= 1.17549435e-38f)) return {0.0f, 0.0f};
    return {d, 1.0f / d};
}
__device__ __forceinline__ int quant_one(float v, float inv)
{
    const float q = fminf(fmaxf(roundf(v * inv), -127.0f), 127.0f);
    return inv == 0.0f ? 0 : (int)q;
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d)
{
    return (uint32_t)(a & 0xFF) | ((uint32_t)(b & 0xFF) << 8) | ((uint32_t)(c & 0xFF) << 16) | ((uint32_t)d << 24);
}

}  // namespace phx
