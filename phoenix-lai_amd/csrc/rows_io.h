// Loads and stores of rows of float, fp16 or bf16 (PHX_F32, PHX_F16, PHX_BF16), the row types of the routing and int8
// entry points.
#pragma once
#include "device_common.h"

namespace phx {

__device__ __forceinline__ float bf2f(uint32_t h) { return __uint_as_float(h << 16); }

// float -> bf16 bits, round to nearest even; a NaN keeps a set fraction bit
__device__ __forceinline__ uint32_t f2bf(float v)
{
    const uint32_t b = __float_as_uint(v);
    return v != v ? (b >> 16) | 0x40u : (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}

template <int DT>
__device__ __forceinline__ float load_one(const void* p, int64_t i)
{
    if (DT == PHX_F32) return ((const float*)p)[i];
    const uint32_t h = ((const uint16_t*)p)[i];
    return DT == PHX_F16 ? h2f(h) : bf2f(h);
}

// eight consecutive values; p + i 16-byte aligned
template <int DT>
__device__ __forceinline__ void load_eight(const void* p, int64_t i, float (&v)[8])
{
    if (DT == PHX_F32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 h = *(const uint4*)((const uint16_t*)p + i);
        const uint32_t u[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = DT == PHX_F16 ? h2f(u[j] & 0xFFFF) : bf2f(u[j] & 0xFFFF);
            v[2 * j + 1] = DT == PHX_F16 ? h2f(u[j] >> 16) : __uint_as_float(u[j] & 0xFFFF0000u);
        }
    }
}

// A product that is stored as fp16 is rounded to float first: left to itself the compiler may round it once, in one mixed
// instruction, in one kernel and not in another.
__device__ __forceinline__ uint32_t f2h_of(float v)
{
    asm("" : "+v"(v));
    return f2h_bits(v);
}

template <int DT>
__device__ __forceinline__ void store_one(void* p, int64_t i, float v)
{
    if (DT == PHX_F32) ((float*)p)[i] = v;
    else ((uint16_t*)p)[i] = (uint16_t)(DT == PHX_F16 ? f2h_of(v) : f2bf(v));
}

// four consecutive values; p + i aligned to four of them
template <int DT>
__device__ __forceinline__ void store_four(void* p, int64_t i, float4 v)
{
    if (DT == PHX_F32) *(float4*)((float*)p + i) = v;
    else if (DT == PHX_F16)
        *(uint2*)((uint16_t*)p + i) = make_uint2(f2h_of(v.x) | (f2h_of(v.y) << 16), f2h_of(v.z) | (f2h_of(v.w) << 16));
    else *(uint2*)((uint16_t*)p + i) = make_uint2(f2bf(v.x) | (f2bf(v.y) << 16), f2bf(v.z) | (f2bf(v.w) << 16));
}

}  // namespace phx
