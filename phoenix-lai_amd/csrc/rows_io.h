// Loads and stores of rows of float, fp16 or bf16 (PHX_F32, PHX_F16, PHX_BF16), the row types of the routing and int8
// entry points.
#pragma once
#include "device_common.h"

namespace phx {

__device__ __forceinline__ float bf2f(uint32_t h) { return __uint_as_float(h << 16); }

typedef float rf2 __attribute__((ext_vector_type(2)));
typedef __bf16 rbf2 __attribute__((ext_vector_type(2)));
// two floats as bf16 bits, to nearest even
__device__ __forceinline__ uint32_t f2bf_pair(float a, float b)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((rf2{a, b}), rbf2));
}
// A float as fp16 bits, to nearest even.  The value is a float first: left to itself the compiler may round a product straight
// to fp16, in one mixed instruction, in one kernel and not in another.
__device__ __forceinline__ uint32_t f2h_of(float v)
{
    asm("" : "+v"(v));
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ uint32_t pair_of(float a, float b)
{
    return DT == PHX_F16 ? f2h_of(a) | (f2h_of(b) << 16) : f2bf_pair(a, b);
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

template <int DT>
__device__ __forceinline__ void store_one(void* p, int64_t i, float v)
{
    if (DT == PHX_F32) ((float*)p)[i] = v;
    else ((uint16_t*)p)[i] = (uint16_t)(DT == PHX_F16 ? f2h_of(v) : f2bf_pair(v, 0.0f));
}

// 16 bytes of consecutive values (4 floats, 8 of the 16-bit types); p + i 16-byte aligned
template <int DT, int V>
__device__ __forceinline__ void store_16(void* p, int64_t i, const float (&v)[V])
{
    static_assert(V == (DT == PHX_F32 ? 4 : 8), "16 bytes");
    if constexpr (DT == PHX_F32) *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *(uint4*)((uint16_t*)p + i) = make_uint4(pair_of<DT>(v[0], v[1]), pair_of<DT>(v[2], v[3]), pair_of<DT>(v[4], v[5]),
                                                 pair_of<DT>(v[6], v[7]));
}

// four consecutive values; p + i aligned to four of them
template <int DT>
__device__ __forceinline__ void store_four(void* p, int64_t i, float4 v)
{
    if (DT == PHX_F32) *(float4*)((float*)p + i) = v;
    else *(uint2*)((uint16_t*)p + i) = make_uint2(pair_of<DT>(v.x, v.y), pair_of<DT>(v.z, v.w));
}

}  // namespace phx
