// What the kernels of products with fp16 and bf16 matrices share (kernels_half.hip, half_tile.h, kernels_lora.hip).
#pragma once
#include "device_common.h"
#include "rows_io.h"

namespace phx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));  // 16 bytes: eight values
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// v_mfma_f32_16x16x32: lane l holds eight values of A row l % 16 and of B row l % 16, both at k = 8 (l / 16); D[i][j] sits
// in lane j + 16 (i / 4), register i % 4.
template <bool BF>
__device__ __forceinline__ f32x4 mma16(w4 a, w4 b, f32x4 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// v_mfma_f32_32x32x16: lane l holds eight values of A row l % 32 and of B row l % 32, both at k = 8 (l / 32); D[i][j] sits in
// lane j + 32 ((i / 4) % 2), register 4 (i / 8) + i % 4.
template <bool BF>
__device__ __forceinline__ f32x16 mma32(w4 a, u32x4 b, f32x16 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// act(g) * u, both activations g * sigmoid(z), the exponential and the reciprocal the hardware's (1 ulp each): a few units of
// 2^-24, and the exponential's argument.  Far below, where the exponential is past every float and the quotient under 2^-120, the
// reciprocal is 0; the gate is then held to a number, so that no infinity meets it.
__device__ __forceinline__ float gated_half(int act, float g, float u)
{
    const float z = act == PHX_QUANT_SILU_MUL ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * z));
    return fmaxf(g, -3.402823466e38f) * r * u;
}

__device__ __forceinline__ void store_as(int type, void* p, int64_t i, float v)
{
    if (type == PHX_F32) store_one<PHX_F32>(p, i, v);
    else if (type == PHX_BF16) store_one<PHX_BF16>(p, i, v);
    else store_one<PHX_F16>(p, i, v);
}

// A value as the sum of N terms of a 16-bit type, each the rounding of what the ones before leave: 16 bits of it with two bf16 terms, 22
// with two of fp16, more than a float's with four; no finer than 2^-25, fp16's half step near zero.  An infinity or a NaN is in
// the first alone.
template <bool BF, int N>
__device__ __forceinline__ void split(float v, uint16_t (&t)[N])
{
#pragma unroll
    for (int i = 0; i < N; i++) {
        t[i] = (uint16_t)(BF ? f2bf_pair(v, 0.0f) : f2h_of(v));
        const float rest = v - (BF ? bf2f(t[i]) : h2f(t[i]));
        v = fabsf(rest) < 3.0e38f ? rest : 0.0f;
    }
}

// 16 bytes of weights; ONCE: no other workgroup reads them, so they need not stay in the caches
template <bool ONCE>
__device__ __forceinline__ w4 load_weights(const uint8_t* p)
{
    if constexpr (ONCE) return __builtin_nontemporal_load((const w4*)p);
    else return *(const w4*)p;
}

// The row of its group of 32 that is stored at slot s: what a lane holds of a 32 x 32 product, slots 8 g + 4 h + 0 .. 3 for
// half h, are then 16 consecutive rows.
__device__ __forceinline__ int slot_row(int s) { return 16 * ((s >> 2) & 1) + 4 * (s >> 3) + (s & 3); }

// ------------------------------------------------------------------------------ products
// The groups that the offsets give, each in tiles of up to cap places, four groups to a lane: every wave looks a tile up for itself.
// EVEN: a group's tiles are of one size, whole 32s (513 places as 192, 192 and 129 cost what 256, 256 and 1 do, and the longest
// tile is what a launch ends with).
template <bool EVEN>
struct Groups {
    int at[5], t[4], first, sum;  // the lane's groups' bounds and tiles, the tiles before them and in them
    __device__ __forceinline__ Groups(const HalfArgs& g)
    {
        // the offsets held to 0 .. n, and each to at least the one before it, so that no two groups share a place; past the last
        // group all are its end
        const int lane = threadIdx.x & 63;
        sum = 0;
#pragma unroll
        for (int i = 0; i < 5; i++) at[i] = min(max(g.offsets[min(4 * lane + i, g.n_mat)], 0), g.n);
#pragma unroll
        for (int i = 1; i < 5; i++) at[i] = max(at[i], at[i - 1]);
        int most = at[3];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int before = __shfl_up(most, d);
            most = lane >= d ? max(most, before) : most;
        }
        const int before = __shfl_up(most, 1);  // lane 0: its own
#pragma unroll
        for (int i = 0; i < 5; i++) at[i] = lane ? max(at[i], before) : at[i];
#pragma unroll
        for (int i = 0; i < 4; i++) sum += t[i] = (at[i + 1] - at[i] + g.cap - 1) / g.cap;
        first = wave_incl_scan_i(sum) - sum;
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(first + sum, 63); }
    // Item `item` of `per` items a tile, a group's tiles following each other for each of its items: the tile, which item, and whether the
    // group has no other tile.
    __device__ __forceinline__ bool find(const HalfArgs& g, int item, int per, Tile* tl, int* which, bool* alone) const
    {
        const unsigned long long here = __ballot(item >= first * per && item < (first + sum) * per);
        if (!here) return false;
        int e = 0, tile = 0, w = 0, f = first;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (item >= f * per && item < (f + t[i]) * per) {
                e = i;
                w = (item - f * per) / t[i];
                tile = (item - f * per) % t[i];
            }
            f += t[i];
        }
        const int l = __builtin_ctzll(here);
        int start = at[0], end = at[1], n = t[0];
#pragma unroll
        for (int i = 1; i < 4; i++)
            if (e == i) start = at[i], end = at[i + 1], n = t[i];
        tl->e = 4 * l + __builtin_amdgcn_readlane(e, l);
        start = __builtin_amdgcn_readlane(start, l);
        end = __builtin_amdgcn_readlane(end, l);
        n = __builtin_amdgcn_readlane(n, l);
        const int size = EVEN ? ((end - start + n - 1) / n + 31) & ~31 : g.cap;
        tl->start = start + __builtin_amdgcn_readlane(tile, l) * size;
        tl->cnt = min(end - tl->start, size);
        *which = __builtin_amdgcn_readlane(w, l);
        *alone = n == 1;
        return true;
    }
};

// The tile of a workgroup: cnt places of one group from start.  False where there is none.
__device__ __forceinline__ bool half_tile(const HalfArgs& g, int tile, Tile* tl)
{
    if (g.ids) {  // a tile per assignment, those without an expert empty
        *tl = {g.ids[tile], tile, 1};
        return (unsigned)tl->e < (unsigned)g.n_mat;
    }
    int one;
    bool alone;
    return Groups<false>(g).find(g, tile, 1, tl, &one, &alone);
}

// Place p's row of x, -1 where src has none.
__device__ __forceinline__ int x_row(const HalfArgs& g, int p)
{
    if (!g.src) return g.ids ? p / g.div : p;
    const int r = g.src[p];
    return (unsigned)r < (unsigned)(g.n_x * g.div) ? r / g.div : -1;
}

// Tile place i's output row, in bytes from out_base (a tile's own rows, or a whole output that dst points into, lie within 2^32
// bytes); NO_ROW where it has none.
constexpr uint32_t NO_ROW = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t out_row(const HalfArgs& g, const Tile& tl, int i)
{
    if (i >= tl.cnt || x_row(g, tl.start + i) < 0) return NO_ROW;
    return (uint32_t)(g.dst ? g.dst[tl.start + i] : i) * (uint32_t)g.out_cols * (g.type == PHX_F32 ? 4u : 2u * g.out_terms);
}
__device__ __forceinline__ char* out_base(const HalfArgs& g, const Tile& tl)
{
    return (char*)g.out + (g.dst ? 0 : (int64_t)tl.start * g.out_cols * (g.type == PHX_F32 ? 4 : 2 * g.out_terms));
}

}  // namespace phx
