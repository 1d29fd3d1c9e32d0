// Low-rank adapters of many requests at once (phx_lora_add): y[t] = y_in[t] + scale * B (A x[t]) with the adapter of slot ids[t].
//
// Two launches: k_lora_down forms A x in parts of the reduction, as floats, and k_lora_up joins the parts in order, scales them and adds
// B's products to the rows.  Both take tiles of 16 consecutive rows and, of a tile, one slot after another: the matrix
// cores form the slot's products with all 16 rows, and the rows of that slot keep theirs.  No sorting, no order that depends on
// timing; rows of one request that follow each other, as a prompt's do, cost one pass.
#include <algorithm>

#include "device_common.h"
#include "rows_io.h"

namespace phx {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <bool BF>
__device__ __forceinline__ f32x4 mma16(w4 a, w4 b, f32x4 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// The slots of 16 rows, one after another: mine is lane l's id (of row l % 16, -1 where it has none), left the rows not
// yet taken.  A slot's rows are taken together, those without one (slot -1) too.
struct TileSlots {
    int mine;
    unsigned left;
    __device__ __forceinline__ TileSlots(const int* ids, int n_slot, int T, int t0)
    {
        const int r = t0 + (int)(threadIdx.x & 15), id = ids[min(r, T - 1)];
        mine = (unsigned)id < (unsigned)n_slot ? id : -1;
        left = (1u << min(16, T - t0)) - 1;
    }
    // the next slot's number and rows; false when no row is left
    __device__ __forceinline__ bool next(int* slot, unsigned* rows)
    {
        if (!left) return false;
        *slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
        *rows = (unsigned)__ballot(mine == *slot) & left;
        left &= ~*rows;
        return true;
    }
};

// ------------------------------------------------------------------------------ slots
__global__ __launch_bounds__(256) void k_lora_set(LoraSlots L, int slot, int rank, const uint16_t* __restrict__ a,
                                                  const uint16_t* __restrict__ b, float scale)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, na = L.a_bytes() / 16;
    if (i == 0) {
        L.rank[slot] = rank;
        L.scale[slot] = scale;
    }
    uint16_t v[8];
    uint8_t* to;
    if (i < na) {
        const int r = (int)(i & 15), kc = (int)((i >> 4) % L.kc), rank0 = (int)((i >> 4) / L.kc) * 16 + r;
        for (int j = 0; j < 8; j++) v[j] = rank0 < rank && kc * 8 < L.cols ? a[(int64_t)rank0 * L.cols + kc * 8 + j] : 0;
        to = L.a + slot * L.a_bytes() + i * 16;
    } else if (i - na < L.b_bytes() / 16) {
        const int64_t k = i - na;
        const int t16 = (int)(k & 15), half = (int)(k >> 4) & 1, m = (int)(k >> 5) & 3, rt = (int)((k >> 7) % L.rt);
        const int64_t row = (k >> 7) / L.rt * 64 + 16 * (t16 >> 2) + 4 * m + (t16 & 3);
        for (int j = 0; j < 8; j++) {
            const int r = rt * 16 + half * 8 + j;
            v[j] = row < L.rows && r < rank ? b[row * rank + r] : 0;
        }
        to = L.b + slot * L.b_bytes() + k * 16;
    } else return;
    *(uint4*)to = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
}

void launch_lora_set(hipStream_t st, const LoraSlots& L, int slot, int rank, const uint16_t* a, const uint16_t* b, float scale)
{
    const int64_t n = (L.a_bytes() + L.b_bytes()) / 16;
    launch(k_lora_set, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, L, slot, rank, a, b, scale);
}

// ------------------------------------------------------------------------------ A x
// A workgroup takes 16 rows (x), every gridDim.y-th slot of theirs (y), and a rank tile of 16 by a part of the reduction (z), which its
// four waves split again; their sums meet in LDS, added in the waves' order.
constexpr int LD_WAVES = 4;
template <bool BF>
__global__ __launch_bounds__(64 * LD_WAVES) void k_lora_down(LoraSlots L, int T, const uint16_t* __restrict__ x,
                                                             const int* __restrict__ ids, int parts, float* __restrict__ part)
{
    __shared__ float red[LD_WAVES * 256];
    constexpr int U = 4;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = blockIdx.x * 16, p = blockIdx.z % parts, rt = blockIdx.z / parts;
    const int steps = L.kc / 4, n = parts * LD_WAVES, w = p * LD_WAVES + wave;
    const int s0 = (int)((int64_t)w * steps / n), s1 = (int)((int64_t)(w + 1) * steps / n);
    const uint16_t* xr = x + (int64_t)min(t0 + r16, T - 1) * L.cols;
    TileSlots S(ids, L.n_slot, T, t0);
    int slot;
    unsigned rows;
    for (int j = 0; S.next(&slot, &rows); j++) {
        if (j % gridDim.y != blockIdx.y || slot < 0 || L.rank[slot] <= rt * 16) continue;  // uniform over the workgroup
        const uint8_t* a = L.a + slot * L.a_bytes() + (int64_t)rt * L.kc * 256 + q * 256 + r16 * 16;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        w4 av[U], xv[U];
        auto load = [&](int u, int s) {
            const int su = min(s, s1 - 1);
            av[u] = *(const w4*)(a + (int64_t)su * 1024);
            xv[u] = *(const w4*)(xr + min(32 * su + 8 * q, L.cols - 8));
        };
        auto mma = [&](int u, int s) {
            if (32 * s + 32 > L.cols && 32 * s + 8 * q >= L.cols) xv[u] = w4{0, 0, 0, 0};  // against zero weights an infinity is none
            acc = mma16<BF>(xv[u], av[u], acc);
        };
        if (s0 < s1) {
#pragma unroll
            for (int u = 0; u < U; u++) load(u, s0 + u);
            int s = s0;
            for (; s + U < s1; s += U)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    mma(u, s + u);
                    load(u, s + u + U);
                }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (s + u < s1) mma(u, s + u);
        }
#pragma unroll
        for (int v = 0; v < 4; v++) red[wave * 256 + (4 * q + v) * 16 + r16] = acc[v];  // [row][rank]
        __syncthreads();
        const int row = tid >> 4;
        if (rows >> row & 1) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < LD_WAVES; i++) s += red[i * 256 + tid];
            part[((int64_t)p * T + t0 + row) * (16 * L.rt) + rt * 16 + (tid & 15)] = s;
        }
        __syncthreads();
    }
}

int lora_parts(const LoraSlots& L, int T, int ncu)
{
    const int tiles = (T + 15) / 16 * L.rt * std::min(L.n_slot, std::min(T, 16));
    return std::max(1, std::min(std::min(8, L.kc / 4 / (4 * LD_WAVES)), ncu / std::max(tiles, 1)));
}

// the slots of a tile side by side where the rows are few, else one after another
static int slots_apart(const LoraSlots& L, int T) { return T <= 256 ? std::min(L.n_slot + 1, std::min(T, 16)) : 1; }

void launch_lora_down(hipStream_t st, const LoraSlots& L, int T, const uint16_t* x, const int* ids, int parts, float* part)
{
    const dim3 grid((T + 15) / 16, slots_apart(L, T), L.rt * parts), blk(64 * LD_WAVES);
    if (L.type == PHX_BF16) launch(k_lora_down<true>, grid, blk, 0, st, L, T, x, ids, parts, part);
    else launch(k_lora_down<false>, grid, blk, 0, st, L, T, x, ids, parts, part);
}

// ------------------------------------------------------------------------------ y
// Eight floats as two terms of the adapters' type, hi + lo; an infinity or a NaN is in hi alone.
template <bool BF>
__device__ __forceinline__ uint32_t pair16(float a, float b) { return pair_of<BF ? PHX_BF16 : PHX_F16>(a, b); }
template <bool BF>
__device__ __forceinline__ float value16(uint32_t h) { return BF ? bf2f(h & 0xFFFF) : h2f(h & 0xFFFF); }
template <bool BF>
__device__ __forceinline__ w4 term(float (&v)[8])
{
    w4 t;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        t[j] = pair16<BF>(v[2 * j], v[2 * j + 1]);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float rest = v[2 * j + h] - value16<BF>(t[j] >> (16 * h));
            v[2 * j + h] = fabsf(rest) < 3.0e38f ? rest : 0.0f;
        }
    }
    return t;
}

// Four waves, each 64 outputs of 16 rows.  The matrix instruction's 32 columns are 16 ranks twice: lanes 0 - 31 bring the value's first
// term, lanes 32 - 63 its second, B's ranks the same for both; for float rows a second instruction takes a third and a fourth.
// A row's values are scaled by a power of two to below 2, so that neither term leaves the type's range, and its sums scaled
// back.  Weights are the first operand, so that a lane's sums are 16 consecutive outputs of one row.
template <int DT, bool BF>
__global__ __launch_bounds__(256) void k_lora_up(LoraSlots L, int T, const int* __restrict__ ids, int parts,
                                                 const float* __restrict__ part, int64_t ld, const void* y_in, void* y)
{
    constexpr int V = DT == PHX_F32 ? 4 : 8;  // values of 16 bytes
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
    const int grp = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (grp >= L.groups) return;
    const int t0 = blockIdx.x * 16, row = t0 + r16;
    const int64_t at = min(row, T - 1) * ld + grp * 64 + q * 16;
    const int cols = L.rows - grp * 64 - q * 16;  // this lane's outputs that there are
    const bool wide = ld % V == 0 && ((uintptr_t)y_in | (uintptr_t)y) % 16 == 0;
    TileSlots S(ids, L.n_slot, T, t0);
    int slot;
    unsigned rows;
    for (int j = 0; S.next(&slot, &rows); j++) {
        if (j % gridDim.z != blockIdx.z) continue;
        const int rank = slot < 0 ? 0 : L.rank[slot];
        if (rank == 0 && y_in == y) continue;
        float v[16];
        const bool here = rows >> r16 & 1;
        if (here) {
#pragma unroll
            for (int i = 0; i < 16; i += V) {
                if (wide && i + V <= cols) {
                    if constexpr (DT == PHX_F32) *(float4*)(v + i) = *(const float4*)((const float*)y_in + at + i);
                    else {
                        float e[8];
                        load_eight<DT>(y_in, at + i, e);
#pragma unroll
                        for (int k = 0; k < 8; k++) v[i + k] = e[k];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++) v[i + k] = i + k < cols ? load_one<DT>(y_in, at + i + k) : 0.0f;
                }
            }
        }
        if (rank > 0) {
            const int tiles = (rank + 15) / 16;
            const float scale = L.scale[slot];
            const float* s = part + (int64_t)min(row, T - 1) * (16 * L.rt) + 8 * (q & 1);
            auto values = [&](int rt, float (&c)[8]) {
#pragma unroll
                for (int k = 0; k < 8; k++) c[k] = 0.0f;
                if (here)
                    for (int p = 0; p < parts; p++) {
                        float e[8];
                        load_eight<PHX_F32>(s, (int64_t)p * T * (16 * L.rt) + rt * 16, e);
#pragma unroll
                        for (int k = 0; k < 8; k++) c[k] += e[k];
                    }
#pragma unroll
                for (int k = 0; k < 8; k++) c[k] = rt * 16 + 8 * (q & 1) + k < rank ? c[k] * scale : 0.0f;  // a NaN past the rank: 0 * infinity
            };
            // the row's largest exponent, over its ranks: lanes r16 and r16 + 16 hold the halves of a rank tile
            unsigned most = 0;
            for (int rt = 0; rt < tiles; rt++) {
                float c[8];
                values(rt, c);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const unsigned m = __float_as_uint(c[k]) & 0x7FFFFFFFu;
                    most = max(most, m >= 0x7F800000u ? 0u : m);
                }
            }
            most = max(most, (unsigned)__shfl_xor((int)most, 16));
            const int ex = most ? (int)(most >> 23) - 127 : 0;  // |values| < 2^(ex + 1)
            f32x4 acc[4];
#pragma unroll
            for (int m = 0; m < 4; m++) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const uint8_t* b = L.b + slot * L.b_bytes() + (int64_t)grp * L.rt * 2048 + (q & 1) * 256 + r16 * 16;
            for (int rt = 0; rt < tiles; rt++) {
                float c[8];
                values(rt, c);
#pragma unroll
                for (int k = 0; k < 8; k++) c[k] = __builtin_amdgcn_ldexpf(c[k], -ex);
                w4 bv[4];
#pragma unroll
                for (int m = 0; m < 4; m++) bv[m] = *(const w4*)(b + (int64_t)rt * 2048 + m * 512);
#pragma unroll
                for (int k = 0; k < (DT == PHX_F32 ? 2 : 1); k++) {
                    const w4 hi = term<BF>(c), lo = term<BF>(c);
                    w4 mine;
#pragma unroll
                    for (int i = 0; i < 4; i++) mine[i] = q < 2 ? hi[i] : lo[i];
#pragma unroll
                    for (int m = 0; m < 4; m++) acc[m] = mma16<BF>(bv[m], mine, acc[m]);
                }
            }
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[4 * m + i] += __builtin_amdgcn_ldexpf(acc[m][i], ex);
        }
        if (!here) continue;
#pragma unroll
        for (int i = 0; i < 16; i += V) {
            if (wide && i + V <= cols) {
                float e[V];
#pragma unroll
                for (int k = 0; k < V; k++) e[k] = v[i + k];
                store_16<DT>(y, at + i, e);
            } else {
#pragma unroll
                for (int k = 0; k < V; k++)
                    if (i + k < cols) store_one<DT>(y, at + i + k, v[i + k]);
            }
        }
    }
}

template <int DT>
static void lora_up(hipStream_t st, const LoraSlots& L, int T, const int* ids, int parts, const float* part, int64_t ld,
                    const void* y_in, void* y)
{
    const dim3 grid((T + 15) / 16, (L.groups + 3) / 4, slots_apart(L, T)), blk(256);
    if (L.type == PHX_BF16) launch(k_lora_up<DT, true>, grid, blk, 0, st, L, T, ids, parts, part, ld, y_in, y);
    else launch(k_lora_up<DT, false>, grid, blk, 0, st, L, T, ids, parts, part, ld, y_in, y);
}

void launch_lora_up(hipStream_t st, const LoraSlots& L, int T, const int* ids, int parts, const float* part, int y_type, int64_t ld,
                    const void* y_in, void* y)
{
    if (y_type == PHX_F16) lora_up<PHX_F16>(st, L, T, ids, parts, part, ld, y_in, y);
    else if (y_type == PHX_BF16) lora_up<PHX_BF16>(st, L, T, ids, parts, part, ld, y_in, y);
    else lora_up<PHX_F32>(st, L, T, ids, parts, part, ld, y_in, y);
}

}  // namespace phx
