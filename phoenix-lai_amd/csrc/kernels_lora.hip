// Low-rank adapters of many requests at once (phx_lora_add): y[t] = y_in[t] + scale * B (A x[t]) with the adapter of slot ids[t].
//
// Two launches: k_lora_down forms A x as floats, scales it and writes it down as terms of the adapters' type, the second
// product's operands; k_lora_up adds B's products to the rows.  Both take tiles of 16 consecutive rows and, of a tile, one slot after
// another: the matrix cores form the slot's products with all 16 rows, and the rows of that slot keep theirs.  No sorting, no order
// that depends on timing; rows of one request that follow each other, as a prompt's do, cost one pass.
#include <algorithm>

#include "half_common.h"

namespace phx {

// The slots of 16 rows, one after another: mine is lane l's id (of row l % 16, -1 where it has none), left the rows not
// yet taken.  A slot's rows are taken together, those without one (slot -1) too.
struct TileSlots {
    int mine;
    unsigned left;
    __device__ __forceinline__ void load(const int* ids, int n_slot, int T, int t0)
    {
        const int r = t0 + (int)(threadIdx.x & 15), id = ids[min(r, T - 1)];
        mine = (unsigned)id < (unsigned)n_slot ? id : -1;
        left = t0 < T ? (1u << min(16, T - t0)) - 1 : 0;
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
    // row r's slot alone, if r is the first of its rows; else nothing
    __device__ __forceinline__ void only(int r)
    {
        const unsigned rows = (unsigned)__ballot(mine == __builtin_amdgcn_readlane(mine, r)) & left;
        left = rows && __builtin_ctz(rows) == r ? rows : 0;
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
// A workgroup takes 16 rows (x) and RT rank tiles of 16 (z), FEW: for the slot of row y of them alone; its NW waves split the
// reduction, all of a wave's loads in flight at once for rows of up to NW U steps, and their sums meet in LDS, added in the waves'
// order.  low [T][rt][TERMS][16 ranks]; fp16's terms are of the value over 2^exps
// [T][rt], which brings the largest of a row's 16 to 2^14 or more and below 2^15: none leaves the type's range, and the half step near
// zero is 2^-39 of that largest, so that values to 2^-17 of it keep their 22 bits.  One row of 4096, rank 16: 4.9 us, a launch and two
// dependent trips to memory; 4096 rows, rank 32: 17.4, the rows' 34 MB in 6 and the trips of a workgroup a compute unit behind each other.
template <int NW, int RT, int TERMS, bool FEW, bool BF>
__global__ __launch_bounds__(64 * NW) void k_lora_down(LoraSlots L, int T, const uint16_t* __restrict__ x,
                                                       const int* __restrict__ ids, uint16_t* __restrict__ low,
                                                       int* __restrict__ exps)
{
    __shared__ float red[NW * RT * 256];
    constexpr int U = RT <= 2 ? 8 : 4;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = blockIdx.x * 16, rt0 = blockIdx.z * RT;
    const int steps = L.kc / 4, s0 = wave * steps / NW, s1 = (wave + 1) * steps / NW;
    const uint16_t* xr = x + (int64_t)min(t0 + r16, T - 1) * L.cols;
    TileSlots S;
    S.load(ids, L.n_slot, T, t0);
    if (FEW) S.only(blockIdx.y);
    int slot;
    unsigned rows;
    while (S.next(&slot, &rows)) {
        if (slot < 0) continue;  // uniform over the workgroup
        const bool here = rows >> r16 & 1;
        const int rank = L.rank[slot];
        if (rank <= rt0 * 16) continue;
        const float scale = L.scale[slot];
        const uint8_t* a[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) a[r] = L.a + slot * L.a_bytes() + (int64_t)min(rt0 + r, L.rt - 1) * L.kc * 256 + q * 256 + r16 * 16;
        f32x4 acc[RT];
        w4 av[U][RT], xv[U];
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        auto load = [&](int u, int s) {
            const int su = min(s, s1 - 1);
#pragma unroll
            for (int r = 0; r < RT; r++) av[u][r] = *(const w4*)(a[r] + (int64_t)su * 1024);
            xv[u] = w4{0, 0, 0, 0};
            if (here) xv[u] = *(const w4*)(xr + min(32 * su + 8 * q, L.cols - 8));
        };
        auto mma = [&](int u, int s) {
            if (32 * s + 32 > L.cols && 32 * s + 8 * q >= L.cols) xv[u] = w4{0, 0, 0, 0};  // against zero weights an infinity is none
#pragma unroll
            for (int r = 0; r < RT; r++) acc[r] = mma16<BF>(xv[u], av[u][r], acc[r]);
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
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int v = 0; v < 4; v++) red[(wave * RT + r) * 256 + (4 * q + v) * 16 + r16] = acc[r][v];  // [row][rank]
        __syncthreads();
        const int row = (tid >> 4) & 15, i = tid & 15;
#pragma unroll
        for (int r = 0; r < RT; r++) {
            if (tid >= 256 || rt0 + r >= L.rt) continue;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) s += red[(w * RT + r) * 256 + (tid & 255)];
            s = (rt0 + r) * 16 + i < rank ? s * scale : 0.0f;  // past the rank A's zeros may have met an infinity
            const int64_t at = (int64_t)(t0 + row) * L.rt + rt0 + r;
            int ex = 0;
            if (!BF) {
                unsigned m = __float_as_uint(s) & 0x7FFFFFFFu;
                m = m >= 0x7F800000u ? 0u : m;
#pragma unroll
                for (int d = 1; d < 16; d *= 2) m = max(m, (unsigned)__shfl_xor((int)m, d));
                ex = m ? (int)(m >> 23) - 127 - 14 : 0;  // |values| < 2^(ex + 15)
                s = __builtin_amdgcn_ldexpf(s, -ex);
            }
            if (rows >> row & 1) {
                uint16_t t[TERMS];
                split<BF, TERMS>(s, t);
#pragma unroll
                for (int k = 0; k < TERMS; k++) low[(at * TERMS + k) * 16 + i] = t[k];
                if (!BF && i == 0) exps[at] = ex;
            }
        }
        __syncthreads();
    }
}

// The slots of a tile side by side where the rows are few, else one after another with weights held and more rows in flight (us, side
// by side and one after another; 4096 x 4096, eight adapters of rank 16, rows of one request in runs of 100: T = 512 13.7, 17.2; 1024
// 19.4, 18.4; each row another request than the last: 512 20, 44; 1000 30, 45; 2000 53, 50; rank 128: 500 94, 105; 1000 140, 114).
static bool few_rows(const LoraSlots& L, int T) { return T <= (L.rt <= 2 ? 1024 : 512); }

template <int NW, int RT, bool FEW, bool BF>
static void lora_down(hipStream_t st, const LoraSlots& L, int T, const uint16_t* x, const int* ids, int terms, uint16_t* low, int* exps)
{
    const dim3 grid((T + 15) / 16, FEW ? std::min(T, 16) : 1, (L.rt + RT - 1) / RT), blk(64 * NW);
    if (terms == 2) launch(k_lora_down<NW, RT, 2, FEW, BF>, grid, blk, 0, st, L, T, x, ids, low, exps);
    else launch(k_lora_down<NW, RT, 4, FEW, BF>, grid, blk, 0, st, L, T, x, ids, low, exps);
}

template <bool BF>
static void lora_down_type(hipStream_t st, const LoraSlots& L, int T, const uint16_t* x, const int* ids, int terms, uint16_t* low,
                           int* exps)
{
    if (few_rows(L, T)) lora_down<16, 1, true, BF>(st, L, T, x, ids, terms, low, exps);
    else if (L.rt == 1) lora_down<8, 1, false, BF>(st, L, T, x, ids, terms, low, exps);
    else lora_down<8, 2, false, BF>(st, L, T, x, ids, terms, low, exps);
}

void launch_lora_down(hipStream_t st, const LoraSlots& L, int T, const uint16_t* x, const int* ids, int terms, uint16_t* low, int* exps)
{
    if (L.type == PHX_BF16) lora_down_type<true>(st, L, T, x, ids, terms, low, exps);
    else lora_down_type<false>(st, L, T, x, ids, terms, low, exps);
}

// ------------------------------------------------------------------------------ y
// Four waves, each 64 outputs of TT tiles of 16 rows (FEW: of one tile, for the slot of row z of it alone).  The matrix instruction's 32
// columns are 16 ranks twice: lanes 0 - 31 bring a value's first term, lanes 32 - 63 its second, B's ranks the same for both; for
// float rows a second instruction takes the third and the fourth.  Weights are the first operand, so that a lane's sums are 16
// consecutive outputs of one row; they stay in registers from tile to tile while the slot does (RM: the rank tiles there can be).
// All tiles' ids and rows are loaded before the first is waited for.  One row, 4096 outputs: 3.6 us; 67 rows of as many adapters of ranks to
// 64, 4224 float outputs: 9.9, B read once a tile and slot (20 MB from the caches); 4096 rows of 5632: 27, 92 MB read and written, 3.4 TB/s.
template <int DT, int RM, int TT, bool FEW, bool BF>
__global__ __launch_bounds__(256) void k_lora_up(LoraSlots L, int T, const int* __restrict__ ids, const uint16_t* __restrict__ low,
                                                 const int* __restrict__ exps, int64_t ld, const void* y_in, void* y)
{
    constexpr int ES = DT == PHX_F32 ? 4 : 2, V = 16 / ES, TERMS = DT == PHX_F32 ? 4 : 2;  // V: values of 16 bytes
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
    const int grp = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (grp >= L.groups) return;
    const int cols = L.rows - grp * 64 - q * 16;  // this lane's outputs that there are
    const bool wide = cols >= 16 && ld % V == 0 && ((uintptr_t)y_in | (uintptr_t)y) % 16 == 0;
    const int first = blockIdx.x * TT * 16;
    auto place = [&](int tt) { return min(first + tt * 16 + r16, T - 1) * ld + grp * 64 + q * 16; };
    TileSlots S[TT];
    w4 yr[TT][16 / V];
#pragma unroll
    for (int tt = 0; tt < TT; tt++) S[tt].load(ids, L.n_slot, T, first + tt * 16);
    if (FEW) S[0].only(blockIdx.z);
#pragma unroll
    for (int tt = 0; tt < TT; tt++)
        if (wide && (!FEW || (S[tt].left >> r16 & 1)))
#pragma unroll
            for (int i = 0; i < 16 / V; i++) yr[tt][i] = *(const w4*)((const char*)y_in + (place(tt) + i * V) * ES);
    w4 bv[RM][4];
    int held = -1, tiles = 0;  // the slot in bv, and its rank tiles
#pragma unroll
    for (int tt = 0; tt < TT; tt++) {
        if (!S[tt].left) break;  // uniform
        const int row = min(first + tt * 16 + r16, T - 1);
        const int64_t at = place(tt);
        float sum[16];
#pragma unroll
        for (int i = 0; i < 16; i++) sum[i] = 0.0f;
        int slot;
        unsigned rows, mine = 0;  // mine: the rows that are stored
        while (S[tt].next(&slot, &rows)) {
            if (slot >= 0 && slot != held) {
                held = slot;
                tiles = (L.rank[slot] + 15) / 16;
                const uint8_t* b = L.b + slot * L.b_bytes() + (int64_t)grp * L.rt * 2048 + (q & 1) * 256 + r16 * 16;
#pragma unroll
                for (int r = 0; r < RM; r++) {
                    if (r > 0 && r >= tiles) break;  // the first while the rank is on its way
#pragma unroll
                    for (int m = 0; m < 4; m++) bv[r][m] = *(const w4*)(b + r * 2048 + m * 512);
                }
            }
            const int n = slot >= 0 ? tiles : 0;
            if (n > 0 || y_in != y) mine |= rows;
            if (n == 0) continue;
            const bool here = rows >> r16 & 1;
            f32x4 acc[4];
#pragma unroll
            for (int m = 0; m < 4; m++) acc[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const uint16_t* lo = low + (int64_t)row * L.rt * (TERMS * 16) + (q >> 1) * 16 + (q & 1) * 8;
#pragma unroll
            for (int r = 0; r < RM; r++) {
                if (r >= n) break;  // uniform
                w4 t[TERMS / 2];
#pragma unroll
                for (int k = 0; k < TERMS / 2; k++) t[k] = *(const w4*)(lo + (r * TERMS + 2 * k) * 16);
                if (BF) {
#pragma unroll
                    for (int k = 0; k < TERMS / 2; k++)
#pragma unroll
                        for (int m = 0; m < 4; m++) acc[m] = mma16<BF>(bv[r][m], t[k], acc[m]);
                } else {
                    const int ex = here ? exps[(int64_t)row * L.rt + r] : 0;
#pragma unroll
                    for (int m = 0; m < 4; m++) {
                        f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < TERMS / 2; k++) p = mma16<BF>(bv[r][m], t[k], p);
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[m][i] += __builtin_amdgcn_ldexpf(p[i], ex);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < 4; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) sum[4 * m + i] = here ? acc[m][i] : sum[4 * m + i];
        }
        if (!(mine >> r16 & 1)) continue;
        if (wide) {
#pragma unroll
            for (int i = 0; i < 16 / V; i++) {
                float e[V];
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const uint32_t u = yr[tt][i][k * ES / 4], h = k & 1 ? u >> 16 : u & 0xFFFFu;
                    e[k] = (DT == PHX_F32 ? __uint_as_float(u) : DT == PHX_F16 ? h2f(h) : bf2f(h)) + sum[i * V + k];
                }
                store_16<DT>(y, at + i * V, e);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i < cols) store_one<DT>(y, at + i, load_one<DT>(y_in, at + i) + sum[i]);
        }
    }
}

template <int DT, int RM, bool BF>
static void lora_up(hipStream_t st, const LoraSlots& L, int T, const int* ids, const uint16_t* low, const int* exps, int64_t ld,
                    const void* y_in, void* y)
{
    const dim3 blk(256);
    if (few_rows(L, T)) {
        const dim3 grid((T + 15) / 16, (L.groups + 3) / 4, std::min(T, 16));
        launch(k_lora_up<DT, RM, 1, true, BF>, grid, blk, 0, st, L, T, ids, low, exps, ld, y_in, y);
    } else {
        constexpr int TT = 4;
        const dim3 grid((T + 16 * TT - 1) / (16 * TT), (L.groups + 3) / 4);
        launch(k_lora_up<DT, RM, TT, false, BF>, grid, blk, 0, st, L, T, ids, low, exps, ld, y_in, y);
    }
}

template <int DT>
static void lora_up_type(hipStream_t st, const LoraSlots& L, int T, const int* ids, const uint16_t* low, const int* exps, int64_t ld,
                         const void* y_in, void* y)
{
    const bool bf = L.type == PHX_BF16;
    if (L.rt == 1 && bf) lora_up<DT, 1, true>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (L.rt == 1) lora_up<DT, 1, false>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (L.rt == 2 && bf) lora_up<DT, 2, true>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (L.rt == 2) lora_up<DT, 2, false>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (L.rt <= 4 && bf) lora_up<DT, 4, true>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (L.rt <= 4) lora_up<DT, 4, false>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (bf) lora_up<DT, 8, true>(st, L, T, ids, low, exps, ld, y_in, y);
    else lora_up<DT, 8, false>(st, L, T, ids, low, exps, ld, y_in, y);
}

void launch_lora_up(hipStream_t st, const LoraSlots& L, int T, const int* ids, const uint16_t* low, const int* exps, int y_type,
                    int64_t ld, const void* y_in, void* y)
{
    if (y_type == PHX_F16) lora_up_type<PHX_F16>(st, L, T, ids, low, exps, ld, y_in, y);
    else if (y_type == PHX_BF16) lora_up_type<PHX_BF16>(st, L, T, ids, low, exps, ld, y_in, y);
    else lora_up_type<PHX_F32>(st, L, T, ids, low, exps, ld, y_in, y);
}

}  // namespace phx
