// Products with fp16 and bf16 matrices in runs of ragged length (phx_matmul_grouped) and the gated FFN over them
// (phx_experts_half).
//
// Sums are the matrix cores' floats.  Where waves split a reduction they meet in LDS in the waves' order, so no result depends
// on timing.  A place's products involve its own row alone: an infinity or a NaN in another row of a tile reaches nothing.
#include "half_common.h"

namespace phx {

// ------------------------------------------------------------------------------ weights
// HalfMat's layout from matrices as the caller holds them: a thread writes 8 columns of one stored row, zeros past the
// last row or column.
__global__ __launch_bounds__(256) void k_half_pack(HalfMat m, int m0, int64_t n16, const uint16_t* __restrict__ w)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n16) return;
    const int s32 = slot_row((int)(i & 31)), kc = (int)((i >> 5) % m.kc);
    const int64_t g = (i >> 5) / m.kc;  // 32-row group over the matrices from m0
    const int rg = (int)(g % m.rg), mi = (int)(g / m.rg);
    const int half = m.rows / 2;
    int r = rg * 32 + s32;
    if (m.paired) r = (rg >> 1) * 32 + s32 + (rg & 1) * half;
    const bool live = m.paired ? (rg >> 1) * 32 + s32 < half : r < m.rows;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (live && kc * 8 < m.cols) {
        const uint16_t* p = w + ((int64_t)mi * m.rows + r) * m.cols + kc * 8;
        if (((uintptr_t)w & 15) == 0) v = *(const uint4*)p;
        else v = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
    }
    *(uint4*)(m.w + (int64_t)m0 * m.mat_bytes() + i * 16) = v;
}

void launch_half_pack(hipStream_t st, const HalfMat& m, int m0, int n_mat, const uint16_t* w)
{
    const int64_t n16 = (int64_t)n_mat * m.mat_bytes() / 16;
    launch(k_half_pack, dim3((unsigned)((n16 + 255) / 256)), dim3(256), 0, st, m, m0, n16, w);
}

// ------------------------------------------------------------------------------ products
// k_half_rows: for few rows per matrix, where the weights' bytes are the time.  A workgroup takes RT tiles of 16 weight rows
// (PAIRED: of 16 channels, their gate and up rows) by a tile of up to 16 TT places, both straight from memory to registers:
// its NW waves split the reduction, so no operand is wanted by two of them, and a matrix of few rows still has loads in
// flight everywhere.  A wave keeps U steps of 32 columns ahead; the waves' sums meet in LDS, added in the waves' order.
// XT: the terms of a row of x, both times a step's weights.
template <int NW, int RT, int TT, int XT, bool PAIRED, bool ONCE, bool BF>
__device__ __forceinline__ void half_rows_product(const HalfArgs& g, const Tile& tl, float* red, uint32_t* orow)
{
    constexpr int NB = PAIRED ? 2 : 1, NR = RT * NB, U = NR + TT * XT <= 3 ? 8 : NR + TT * XT <= 6 ? 4 : 3;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bx = blockIdx.x, tiles16 = g.rgs * 2 / NB;  // the matrix's row (channel) tiles of 16
    const uint16_t* xr[TT];
#pragma unroll
    for (int t = 0; t < TT; t++)
        xr[t] = g.x + (int64_t)max(x_row(g, tl.start + min(16 * t + r16, tl.cnt - 1)), 0) * (g.cols * XT);
    const uint8_t* wb[NR];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int i = min(bx * RT + r, tiles16 - 1);
            wb[r * NB + b] = g.w + (int64_t)tl.e * g.mat_bytes + ((int64_t)(i >> 1) * NB + b) * g.kc * 512 + (i & 1) * 256;
        }
    const int lo = q * 512 + r16 * 16;
    if (tid < TT * 16) orow[tid] = out_row(g, tl, tid);
    f32x4 acc[TT][NR];
    w4 w[U][NR], x[U][TT][XT];
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < NR; r++) acc[t][r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (g.cols + 31) / 32, s0 = wave * steps / NW, s1 = (wave + 1) * steps / NW;
    auto load = [&](int u, int s) {
        const int su = min(s, s1 - 1), k = min(32 * su + 8 * q, g.cols - 8);
#pragma unroll
        for (int r = 0; r < NR; r++) w[u][r] = load_weights<ONCE>(wb[r] + (int64_t)su * 2048 + lo);
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int z = 0; z < XT; z++) x[u][t][z] = *(const w4*)(xr[t] + z * g.cols + k);
    };
    auto mma = [&](int u, int s) {
        if (32 * s + 32 > g.cols) {  // uniform: the lanes past the row hold its last values; against zero weights an infinity is none
            const bool past = 32 * s + 8 * q >= g.cols;
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int z = 0; z < XT; z++) x[u][t][z] = past ? w4{0, 0, 0, 0} : x[u][t][z];
        }
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int z = 0; z < XT; z++) acc[t][r] = mma16<BF>(x[u][t][z], w[u][r], acc[t][r]);
    };
    if (s0 < s1) {  // uniform over the wave
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
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int v = 0; v < 4; v++) red[(wave * TT * NR + t * NR + r) * 256 + v * 64 + lane] = acc[t][r][v];
    __syncthreads();
    // a thread keeps one column, C threads a place, P places at a time
    constexpr int C = RT * 16, P = 64 * NW / C;
    const int c = tid % C, slot = bx * C + c, col = (slot & ~31) + slot_row(slot & 31);
    if (col >= g.out_cols) return;
    char* out = out_base(g, tl);
#pragma unroll
    for (int it = 0; it < (TT * 16 + P - 1) / P; it++) {
        const int tok = it * P + tid / C, i = tok & 15;
        if (tok >= tl.cnt) break;
        if (orow[tok] == NO_ROW) continue;
        const int at = ((tok >> 4) * NR + (c >> 4) * NB) * 256 + (i & 3) * 64 + (c & 15) + 16 * (i >> 2);
        float y = 0.0f, up = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) {
            y += red[k * TT * NR * 256 + at];
            if (PAIRED) up += red[k * TT * NR * 256 + at + 256];
        }
        if (PAIRED) y = gated_half(g.act, y, up);
        if (PAIRED && g.out_terms == 2) {
            uint16_t t[2];
            split<BF>(y, t);
            for (int z = 0; z < 2; z++) ((uint16_t*)(out + orow[tok]))[z * g.out_cols + col] = t[z];
        } else store_as(g.type, out + orow[tok], col, y);
    }
}

// CT: the most place tiles of 16 that a tile may hold (its capacity); a tile takes the product of its own count
template <int NW, int RT, int CT, int XT, bool PAIRED, bool ONCE, bool BF>
__global__ __launch_bounds__(64 * NW) void k_half_rows(HalfArgs g)
{
    __shared__ float red[NW * RT * CT * (PAIRED ? 2 : 1) * 256];
    __shared__ uint32_t orow[CT * 16];
    Tile tl;
    if (!half_tile(g, blockIdx.y, &tl)) return;  // uniform over the workgroup
    const int n = (tl.cnt + 15) / 16;
    if (CT == 1 || n == 1) half_rows_product<NW, RT, 1, XT, PAIRED, ONCE, BF>(g, tl, red, orow);
    else half_rows_product<NW, RT, CT < 2 ? 1 : 2, XT, PAIRED, ONCE, BF>(g, tl, red, orow);
}

static void set_matrix(HalfArgs& g, const HalfMat& m)
{
    g.w = m.w;
    g.mat_bytes = m.mat_bytes();
    g.kc = m.kc;
    g.cols = m.cols;
    g.out_cols = m.paired ? m.rows / 2 : m.rows;
    g.rgs = m.rg;
    g.n_mat = m.n_mat;
}

template <int NW, int RT, int CT, bool PAIRED, bool ONCE>
static void half_rows(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    const dim3 grid(((g.out_cols + 31) / 32 * 32 + 16 * RT - 1) / (16 * RT), max_tiles), blk(64 * NW);  // stored rows in whole groups
    constexpr int XT = PAIRED ? 1 : 2;
    if (m.type == PHX_BF16 && g.x_terms < XT) launch(k_half_rows<NW, RT, CT, 1, PAIRED, ONCE, true>, grid, blk, 0, st, g);
    else if (m.type == PHX_BF16) launch(k_half_rows<NW, RT, CT, XT, PAIRED, ONCE, true>, grid, blk, 0, st, g);
    else if (g.x_terms < XT) launch(k_half_rows<NW, RT, CT, 1, PAIRED, ONCE, false>, grid, blk, 0, st, g);
    else launch(k_half_rows<NW, RT, CT, XT, PAIRED, ONCE, false>, grid, blk, 0, st, g);
}

// Four waves and 32 channels or 64 outputs; plain matrices with at most a workgroup a compute unit then, eight waves and 32 outputs (us, four
// waves with 64 outputs, with 32, eight with 64, with 32; 96 places in 64 groups of 4096 x 1408: 60, 68, 80, 80; one matrix of 4096 x
// 4096: 1 place 10.4, 9.3, 10.4, 8.9; 16 places 12.9, 10.7, 12.4, 10.2; 128 places 17.5, 23.5, 18.1, 23.5; 16384 x 4096, 12 places 29,
// 28, 28, 27; paired, of 32 or 16 channels: 512 places in 128 groups of 1408 x 2816 134, 139, 135, 155; 192 in 32 of 1024 x 1024 12.9,
// 13.4, 14.1, 15.2).
template <int CT, bool ONCE>
static void rows_by_pair(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    if (m.paired) half_rows<4, 2, CT, true, ONCE>(st, m, g, max_tiles);
    else if (CT == 1 && max_tiles * ((m.rg + 1) / 2) <= 256) half_rows<8, 2, 1, false, ONCE>(st, m, g, max_tiles);
    else half_rows<4, 4, CT, false, ONCE>(st, m, g, max_tiles);
}

void launch_half_product(hipStream_t st, const HalfMat& m, HalfArgs g, int max_tiles)
{
    set_matrix(g, m);
    if (g.cap <= 16 && g.once) rows_by_pair<1, true>(st, m, g, max_tiles);
    else if (g.cap <= 16) rows_by_pair<1, false>(st, m, g, max_tiles);
    else if (g.cap <= kHalfRows && g.once) rows_by_pair<2, true>(st, m, g, max_tiles);
    else if (g.cap <= kHalfRows) rows_by_pair<2, false>(st, m, g, max_tiles);
    else if (g.x_terms == 2 || g.out_terms == 2) {
        if (m.type == PHX_BF16) launch_half_tiles<true, true>(st, m, g, max_tiles);
        else launch_half_tiles<false, true>(st, m, g, max_tiles);
    } else if (m.type == PHX_BF16) launch_half_tiles<true, false>(st, m, g, max_tiles);
    else launch_half_tiles<false, false>(st, m, g, max_tiles);
}

// ------------------------------------------------------------------------------ experts
// The down products of few assignments and their weighted sum, for a token (blockIdx.y) and 16 of its outputs: wave w takes
// the token's places w, w + NW, ..., and the places' values meet in LDS in order.  No lists and no partial outputs go through
// memory.  One instruction takes both terms of a place's row, as its even and its odd rows.  One token's eight experts of 2816 x 704 take
// 8.1 us (a launch 3.4, two dependent trips to memory).
template <int NW, bool BF>
__global__ __launch_bounds__(64 * NW) void k_half_down_few(HalfArgs g, int k, const float* __restrict__ weights)
{
    __shared__ float vals[PHX_MAX_USED][16];
    constexpr int U = 12;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4, bx = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = blockIdx.y;
    const int steps = (g.cols + 31) / 32;
    for (int j = wave; j < k; j += NW) {
        const int e = g.ids[t * k + j];  // uniform
        if ((unsigned)e >= (unsigned)g.n_mat) continue;
        const uint8_t* wb = g.w + (int64_t)e * g.mat_bytes + (int64_t)(bx >> 1) * g.kc * 512 + (bx & 1) * 256 + q * 512 + r16 * 16;
        // every even row of the first operand is the place's first terms, every odd one its second
        const uint16_t* row = g.x + ((t * k + j) * 2 + (lane & 1)) * g.cols;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < steps; s += U) {
            w4 w[U], x[U];
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = load_weights<false>(wb + (int64_t)min(s + u, steps - 1) * 2048);
#pragma unroll
            for (int u = 0; u < U; u++) x[u] = *(const w4*)(row + min(32 * (s + u) + 8 * q, g.cols - 8));
#pragma unroll
            for (int u = 0; u < U; u++)
                if (s + u < steps) {  // uniform
                    if (32 * (s + u) + 8 * q >= g.cols) x[u] = w4{0, 0, 0, 0};
                    acc = mma16<BF>(x[u], w[u], acc);
                }
        }
        if (lane < 16) vals[j][lane] = acc[0] + acc[1];
    }
    __syncthreads();
    const int slot = bx * 16 + threadIdx.x, col = (slot & ~31) + slot_row(slot & 31);
    if (threadIdx.x < 16 && col < g.out_cols) {
        float acc = 0.0f;
        for (int j = 0; j < k; j++)
            if ((unsigned)g.ids[t * k + j] < (unsigned)g.n_mat) acc += vals[j][threadIdx.x] * weights[t * k + j];
        store_as(g.type, g.out, t * g.out_cols + col, acc);
    }
}

void launch_half_down_few(hipStream_t st, const HalfMat& m, int T, int k, const uint16_t* h, const int* ids, const float* weights,
                          int out_type, void* out)
{
    HalfArgs g{};
    set_matrix(g, m);
    g.x = h;
    g.ids = ids;
    g.type = out_type;
    g.out = out;
    const dim3 grid((g.out_cols + 31) / 32 * 2, T);
    if (k <= 4 && m.type == PHX_BF16) launch(k_half_down_few<4, true>, grid, dim3(256), 0, st, g, k, weights);
    else if (k <= 4) launch(k_half_down_few<4, false>, grid, dim3(256), 0, st, g, k, weights);
    else if (m.type == PHX_BF16) launch(k_half_down_few<8, true>, grid, dim3(512), 0, st, g, k, weights);
    else launch(k_half_down_few<8, false>, grid, dim3(512), 0, st, g, k, weights);
}

}  // namespace phx
