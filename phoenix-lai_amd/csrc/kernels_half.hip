// Products with fp16 and bf16 matrices in runs of ragged length (phx_matmul_grouped) and the gated FFN over them
// (phx_experts_half).
//
// Sums are the matrix cores' floats.  Where waves split a reduction they meet in LDS in the waves' order, so no result depends
// on timing.  A place's products involve its own row alone: an infinity or a NaN in another row of a tile reaches nothing.
#include <algorithm>

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

// 16 bytes of weights; ONCE: no other workgroup reads them, so they need not stay in the caches
template <bool ONCE>
__device__ __forceinline__ w4 load_weights(const uint8_t* p)
{
    if constexpr (ONCE) return __builtin_nontemporal_load((const w4*)p);
    else return *(const w4*)p;
}

// act(g) * u, both activations g * sigmoid(z), the exponential and the reciprocal the hardware's (1 ulp each): a few units of
// 2^-24, and the exponential's argument.  Far below, where the quotient is under every number, the reciprocal is 0; the gate
// is then held to a number, so that no infinity meets it.
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

// ------------------------------------------------------------------------------ weights
// The row of its group of 32 that is stored at slot s: what a lane holds of a 32 x 32 product, slots 8 g + 4 h + 0 .. 3 for
// half h, are then 16 consecutive rows.
__device__ __forceinline__ int slot_row(int s) { return 16 * ((s >> 2) & 1) + 4 * (s >> 3) + (s & 3); }

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
    // Item `item` of `per` items a tile, a group's tiles following each other for each of its items: the tile, and which item.
    __device__ __forceinline__ bool find(const HalfArgs& g, int item, int per, Tile* tl, int* which) const
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
    return Groups<false>(g).find(g, tile, 1, tl, &one);
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
    return (uint32_t)(g.dst ? g.dst[tl.start + i] : i) * (uint32_t)g.out_cols * (g.type == PHX_F32 ? 4u : 2u);
}
__device__ __forceinline__ char* out_base(const HalfArgs& g, const Tile& tl)
{
    return (char*)g.out + (g.dst ? 0 : (int64_t)tl.start * g.out_cols * (g.type == PHX_F32 ? 4 : 2));
}

// k_half_rows: for few rows per matrix, where the weights' bytes are the time.  A workgroup takes RT tiles of 16 weight rows
// (PAIRED: of 16 channels, their gate and up rows) by a tile of up to 16 TT places, both straight from memory to registers:
// its NW waves split the reduction, so no operand is wanted by two of them, and a matrix of few rows still has loads in
// flight everywhere.  A wave keeps U steps of 32 columns ahead; the waves' sums meet in LDS, added in the waves' order.
template <int NW, int RT, int TT, bool PAIRED, bool ONCE, bool BF>
__device__ __forceinline__ void half_rows_product(const HalfArgs& g, const Tile& tl, float* red, uint32_t* orow)
{
    constexpr int NB = PAIRED ? 2 : 1, NR = RT * NB, U = NR + TT <= 3 ? 8 : NR + TT <= 6 ? 4 : 3;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bx = blockIdx.x, tiles16 = g.rgs * 2 / NB;  // the matrix's row (channel) tiles of 16
    const uint16_t* xr[TT];
#pragma unroll
    for (int t = 0; t < TT; t++)
        xr[t] = g.x + (int64_t)max(x_row(g, tl.start + min(16 * t + r16, tl.cnt - 1)), 0) * g.cols;
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
    w4 w[U][NR], x[U][TT];
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
        for (int t = 0; t < TT; t++) x[u][t] = *(const w4*)(xr[t] + k);
    };
    auto mma = [&](int u, int s) {
        if (32 * s + 32 > g.cols) {  // uniform: the lanes past the row hold its last values; against zero weights an infinity is none
            const bool past = 32 * s + 8 * q >= g.cols;
#pragma unroll
            for (int t = 0; t < TT; t++) x[u][t] = past ? w4{0, 0, 0, 0} : x[u][t];
        }
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < NR; r++) acc[t][r] = mma16<BF>(x[u][t], w[u][r], acc[t][r]);
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
        store_as(g.type, out + orow[tok], col, y);
    }
}

// CT: the most place tiles of 16 that a tile may hold (its capacity); a tile takes the product of its own count
template <int NW, int RT, int CT, bool PAIRED, bool ONCE, bool BF>
__global__ __launch_bounds__(64 * NW) void k_half_rows(HalfArgs g)
{
    __shared__ float red[NW * RT * CT * (PAIRED ? 2 : 1) * 256];
    __shared__ uint32_t orow[CT * 16];
    Tile tl;
    if (!half_tile(g, blockIdx.y, &tl)) return;  // uniform over the workgroup
    const int n = (tl.cnt + 15) / 16;
    if (CT == 1 || n == 1) half_rows_product<NW, RT, 1, PAIRED, ONCE, BF>(g, tl, red, orow);
    else half_rows_product<NW, RT, CT < 2 ? 1 : 2, PAIRED, ONCE, BF>(g, tl, red, orow);
}

// k_half_tile: four waves, each 64 stored weight rows (PAIRED: the gate and up rows of 32 channels), by a tile of up to 256 places.
// The weights go straight from memory to each wave's registers (the layout has every operand as one run of 1 KB, and no other wave
// of the workgroup wants it), nearly two steps of 64 columns ahead; the places' rows, which all four waves read, go through an LDS
// ring by direct loads three to five steps ahead, row-major runs of 128 bytes with the 16-byte chunks XOR-swizzled by half the row's number
// (16 lanes of a 16-byte read then have 16 distinct bank groups).
constexpr int TI_WAVE = 32 * (64 * 4 + 16);  // a wave's part of the ring in the epilogue: 32 places' rows of 64 floats
// slots: as many steps as the ring holds, up to six (MT: the row tiles it is made for, 16 KB each)
constexpr int ti_ring(int nt, int mt) { return std::min(mt * 4 / nt, 6); }

template <int NT, int MT, bool PAIRED, bool ONCE, bool BF>
__device__ __forceinline__ void half_tile_product(const HalfArgs& g, const Tile& tl, int bx, unsigned char* ring, uint32_t* orow)
{
    constexpr int STAGE = NT * 32 * 128, RING = ti_ring(NT, MT);
    const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = g.kc / 8, row_bytes = g.cols * 2;
    // this lane's rows of the direct loads: one per load, the last row again past the tile's end
    const int chunk = ((lane & 7) ^ (lane >> 4)) * 16;  // of the loads whose first row is a multiple of 16; 4 chunks on for 8
    const __amdgpu_buffer_rsrc_t rsrc = buf_rsrc(g.x + (g.src ? 0 : (int64_t)tl.start * g.cols));
    uint32_t xr[NT];  // rows that src names lie within 2^32 bytes of x, a tile's own of its first
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int at = min(8 * (wave * NT + i) + (lane >> 3), tl.cnt - 1);
        xr[i] = (uint32_t)(g.src ? max(x_row(g, tl.start + at), 0) : at) * (uint32_t)row_bytes;
    }
    for (int i = tid; i < NT * 32; i += 256) orow[i] = out_row(g, tl, i);
    int slot = 0;  // the ring's slot of a step; the one before it takes the rows of the step RING - 1 on
    auto after = [&](int at) { return at == (RING - 1) * STAGE ? 0 : at + STAGE; };
    auto before = [&](int at) { return at == 0 ? (RING - 1) * STAGE : at - STAGE; };
    auto column = [&](int s, int i) { return s * 128 + (chunk ^ (64 * ((wave * NT + i) & 1))); };  // the lane's byte of load i's rows
    auto dma = [&](int s, int to, auto I) {          // load I of step s's rows
        constexpr int i = decltype(I)::value;
        const int off = column(min(s, S - 1), i);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t)(ring + to + (wave * NT + i) * 1024), 16,
                                                 xr[i] + (off < row_bytes ? off : 0), 0, 0, 0);
    };
    // zeros where a last step's loads, landed, hold columns past the row: against zero weights an infinity is none
    auto clear = [&](int s, int to) {
        if (s != S - 1 || row_bytes == S * 128) return;  // uniform
#pragma unroll
        for (int i = 0; i < NT; i++)
            if (column(s, i) >= row_bytes) *(uint4*)(ring + to + (wave * NT + i) * 1024 + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    const int rg0 = (bx * 4 + wave) * 2, rgs = g.rgs;
    const uint8_t* wb[2];
#pragma unroll
    for (int b = 0; b < 2; b++)
        wb[b] = g.w + (int64_t)tl.e * g.mat_bytes + (int64_t)min(rg0 + b, rgs - 1) * g.kc * 512;
    const uint32_t lane16 = lane * 16;
    w4 wv[2][2][4];
    auto weight = [&](int s, int b, auto P, auto KK) {
        const uint8_t* at = wb[b] + (int64_t)min(s, S - 1) * 4096 + decltype(KK)::value * 1024;  // uniform
        wv[decltype(P)::value][b][decltype(KK)::value] = load_weights<ONCE>(at + lane16);
    };
    f32x16 acc[NT][2];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[j][b][v] = 0.0f;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void_t)ring + r32 * 128, swz = (h ^ ((r32 >> 1) & 7)) * 16;
    u32x4 a[2][NT];
    auto read = [&](int from, auto KK, auto J) {  // row tile J's columns of group KK
        constexpr int kk = decltype(KK)::value, j = decltype(J)::value;
        a[kk & 1][j] = ds_r128<j * 4096>(lds + from + (swz ^ (kk * 32)));
    };
    auto landed = [&](auto Q) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int j = 0; j < NT; j++) tie(a[decltype(Q)::value][j]);
    };
    // A step is four groups of products on 16 columns.  Behind each of a group's first products goes a read of the next group's
    // rows (the last group: of the next step's, once they have landed in every wave, which also says that nobody reads this step's
    // slot any more): all at the group's start, the four waves' reads held up each other and the products behind them (8192 x
    // 8192 x 8192 READS_AT_START us).  Behind the others go the loads: the weights that the group before has just used the
    // registers of, two steps on, and the group's share of the rows RING - 1 steps on.  The order is fixed by scheduling barriers:
    // the wait for the rows counts the loads issued after them.
    constexpr int DPG = (NT + 3) / 4;                                     // direct loads of a group
    constexpr int LAST = (NT - 1) / DPG, AFTER = 2 * (3 - LAST);          // the group of a step's last one, the weights after it
    constexpr int NEWER = AFTER + (RING - 3) * (8 + NT) + 6 + (NT < 3 * DPG ? NT : 3 * DPG);
    // the loads behind the first step's rows
    constexpr int NEWER_AT_START = (RING - 2) * NT + 14;
    static_assert(NEWER < 64 && NEWER_AT_START < 64 && RING > 3, "vmcnt's range, and the first step's rows before any weights");
    auto step = [&](int s, auto P) {
        constexpr int p = decltype(P)::value;
        const int next = after(slot), far = before(slot);
        static_for<4>([&](auto KK) {
            constexpr int kk = decltype(KK)::value;
            static_for<2 * NT>([&](auto M) {
                constexpr int m = decltype(M)::value, j = m / 2, b = m % 2;
                __builtin_amdgcn_sched_barrier(0);
                acc[j][b] = mma32<BF>(wv[p][b][kk], a[kk & 1][j], acc[j][b]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (m == 0 && kk == 3) {
                    __builtin_amdgcn_s_waitcnt(vm_wait(NEWER));
                    clear(s + 1, next);
                    __builtin_amdgcn_s_barrier();
                }
                if constexpr (m < NT) read(kk < 3 ? slot : next, ic<(kk + 1) % 4>{}, ic<(m < NT ? m : 0)>{});
                static_for<2 + DPG>([&](auto I) {
                    constexpr int i = decltype(I)::value, d = kk * DPG + i - 2;
                    if constexpr (m == NT + i * NT / (2 + DPG)) {
                        if constexpr (i < 2 && kk == 0) weight(s + 1, i, ic<1 - p>{}, ic<3>{});
                        else if constexpr (i < 2) weight(s + 2, i, ic<p>{}, ic<(kk + 3) % 4>{});
                        else if constexpr (d < NT) dma(s + RING - 1, far, ic<d>{});
                    }
                });
            });
            __builtin_amdgcn_sched_barrier(0);
            landed(ic<(kk + 1) & 1>{});
        });
        slot = next;
    };
    // The loads before the first step in the order of the steps that would have issued them: the waits for weights inside the loop
    // hold for its first pass too, and in another order would have to count fewer loads ever after.
    static_for<RING - 3>([&](auto R) {
        static_for<NT>([&](auto I) { dma(decltype(R)::value, decltype(R)::value * STAGE, I); });
    });
    static_for<2>([&](auto P) {
        constexpr int p = decltype(P)::value, r = RING - 3 + p;  // step p - 2, its rows those of step r
        static_for<4>([&](auto KK) {
            constexpr int kk = decltype(KK)::value;
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kk > 0) weight(p, 0, ic<p>{}, ic<(kk + 3) % 4>{}), weight(p, 1, ic<p>{}, ic<(kk + 3) % 4>{});
            else if constexpr (p == 1) weight(0, 0, ic<0>{}, ic<3>{}), weight(0, 1, ic<0>{}, ic<3>{});
            __builtin_amdgcn_sched_barrier(0);
            static_for<DPG>([&](auto D) {
                constexpr int d = kk * DPG + decltype(D)::value;
                if constexpr (d < NT) dma(r, r * STAGE, ic<d>{});
            });
        });
    });
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(vm_wait(NEWER_AT_START));
    clear(0, slot);
    __builtin_amdgcn_s_barrier();
    static_for<NT>([&](auto J) { read(slot, ic<0>{}, J); });
    landed(ic<0>{});
    for (int s = 0; s + 1 < S; s += 2) {
        step(s, ic<0>{});
        step(s + 1, ic<1>{});
    }
    if (S & 1) step(S - 1, ic<0>{});
    __builtin_amdgcn_s_waitcnt(0);  // the direct loads past the last step land before the workgroup's LDS goes
    __syncthreads();
    char* out = out_base(g, tl);
    // A lane holds 16 consecutive channels of one place (twice, or gate and up).  Each 32 places' values go through the wave's own part
    // of the ring as they are stored, so that an instruction stores whole runs of a place's row: 128 bytes where the lane alone
    // has 32.  A row's 16 bytes more than its values keep 16 lanes of a write or read on distinct banks.
    constexpr int WC = PAIRED ? 32 : 64;
    unsigned char* mine = ring + wave * TI_WAVE;
    const int col0 = PAIRED ? (rg0 >> 1) * 32 : rg0 * 32;
    const bool bf = g.type == PHX_BF16;
    auto store = [&](auto ESC, auto J) {
        constexpr int j = decltype(J)::value, ES = decltype(ESC)::value, V = 16 / ES, LPT = WC / V, TPI = 64 / LPT, PITCH = WC * ES + 16;
#pragma unroll
        for (int b = 0; b < (PAIRED ? 1 : 2); b++)
#pragma unroll
            for (int i = 0; i < 16; i += V) {
                float y[V];
#pragma unroll
                for (int v = 0; v < V; v++) y[v] = PAIRED ? gated_half(g.act, acc[j][0][i + v], acc[j][1][i + v]) : acc[j][b][i + v];
                unsigned char* to = mine + r32 * PITCH + (32 * b + 16 * h + i) * ES;
                if constexpr (ES == 4) *(float4*)to = make_float4(y[0], y[1], y[2], y[3]);
                else {
                    uint32_t u[4];
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const uint32_t as_bf = pair_of<PHX_BF16>(y[2 * v], y[2 * v + 1]), as_f16 = pair_of<PHX_F16>(y[2 * v], y[2 * v + 1]);
                        u[v] = bf ? as_bf : as_f16;
                    }
                    *(uint4*)to = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int c = (lane % LPT) * V, col = col0 + c;  // LPT lanes a place, TPI places a round
        const bool whole = g.out_cols % V == 0;          // rows and columns then start on 16 bytes
#pragma unroll
        for (int it = 0; it < 32 / TPI; it++) {
            const int tok = it * TPI + lane / LPT;
            const uint32_t o = orow[32 * j + tok];
            const uint4 y = *(const uint4*)(mine + tok * PITCH + c * ES);
            if (o == NO_ROW) continue;
            if (whole) {
                if (col < g.out_cols) *(uint4*)(out + o + (int64_t)col * ES) = y;
            } else {
                const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (col + i < g.out_cols) {
                        if constexpr (ES == 4) *(uint32_t*)(out + o + (int64_t)(col + i) * 4) = u[i];
                        else *(uint16_t*)(out + o + (int64_t)(col + i) * 2) = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
                    }
            }
        }
        // this tile's reads end before the next one's writes
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_sched_barrier(0);
    };
    if (g.type == PHX_F32) static_for<NT>([&](auto J) { store(ic<4>{}, J); });
    else static_for<NT>([&](auto J) { store(ic<2>{}, J); });
}

// Workgroup L runs on XCD L % 8.  The items (a tile's block of 256 stored rows) are in the order of groups, blocks, tiles, and
// each XCD takes an eighth of them as one run: a group's tiles meet a block's weights in one L2 at about one time, and the weights
// leave memory once.
template <int MT, bool PAIRED, bool ONCE, bool BF>
__global__ __launch_bounds__(256, MT > 4 ? 1 : 2) void k_half_tile(HalfArgs g)
{
    __shared__ __align__(16) unsigned char ring[MT * 16 * 1024];
    static_assert(sizeof(ring) >= 4 * TI_WAVE, "the epilogue's part of each wave");
    __shared__ __align__(16) uint32_t orow[MT * 32];
    const Groups<true> G(g);
    const int blocks = (g.rgs + 7) / 8, all = G.total() * blocks, run = (all + 7) / 8, k = blockIdx.x >> 3;
    const int item = (blockIdx.x & 7) * run + k;
    Tile tl;
    int bx;
    if (k >= run || item >= all || !G.find(g, item, blocks, &tl, &bx)) return;  // uniform over the workgroup
    // said once more, so that addresses stay in scalar registers: a buffer in vector ones costs a loop for each load
    tl = {__builtin_amdgcn_readfirstlane(tl.e), __builtin_amdgcn_readfirstlane(tl.start), __builtin_amdgcn_readfirstlane(tl.cnt)};
    bx = __builtin_amdgcn_readfirstlane(bx);
    const int n = (tl.cnt + 31) / 32;
    if constexpr (MT == 4) {
        switch (n) {
        case 1: half_tile_product<1, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 2: half_tile_product<2, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 3: half_tile_product<3, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        default: half_tile_product<4, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow);
        }
    } else {
        switch (n) {
        case 1: half_tile_product<1, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 2: half_tile_product<2, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 3: half_tile_product<3, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 4: half_tile_product<4, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 5: half_tile_product<5, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 6: half_tile_product<6, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        case 7: half_tile_product<7, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow); break;
        default: half_tile_product<8, MT, PAIRED, ONCE, BF>(g, tl, bx, ring, orow);
        }
    }
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
    if (m.type == PHX_BF16) launch(k_half_rows<NW, RT, CT, PAIRED, ONCE, true>, grid, blk, 0, st, g);
    else launch(k_half_rows<NW, RT, CT, PAIRED, ONCE, false>, grid, blk, 0, st, g);
}

template <int CT, bool ONCE>
static void rows_by_pair(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    if (m.paired) half_rows<4, 2, CT, true, ONCE>(st, m, g, max_tiles);
    else half_rows<4, 4, CT, false, ONCE>(st, m, g, max_tiles);
}

template <int MT, bool PAIRED>
static void half_tiles(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    const dim3 grid((max_tiles * ((m.rg + 7) / 8) + 7) / 8 * 8), blk(256);
    if (m.type == PHX_BF16) launch(k_half_tile<MT, PAIRED, false, true>, grid, blk, 0, st, g);
    else launch(k_half_tile<MT, PAIRED, false, false>, grid, blk, 0, st, g);
}

void launch_half_product(hipStream_t st, const HalfMat& m, HalfArgs g, int max_tiles)
{
    set_matrix(g, m);
    if (g.cap <= 16) rows_by_pair<1, false>(st, m, g, max_tiles);
    else if (g.cap <= kHalfRows) rows_by_pair<2, false>(st, m, g, max_tiles);
    else if (g.cap <= kHalfNarrow) {
        if (m.paired) half_tiles<4, true>(st, m, g, max_tiles);
        else half_tiles<4, false>(st, m, g, max_tiles);
    } else if (m.paired) half_tiles<8, true>(st, m, g, max_tiles);
    else half_tiles<8, false>(st, m, g, max_tiles);
}

// ------------------------------------------------------------------------------ experts
// The down products of few assignments and their weighted sum, for a token (blockIdx.y) and 16 of its outputs: wave w takes
// the token's places w, w + NW, ..., and the places' values meet in LDS in order.  No lists and no partial outputs go through
// memory.
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
        const uint16_t* row = g.x + (t * k + j) * g.cols;
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < steps; s += U) {
            w4 w[U], x[U];
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = *(const w4*)(wb + (int64_t)min(s + u, steps - 1) * 2048);
#pragma unroll
            for (int u = 0; u < U; u++) x[u] = *(const w4*)(row + min(32 * (s + u) + 8 * q, g.cols - 8));
#pragma unroll
            for (int u = 0; u < U; u++)
                if (s + u < steps) {  // uniform
                    if (32 * (s + u) + 8 * q >= g.cols) x[u] = w4{0, 0, 0, 0};
                    acc = mma16<BF>(x[u], w[u], acc);  // every row of the first operand is the place's
                }
        }
        if (lane < 16) vals[j][lane] = acc[0];
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
