// int8 products with a scale per token and per output channel (phx_quant_i8, phx_matmul_i8, phx_experts_i8).
//
// Every sum of products is a whole number below 2^31 (65536 columns of at most 128 x 128), so the matrix cores' int32 sums
// are exact in any order: reductions are split over waves and joined by integer additions without a word about order.  What
// is rounded is stated at phx_matmul_i8: the sum to float, the scales' product, the value; nothing else between a row's
// integers and an output.
#include <algorithm>

#include "device_common.h"
#include "i8_rows.h"
#include "rows_io.h"

namespace phx {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// 16 bytes of weights; ONCE: no other workgroup reads them, so they need not stay in the caches
template <bool ONCE>
__device__ __forceinline__ i32x4 load_weights(const int8_t* p)
{
    if constexpr (ONCE) return __builtin_nontemporal_load((const i32x4*)p);
    else return *(const i32x4*)p;
}

// ------------------------------------------------------------------------------ rows to int8
__device__ __forceinline__ float silu_ref(float v) { return v / (1.0f + (float)exp(-(double)v)); }

// 2^f on [-1/2, 1/2] in double, the Taylor series of exp(f ln 2) to f^11: within 2^-46
__device__ __forceinline__ double exp2_frac(double f)
{
    const double x = f * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, x, 1.0 / 3628800.0);
    p = __builtin_fma(p, x, 1.0 / 362880.0);
    p = __builtin_fma(p, x, 1.0 / 40320.0);
    p = __builtin_fma(p, x, 1.0 / 5040.0);
    p = __builtin_fma(p, x, 1.0 / 720.0);
    p = __builtin_fma(p, x, 1.0 / 120.0);
    p = __builtin_fma(p, x, 1.0 / 24.0);
    p = __builtin_fma(p, x, 1.0 / 6.0);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    return __builtin_fma(p, x, 1.0);
}
// exp(x) in double for |x| <= 128, within 2^-45 of it: past the float it is rounded to by 21 bits
__device__ __forceinline__ double exp_near(double x)
{
    const double t = x * 1.44269504088896340736, n = __builtin_rint(t);
    return __builtin_amdgcn_ldexp(exp2_frac(t - n), (int)n);
}
// silu_ref and gelu_ref without the library's exponential and the table: 27 and 45 instructions a value (a gate|up tile's
// epilogue 24 us; by the exponential and a gather a value it took as long as the tile's products).  The same roundings:
// silu's quotient by the reciprocal, one refinement and two corrections, which round it correctly while nothing leaves
// the normal numbers (|v| < 80); gelu equals the table at every fp16 value (tests).
__device__ __forceinline__ float silu_near(float v)
{
    if (fabsf(v) >= 80.0f || v != v) return silu_ref(v);
    const float d = 1.0f + (float)exp_near(-(double)v);
    float y = __builtin_amdgcn_rcpf(d);
    y = __builtin_fmaf(__builtin_fmaf(-d, y, 1.0f), y, y);
    float q = v * y;
    q = __builtin_fmaf(__builtin_fmaf(-d, q, v), y, q);
    q = __builtin_fmaf(__builtin_fmaf(-d, q, v), y, q);
    return __builtin_copysignf(q, v);  // of -0 the corrections make +0
}
__device__ __forceinline__ float gelu_near(float x)
{
    if (!(x > -10.0f)) return 0.0f;  // and for a NaN, as the table has it
    if (x >= 10.0f) return x;
    const float h = h2f(f2h_bits(x));
    if (h <= -10.0f) return 0.0f;
    if (h >= 10.0f) return h;
    const float inner = 0.79788456080286535587989211986876f * h * (1.0f + 0.044715f * h * h);
    // tanh(z) = 1 - 2 / (1 + exp(2 z)), 1 from |z| = 22 on; the reciprocal from the hardware's by two refinements
    const double z2 = 2.0 * (double)fminf(fmaxf(inner, -22.0f), 22.0f), e = 1.0 + exp_near(z2);
    double y = __builtin_amdgcn_rcp(e);
    y = __builtin_fma(__builtin_fma(-e, y, 1.0), y, y);
    y = __builtin_fma(__builtin_fma(-e, y, 1.0), y, y);
    const float t = (float)__builtin_fma(-2.0, y, 1.0);
    return h2f(f2h_of(0.5f * h * (1.0f + t)));
}

// act(gate) * up
__device__ __forceinline__ float gated(int act, float gate, float up)
{
    return (act == PHX_QUANT_SILU_MUL ? silu_near(gate) : gelu_near(gate)) * up;
}
// h as phx_quant_i8 forms it: a NaN gate stays one, so that the row which held it says so in its scale (gelu_near, like
// the table, has 0 there)
__device__ __forceinline__ float gated_kept(int act, float gate, float up)
{
    const float h = gated(act, gate, up);
    return gate != gate ? gate : h;
}

// NT threads per row, eight consecutive values per thread and step, the row held in registers between its statistics and its
// integers: one pass over memory, which bounds it (8192 rows of 4096 fp16 values: 20 to 24 us, 4.2 to 5.0 TB/s).  The row's own
// loads all go out before the first wait; a norm's weights are loaded after the sum's barrier, a second trip (2048 rows of 4096
// bf16, normed: 9 us, of which their bytes take 6).  A row of one wave needs no barrier, and a workgroup then takes four.  A
// thread's steps past its row load and form the row's last values again: 2112 values pay for 4096, 14336 for 65536.
template <int NT, int STEPS, int MODE, int DT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_quant_i8(int rows, int n, int64_t ld, float eps,
                                                                  const void* __restrict__ x, const void* __restrict__ aux,
                                                                  int8_t* __restrict__ qs, float* __restrict__ d)
{
    constexpr int RPB = NT < 256 ? 256 / NT : 1, NW = NT / 64;
    __shared__ double red[NW];
    __shared__ unsigned redu[NW];
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
    if (NT == 64 && row >= rows) return;  // a whole wave, and no barrier with one wave a row
    const int tid = threadIdx.x % NT, lane = tid & 63, wave = tid >> 6;
    float v[STEPS][8];
    auto at = [&](int s) { return min((s * NT + tid) * 8, n - 8); };  // past the row its last values
#pragma unroll
    for (int s = 0; s < STEPS; s++) load_eight<DT>(x, row * ld + at(s), v[s]);
    float scale = 0.0f;
    if (MODE == PHX_QUANT_RMS_NORM) {
        double sum = 0.0;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
            if ((s * NT + tid) * 8 < n)
#pragma unroll
                for (int j = 0; j < 8; j++) sum += (double)v[s][j] * (double)v[s][j];
        sum = wave_sum_dpp(sum);
        if (NW > 1) {
            if (lane == 0) red[wave] = sum;
            __syncthreads();
            sum = 0.0;
            for (int w = 0; w < NW; w++) sum += red[w];
        }
        scale = rms_scale_from_mean((float)(sum / (double)n), eps);
    }
    unsigned am = 0;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        if (MODE != PHX_QUANT_PLAIN) {
            float a[8];
            if (MODE == PHX_QUANT_RMS_NORM) load_eight<PHX_F32>(aux, at(s), a);
            else load_eight<DT>(aux, row * ld + at(s), a);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float u = v[s][j];
                // silu by the library's exponential: the rows' bytes bound this kernel, and the shorter code is the faster one
                // (77 rows of 2112: 4.1 us, by silu_near 5.1)
                v[s][j] = MODE == PHX_QUANT_RMS_NORM ? u * scale * a[j] : (MODE == PHX_QUANT_SILU_MUL ? silu_ref(u) : gelu_near(u)) * a[j];
                if (MODE == PHX_QUANT_GELU_MUL && u != u) v[s][j] = u;  // gelu_near has 0 there
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) am = max(am, __float_as_uint(v[s][j]) & 0x7FFFFFFFu);  // the last values again are no more
    }
    am = wave_max_u32(am);
    if (NW > 1) {
        if (lane == 0) redu[wave] = am;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) am = max(am, redu[w]);
    }
    const RowScale rs = row_scale(am);
    if (tid == 0) d[row] = rs.d;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int i = (s * NT + tid) * 8;
        if (i >= n) continue;
        int q[8];
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = quant_one(v[s][j], rs.inv);
        *(uint2*)(qs + row * n + i) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    }
}

template <int NT, int STEPS, int MODE, int DT>
static void quant_as(hipStream_t st, int rows, int n, int64_t ld, float eps, const void* x, const void* aux, int8_t* qs,
                     float* d)
{
    constexpr int RPB = NT < 256 ? 256 / NT : 1;
    launch(k_quant_i8<NT, STEPS, MODE, DT>, dim3((rows + RPB - 1) / RPB), dim3(NT * RPB), 0, st, rows, n, ld, eps, x, aux, qs, d);
}

// a wave a row up to 1024 values, and up to 2048 where the rows are many (16384 of 1408: 63 us with the product behind it,
// four waves a row 91; 256: 17 against 16)
template <int MODE, int DT>
static void quant_rows(hipStream_t st, int rows, int n, int64_t ld, float eps, const void* x, const void* aux, int8_t* qs,
                       float* d)
{
    if (n <= 1024) quant_as<64, 2, MODE, DT>(st, rows, n, ld, eps, x, aux, qs, d);
    else if (n <= 2048 && rows >= 1024) quant_as<64, 4, MODE, DT>(st, rows, n, ld, eps, x, aux, qs, d);
    else if (n <= 4096) quant_as<256, 2, MODE, DT>(st, rows, n, ld, eps, x, aux, qs, d);
    else if (n <= 8192) quant_as<512, 2, MODE, DT>(st, rows, n, ld, eps, x, aux, qs, d);
    else quant_as<1024, 8, MODE, DT>(st, rows, n, ld, eps, x, aux, qs, d);
}

template <int DT>
static void quant_mode(hipStream_t st, int mode, int rows, int n, int64_t ld, float eps, const void* x, const void* aux, int8_t* qs,
                       float* d)
{
    switch (mode) {
    case PHX_QUANT_SILU_MUL: quant_rows<PHX_QUANT_SILU_MUL, DT>(st, rows, n, ld, eps, x, aux, qs, d); break;
    case PHX_QUANT_RMS_NORM: quant_rows<PHX_QUANT_RMS_NORM, DT>(st, rows, n, ld, eps, x, aux, qs, d); break;
    case PHX_QUANT_GELU_MUL: quant_rows<PHX_QUANT_GELU_MUL, DT>(st, rows, n, ld, eps, x, aux, qs, d); break;
    default: quant_rows<PHX_QUANT_PLAIN, DT>(st, rows, n, ld, eps, x, aux, qs, d);
    }
}

void launch_quant_i8(hipStream_t st, int mode, int type, int rows, int n, int64_t ld, float eps, const void* x,
                     const void* aux, int8_t* qs, float* d)
{
    switch (type) {
    case PHX_F16: quant_mode<PHX_F16>(st, mode, rows, n, ld, eps, x, aux, qs, d); break;
    case PHX_BF16: quant_mode<PHX_BF16>(st, mode, rows, n, ld, eps, x, aux, qs, d); break;
    default: quant_mode<PHX_F32>(st, mode, rows, n, ld, eps, x, aux, qs, d);
    }
}

// ------------------------------------------------------------------------------ weights
// I8Mat's layout from matrices as the caller holds them: a thread writes 16 columns of one stored row, zeros past the
// last row or column.
__global__ __launch_bounds__(256) void k_i8_pack(I8Mat m, int m0, int64_t n16, const int8_t* __restrict__ w,
                                                 const float* __restrict__ scale)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n16) return;
    const int s32 = (int)(i & 31), kc = (int)((i >> 5) % m.kc);
    const int64_t g = (i >> 5) / m.kc;  // 32-row group over the matrices from m0
    const int rg = (int)(g % m.rg), mi = (int)(g / m.rg);
    const int half = m.rows / 2;
    int r = rg * 32 + s32;
    if (m.paired) r = (rg >> 1) * 32 + s32 + (rg & 1) * half;
    const bool live = r < m.rows && (!m.paired || (rg >> 1) * 32 + s32 < half);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (live && kc * 16 < m.cols) {
        const int8_t* p = w + ((int64_t)mi * m.rows + r) * m.cols + kc * 16;
        if (((uintptr_t)w & 15) == 0) v = *(const uint4*)p;
        else {
            uint32_t u[4];
            for (int j = 0; j < 4; j++) u[j] = pack4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
            v = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    *(uint4*)(m.w + (int64_t)m0 * m.mat_bytes() + i * 16) = v;
    if (kc == 0) m.scale[((int64_t)m0 * m.rg + g) * 32 + s32] = live ? scale[(int64_t)mi * m.rows + r] : 0.0f;
}

void launch_i8_pack(hipStream_t st, const I8Mat& m, int m0, int n_mat, const int8_t* w, const float* scale)
{
    const int64_t n16 = (int64_t)n_mat * m.mat_bytes() / 16;
    launch(k_i8_pack, dim3((unsigned)((n16 + 255) / 256)), dim3(256), 0, st, m, m0, n16, w, scale);
}

// ------------------------------------------------------------------------------ products
// The tile of a workgroup: cnt rows of one matrix, the list's places start .. start + cnt - 1 (without a list those rows
// themselves).  False past the last tile.
__device__ __forceinline__ bool i8_tile(const I8Args& g, int tile, Tile* tl)
{
    if (g.ids) {  // a tile per assignment, those without an expert empty
        *tl = {g.ids[tile], tile, 1};
        return (unsigned)tl->e < (unsigned)g.n_expert;
    }
    if (!g.tiles) {
        tl->e = 0;
        tl->start = tile * g.cap;
        tl->cnt = min(g.cap, g.nrows - tl->start);
        return tl->cnt > 0;
    }
    if (tile >= *g.ntiles) return false;
    *tl = g.tiles[tile];
    return true;
}

// Place i's output row as a byte offset from out_base (a tile's dense rows, or a list's whole output, lie within 2^32
// bytes), and its input row's scale.  Past the tile's end the last row again: its product is then computed, and stored,
// more than once, the same value to the same place.
template <int DT>
__device__ __forceinline__ void tile_rows(const I8Args& g, const Tile& tl, int i, uint32_t* orow, float* dxs)
{
    const int p = min(i, tl.cnt - 1), a = g.perm ? g.perm[tl.start + p] : tl.start + p;
    orow[i] = (uint32_t)(g.perm ? a : p) * (uint32_t)g.out_cols * (DT == PHX_F32 ? 4u : 2u);
    dxs[i] = g.xd[a / g.div];
}
template <int DT>
__device__ __forceinline__ char* out_base(const I8Args& g, const Tile& tl)
{
    return (char*)g.out + (g.perm ? 0 : (int64_t)tl.start * g.out_cols * (DT == PHX_F32 ? 4 : 2));
}

// v_mfma_i32_32x32x32_i8: lane l holds 16 bytes of A row l % 32 and of B row l % 32, both at k = 16 (l / 32); the
// result D[i][j] sits in lane j + 32 ((i / 4) % 2), register 4 (i / 8) + i % 4.  Tokens are A, weight rows B, so a
// register's 32 lanes store 32 consecutive outputs of one token.
//
// v_mfma_i32_16x16x64_i8 is the same on 16 rows: lane l holds row l % 16 at k = 16 (l / 16), and D[i][j] sits in lane
// j + 16 (i / 4), register i % 4.
//
// k_i8_rows: for few rows per matrix, where the weights' bytes are the time.  A workgroup takes RT tiles of 16 weight rows
// (PAIRED: of 16 channels, their gate and up rows) by a tile of up to 16 TT tokens, both straight from memory to registers:
// its NW waves split the reduction, so no operand is wanted by two of them, and a matrix of few rows still has loads in
// flight everywhere.  A wave keeps U steps of 64 columns ahead; the waves' int32 sums meet in LDS by atomic additions (exact
// in any order).
template <int NW, int RT, int TT, bool PAIRED, bool ONCE, int DT>
__device__ __forceinline__ void i8_rows_product(const I8Args& g, const Tile& tl, int* red, uint32_t* orow, float* dxs)
{
    constexpr int NB = PAIRED ? 2 : 1, NR = RT * NB, U = NR + TT <= 3 ? 8 : NR + TT <= 6 ? 4 : NR + TT <= 8 ? 3 : 2;
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bx = blockIdx.x, tiles16 = g.rgs * 2 / NB;  // the matrix's row (channel) tiles of 16
    const int8_t* xr[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
        const int at = tl.start + min(16 * t + r16, tl.cnt - 1);
        xr[t] = g.xq + (int64_t)((g.perm ? g.perm[at] : at) / g.div) * g.cols;
    }
    const int8_t* wb[NR];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int i = min(bx * RT + r, tiles16 - 1);
            wb[r * NB + b] = g.w + (int64_t)tl.e * g.mat_bytes + ((int64_t)(i >> 1) * NB + b) * g.kc * 512 + (i & 1) * 256;
        }
    const int lo = q * 512 + r16 * 16;
    // the epilogue's: a thread keeps one column, C threads a token, P tokens at a time
    constexpr int C = RT * 16, P = 64 * NW / C;
    const int c = tid % C, col = bx * C + c;
    float sg = 0.0f, su = 0.0f;
    if (col < g.out_cols) {
        const float* sc = g.scale + (int64_t)tl.e * g.mat_scales + (col >> 5) * NB * 32 + (col & 31);
        sg = sc[0];
        if (PAIRED) su = sc[32];
    }
    if (tid < TT * 16) tile_rows<DT>(g, tl, tid, orow, dxs);
    for (int o = tid; o < NR * TT * 256; o += 64 * NW) red[o] = 0;
    i32x4 acc[TT][NR], w[U][NR], x[U][TT];
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < NR; r++) acc[t][r] = i32x4{0, 0, 0, 0};
    const int steps = g.kc / 4, s0 = wave * steps / NW, s1 = (wave + 1) * steps / NW;
    auto load = [&](int u, int s) {
        const int su = min(s, s1 - 1), k = 64 * su + 16 * q, kx = k < g.cols ? k : 0;  // the weights past cols are zero
#pragma unroll
        for (int r = 0; r < NR; r++) w[u][r] = load_weights<ONCE>(wb[r] + (int64_t)su * 2048 + lo);
#pragma unroll
        for (int t = 0; t < TT; t++) x[u][t] = *(const i32x4*)(xr[t] + kx);
    };
    auto mma = [&](int u) {
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < NR; r++)
                acc[t][r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[u][t], w[u][r], acc[t][r], 0, 0, 0);
    };
    if (s0 < s1) {  // uniform over the wave
#pragma unroll
        for (int u = 0; u < U; u++) load(u, s0 + u);
        int s = s0;
        for (; s + U < s1; s += U)
#pragma unroll
            for (int u = 0; u < U; u++) {
                mma(u);
                load(u, s + u + U);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (s + u < s1) mma(u);
    }
    __syncthreads();  // the zeros are there
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int v = 0; v < 4; v++) atomicAdd(&red[((t * NR + r) * 4 + v) * 64 + lane], acc[t][r][v]);
    __syncthreads();
    if (col >= g.out_cols) return;
    char* out = out_base<DT>(g, tl);
#pragma unroll
    for (int it = 0; it < (TT * 16 + P - 1) / P; it++) {
        const int tok = it * P + tid / C, i = tok & 15;
        if (tok >= tl.cnt) break;
        const int at = (((tok >> 4) * NR + (c >> 4) * NB) * 4 + (i & 3)) * 64 + (c & 15) + 16 * (i >> 2);
        float y = (float)red[at] * (dxs[tok] * sg);
        if (PAIRED) y = gated_kept(g.act, y, (float)red[at + 256] * (dxs[tok] * su));
        store_one<DT>(out + orow[tok], col, y);
    }
}

// CT: the most token tiles of 16 that a tile may hold (its capacity); a tile takes the product of its own count
template <int NW, int RT, int CT, bool PAIRED, bool ONCE, int DT>
__global__ __launch_bounds__(64 * NW) void k_i8_rows(I8Args g)
{
    __shared__ int red[RT * CT * (PAIRED ? 2 : 1) * 256];
    __shared__ uint32_t orow[CT * 16];
    __shared__ float dxs[CT * 16];
    Tile tl;
    if (!i8_tile(g, blockIdx.y, &tl)) return;  // uniform over the workgroup
    const int n = (tl.cnt + 15) / 16;
    if (CT == 1 || n == 1) i8_rows_product<NW, RT, 1, PAIRED, ONCE, DT>(g, tl, red, orow, dxs);
    else if (CT == 2 || n == 2) i8_rows_product<NW, RT, CT < 2 ? 1 : 2, PAIRED, ONCE, DT>(g, tl, red, orow, dxs);
    else if (CT == 4 || n <= 4) i8_rows_product<NW, RT, CT < 4 ? 1 : 4, PAIRED, ONCE, DT>(g, tl, red, orow, dxs);
    else i8_rows_product<NW, RT, CT < 8 ? 1 : 8, PAIRED, ONCE, DT>(g, tl, red, orow, dxs);
}

// The down products of few assignments and their weighted sum, for a token (blockIdx.y) and 16 of its outputs: wave w takes
// the token's places w, w + NW, ...  It issues the place's weights, forms the int8 row of its h meanwhile (every
// workgroup of the token forms it again: nf floats from L2), and the places' values meet in LDS in order.  No lists, no
// int8 rows and no partial outputs go through memory.  Bound by its chains of dependent trips (ids, h twice, the weights; at the
// end the id and the weight of each place in turn): 6.8 to 8.1 us for one token of 8 x 704, d = 2816, whose 16 MB take 2.5.
template <int NW, int DT>
__global__ __launch_bounds__(64 * NW) void k_i8_down_few(I8Args g, int k, int nf, const float* __restrict__ h,
                                                         const float* __restrict__ weights)
{
    extern __shared__ __align__(16) int8_t rows[];  // [NW][kc * 16]
    __shared__ float vals[PHX_MAX_USED][16];
    constexpr int U = 12;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4, bx = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = blockIdx.y;
    const int steps = g.kc / 4;
    int8_t* row = rows + wave * g.kc * 16;
    for (int j = wave; j < k; j += NW) {
        const int e = g.ids[t * k + j];  // uniform
        if ((unsigned)e >= (unsigned)g.n_expert) continue;
        const int8_t* wb = g.w + (int64_t)e * g.mat_bytes + (int64_t)(bx >> 1) * g.kc * 512 + (bx & 1) * 256 + q * 512 + r16 * 16;
        i32x4 w[U];
        auto load = [&](int s) {
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = *(const i32x4*)(wb + (int64_t)min(s + u, steps - 1) * 2048);
        };
        load(0);
        __builtin_amdgcn_sched_barrier(0);
        const float* hr = h + (t * k + j) * nf;
        unsigned am = 0;
        for (int i = lane * 4; i < nf; i += 256) {
            const uint4 v = *(const uint4*)(hr + i);
            am = max(max(am, v.x & 0x7FFFFFFFu), max(max(v.y & 0x7FFFFFFFu, v.z & 0x7FFFFFFFu), v.w & 0x7FFFFFFFu));
        }
        const RowScale rs = row_scale(wave_max_u32(am));
        for (int i = lane * 4; i < g.kc * 16; i += 256) {
            uint32_t p = 0;
            if (i < nf) {
                const float4 v = *(const float4*)(hr + i);
                p = pack4(quant_one(v.x, rs.inv), quant_one(v.y, rs.inv), quant_one(v.z, rs.inv), quant_one(v.w, rs.inv));
            }
            *(uint32_t*)(row + i) = p;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        i32x4 acc = {0, 0, 0, 0};
        for (int s = 0; s < steps; s += U) {
            if (s) load(s);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (s + u < steps)  // uniform
                    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(row + 64 * (s + u) + 16 * q), w[u], acc, 0, 0, 0);
        }
        if (lane < 16) {
            const float dw = g.scale[(int64_t)e * g.mat_scales + bx * 16 + lane];
            vals[j][lane] = (float)acc[0] * (rs.d * dw);
        }
        // this wave's reads of the row end before the next place's writes
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    __syncthreads();
    const int col = bx * 16 + threadIdx.x;
    if (threadIdx.x < 16 && col < g.out_cols) {
        float acc = 0.0f;
        for (int j = 0; j < k; j++)
            if ((unsigned)g.ids[t * k + j] < (unsigned)g.n_expert) acc += vals[j][threadIdx.x] * weights[t * k + j];
        store_one<DT>(g.out, t * g.out_cols + col, acc);
    }
}

// k_i8_tile: four waves, each 64 stored weight rows (PAIRED: the gate and up rows of 32 channels), by a tile of up to 128
// tokens.  The weights go straight from memory to each wave's registers (the layout has every operand as one run of
// 1 KB, and no other wave of the workgroup wants it), one 128-column step ahead; the tokens, which all four waves read, go
// through an LDS ring by direct loads two steps ahead, row-major runs of 128 bytes with the 16-byte chunks XOR-swizzled by
// half the row's number: LDS serves a 16-byte read in four turns of 16 lanes, {0-3, 12-15, 20-27}, {4-11, 16-19, 28-31} and the
// same from lane 32, over 64 banks, and each turn then has 16 distinct bank groups (by the row's number itself, two rows of
// a turn share one: 8 cycles a read against 4).
//
// What it reaches: 8192 x 5632 x 4096 173 to 195 us by the clock, 1.9 to 2.2 POP/s (a library product of that size 181); T = 2048 of
// 4096 x 4096 30 to 35 us.  Under 256 workgroups the time is one workgroup's chain: 4096 x 4096 takes 24 us from T = 129 to 512.  The
// matrix cores run in 60% of a tile's cycles at the 2.0 GHz that they leave the clock; without any load from memory a step
// takes 1.13 us against 1.5, the rest is the issue and the wait of the loads.  Two 128-token halves on eight waves that share
// the weights in the L1 (experts, T = 2048: gate|up 176 -> 197 us), four ring slots (the same), wave priorities (the same) and
// experts' tiles longest first (297 -> 316 us: an expert's tiles no longer meet in the caches) were no faster.
constexpr int TI_RING = 3, TI_PITCH = 68;  // ring slots; ints between two tokens' rows of 64 in the epilogue

template <int NT, bool PAIRED, bool ONCE, int DT>
__device__ __forceinline__ void i8_tile_product(const I8Args& g, const Tile& tl, int bx, unsigned char* ring, uint32_t* orow, float* dxs)
{
    constexpr int STAGE = NT * 32 * 128;
    const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = g.kc / 8;
    // this lane's rows of the direct loads: one per load, the last row again past the tile's end
    const int chunk = ((lane & 7) ^ (lane >> 4)) * 16;  // of the loads whose first row is a multiple of 16; 4 chunks on for 8
    const __amdgpu_buffer_rsrc_t rsrc = buf_rsrc(g.xq + (g.perm ? 0 : (int64_t)tl.start * g.cols));
    uint32_t xr[NT];  // a list's rows lie within 2^32 bytes of xq (phx_experts_i8's chunks), a dense tile's of its first
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int at = min(8 * (wave * NT + i) + (lane >> 3), tl.cnt - 1);
        xr[i] = (uint32_t)(g.perm ? g.perm[tl.start + at] / g.div : at) * (uint32_t)g.cols;
    }
    if (tid < NT * 32) tile_rows<DT>(g, tl, tid, orow, dxs);
    int slot = 0, slot1 = STAGE, slot2 = 2 * STAGE;  // the ring's slots of a step and the two after it
    auto dma = [&](int s, int to, auto I) {          // load I of step s's rows
        constexpr int i = decltype(I)::value;
        const uint32_t off = min(s, S - 1) * 128 + (chunk ^ (64 * ((wave * NT + i) & 1)));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t)(ring + to + (wave * NT + i) * 1024), 16,
                                                 xr[i] + (off < (uint32_t)g.cols ? off : 0), 0, 0, 0);  // the weights past cols are zero
    };
    const int rg0 = (bx * 4 + wave) * 2, rgs = g.rgs;
    const int8_t* wb[2];
#pragma unroll
    for (int b = 0; b < 2; b++)
        wb[b] = g.w + (int64_t)tl.e * g.mat_bytes + (int64_t)min(rg0 + b, rgs - 1) * g.kc * 512;
    const uint32_t lane16 = lane * 16;
    i32x4 wv[2][2][4];
    auto weight = [&](int s, int b, auto P, auto KK) {
        const int8_t* at = wb[b] + (int64_t)min(s, S - 1) * 4096 + decltype(KK)::value * 1024;  // uniform
        wv[decltype(P)::value][b][decltype(KK)::value] = load_weights<ONCE>(at + lane16);
    };
    i32x16 acc[NT][2];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[j][b][v] = 0;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void_t)ring + r32 * 128, swz = (h ^ ((r32 >> 1) & 7)) * 16;
    u32x4 a[2][NT];
    auto read = [&](int from, auto KK) {
        constexpr int kk = decltype(KK)::value;
        const uint32_t ad = lds + from + (swz ^ (kk * 32));
        static_for<NT>([&](auto J) { a[kk & 1][decltype(J)::value] = ds_r128<decltype(J)::value * 4096>(ad); });
    };
    auto landed = [&](auto Q) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int j = 0; j < NT; j++) tie(a[decltype(Q)::value][j]);
    };
    // A step is four groups of products on 32 columns.  A group first reads the next one's tokens (the last: the next step's,
    // once its rows have landed in every wave, which also says that nobody reads this step's slot any more), and among its
    // products issues the loads: the weights that the group before has just used the registers of, two steps on, and
    // one load of the rows two steps on.  The order is fixed by scheduling barriers: the wait for the rows counts the loads
    // issued after them.
    constexpr int NEWER = 6 + (NT < 3 ? NT : 3) + 2 * (4 - NT);
    auto step = [&](int s, auto P) {
        constexpr int p = decltype(P)::value;
        static_for<4>([&](auto KK) {
            constexpr int kk = decltype(KK)::value;
            if constexpr (kk < 3) read(slot, ic<kk + 1>{});
            else {
                __builtin_amdgcn_s_waitcnt(vm_wait(NEWER));
                __builtin_amdgcn_s_barrier();
                read(slot1, ic<0>{});
            }
            static_for<2 * NT>([&](auto M) {
                constexpr int m = decltype(M)::value, j = m / 2, b = m % 2;
                __builtin_amdgcn_sched_barrier(0);
                acc[j][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a[kk & 1][j]), wv[p][b][kk], acc[j][b],
                                                                  0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (m == 0 || m == 1) {
                    if constexpr (kk == 0) weight(s + 1, m, ic<1 - p>{}, ic<3>{});
                    else weight(s + 2, m, ic<p>{}, ic<kk - 1>{});
                }
                if constexpr (m == (NT > 1 ? 3 : 1)) {
                    if constexpr (kk < NT) dma(s + 2, slot2, ic<kk < NT ? kk : 0>{});
                }
            });
            __builtin_amdgcn_sched_barrier(0);
            landed(ic<(kk + 1) & 1>{});
        });
        const int done = slot;
        slot = slot1;
        slot1 = slot2;
        slot2 = done;
    };
    static_for<NT>([&](auto I) { dma(0, slot, I); });
    static_for<NT>([&](auto I) { dma(1, slot1, I); });
    static_for<4>([&](auto KK) {
        weight(0, 0, ic<0>{}, KK);
        weight(0, 1, ic<0>{}, KK);
    });
    static_for<3>([&](auto KK) {
        weight(1, 0, ic<1>{}, KK);
        weight(1, 1, ic<1>{}, KK);
    });
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(vm_wait(NT + 14));
    __builtin_amdgcn_s_barrier();
    read(slot, ic<0>{});
    landed(ic<0>{});
    for (int s = 0; s + 1 < S; s += 2) {
        step(s, ic<0>{});
        step(s + 1, ic<1>{});
    }
    if (S & 1) step(S - 1, ic<0>{});
    __builtin_amdgcn_s_waitcnt(0);  // the direct loads past the last step land before the workgroup's LDS goes
    __syncthreads();
    char* out = out_base<DT>(g, tl);
    const float* sc = g.scale + (int64_t)tl.e * g.mat_scales;
    // Each 32 tokens' sums go through the wave's own part of the ring, so that a lane stores 16 bytes of one token's row: straight
    // from the accumulators an instruction stores 4 or 2 bytes a lane, and the stores alone took a third of the time.
    constexpr int V = DT == PHX_F32 ? 4 : 8, WC = PAIRED ? 32 : 64, LPT = WC / V, TPI = 64 / LPT;  // lanes a token, tokens a round
    int* mine = (int*)ring + wave * 32 * TI_PITCH;
    const int col0 = PAIRED ? (rg0 >> 1) * 32 : rg0 * 32, c = (lane % LPT) * V, col = col0 + c;
    float dw[V], du[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int r = min(rg0 * 32 + c + i, rgs * 32 - 1);
        dw[i] = sc[r];
        du[i] = PAIRED ? sc[min(r + 32, rgs * 32 - 1)] : 0.0f;
    }
    const bool whole = g.out_cols % V == 0;  // rows and columns then start on 16 bytes
    __builtin_amdgcn_s_waitcnt(0);           // the scales: a later wait for them would wait for the stores before it too
#pragma unroll
    for (int j = 0; j < NT; j++) {
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int v = 0; v < 16; v++) mine[(8 * (v >> 2) + 4 * h + (v & 3)) * TI_PITCH + 32 * b + r32] = acc[j][b][v];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // two rounds at a time: a workgroup runs this once, and unrolled further the instructions take longer to fetch than to run
#pragma unroll 2
        for (int it = 0; it < 32 / TPI; it++) {
            const int tok = it * TPI + lane / LPT;
            const float dx = dxs[32 * j + tok];
            char* o = out + orow[32 * j + tok];
            int s[V], u[V];
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                *(int4*)(s + i) = *(const int4*)(mine + tok * TI_PITCH + c + i);
                if (PAIRED) *(int4*)(u + i) = *(const int4*)(mine + tok * TI_PITCH + 32 + c + i);
            }
            float y[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                y[i] = (float)s[i] * (dx * dw[i]);
                if (PAIRED) y[i] = gated_kept(g.act, y[i], (float)u[i] * (dx * du[i]));
            }
            if (whole) {
                if (col < g.out_cols) store_16<DT>(o, col, y);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (col + i < g.out_cols) store_one<DT>(o, col + i, y[i]);
            }
        }
        // this tile's reads end before the next one's writes
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <bool PAIRED, bool ONCE, int DT>
__global__ __launch_bounds__(256, 2) void k_i8_tile(I8Args g)
{
    __shared__ __align__(16) unsigned char ring[TI_RING * 128 * 128];
    static_assert(sizeof(ring) >= 4 * 32 * TI_PITCH * 4, "the epilogue's part of each wave");
    __shared__ __align__(16) uint32_t orow[128];
    __shared__ __align__(16) float dxs[128];
    // Workgroup L runs on XCD L % 8.  The XCDs share the tiles in xt parts and the row blocks in 8 / xt; an XCD takes runs of
    // tiles of its part, and of a run's row blocks by tiles 8 row blocks at a time, tile by tile: what it runs together
    // shares few rows of both operands in its L2.
    const int L = blockIdx.x, k = L >> 3, xcd = L & 7, per = g.run * g.blocks, in = k % per;
    const int band = in / (8 * g.run), wide = min(8, g.blocks - 8 * band), at = in - band * 8 * g.run;
    const int tile = ((k / per) * g.xt + xcd % g.xt) * g.run + at / wide, bx = xcd / g.xt * g.blocks + band * 8 + at % wide;
    if (bx * 8 >= g.rgs) return;
    Tile tl;
    if (!i8_tile(g, tile, &tl)) return;  // uniform over the workgroup
    switch ((tl.cnt + 31) / 32) {
    case 1: i8_tile_product<1, PAIRED, ONCE, DT>(g, tl, bx, ring, orow, dxs); break;
    case 2: i8_tile_product<2, PAIRED, ONCE, DT>(g, tl, bx, ring, orow, dxs); break;
    case 3: i8_tile_product<3, PAIRED, ONCE, DT>(g, tl, bx, ring, orow, dxs); break;
    default: i8_tile_product<4, PAIRED, ONCE, DT>(g, tl, bx, ring, orow, dxs);
    }
}

static void set_matrix(I8Args& g, const I8Mat& m)
{
    g.w = m.w;
    g.scale = m.scale;
    g.mat_bytes = m.mat_bytes();
    g.mat_scales = (int64_t)m.rg * 32;
    g.kc = m.kc;
    g.cols = m.cols;
    g.out_cols = m.paired ? m.rows / 2 : m.rows;
    g.rgs = m.rg;
    g.n_expert = m.n_mat;
}

template <int NW, int RT, int CT>
static void rows_dense(hipStream_t st, const I8Args& g, int max_tiles, int out_type)
{
    const dim3 grid((g.out_cols + 16 * RT - 1) / (16 * RT), max_tiles), blk(64 * NW);
    if (out_type == PHX_F16) launch(k_i8_rows<NW, RT, CT, false, false, PHX_F16>, grid, blk, 0, st, g);
    else if (out_type == PHX_BF16) launch(k_i8_rows<NW, RT, CT, false, false, PHX_BF16>, grid, blk, 0, st, g);
    else launch(k_i8_rows<NW, RT, CT, false, false, PHX_F32>, grid, blk, 0, st, g);
}

template <int NW, int RT, int CT, bool PAIRED, bool ONCE>
static void rows_float(hipStream_t st, const I8Args& g, int max_tiles)
{
    const dim3 grid((g.out_cols + 16 * RT - 1) / (16 * RT), max_tiles), blk(64 * NW);
    launch(k_i8_rows<NW, RT, CT, PAIRED, ONCE, PHX_F32>, grid, blk, 0, st, g);
}

// 32 channels, 64 outputs a workgroup: 64 experts of d = 4096, nf = 1408, T = 24 127 us; 64 channels 136, 32 outputs 125;
// 128 of 2816, 704, T = 128: 148; 16 channels 158, 32 outputs 156 (all before weights read once passed the caches by, with
// which the two kept forms take 114 and 139)
template <int CT, bool ONCE>
static void rows_lists(hipStream_t st, const I8Mat& m, const I8Args& g, int max_tiles)
{
    if (m.paired) rows_float<4, 2, CT, true, ONCE>(st, g, max_tiles);
    else rows_float<4, 4, CT, false, ONCE>(st, g, max_tiles);
}

template <bool ONCE>
static void rows_by_cap(hipStream_t st, const I8Mat& m, const I8Args& g, int max_tiles)
{
    if (g.cap <= 16) rows_lists<1, ONCE>(st, m, g, max_tiles);
    else if (g.cap <= 32) rows_lists<2, ONCE>(st, m, g, max_tiles);
    else rows_lists<4, ONCE>(st, m, g, max_tiles);
}

void launch_i8_product(hipStream_t st, const I8Mat& m, I8Args g, bool tile, int max_tiles, int ncu, int out_type)
{
    set_matrix(g, m);
    if (tile) {
        // Lists: every XCD takes pairs of tiles and all their row blocks (64 experts of d = 4096, nf = 1408, T = 4096: gate|up
        // 275 us, tile by tile 304).  A pair starts at an even tile whatever its expert: of the tiles that follow one of the same
        // expert about half fall into the next pair, on another XCD, and read the expert's weights from memory again.  A dense
        // product: the split with the fewest workgroups on an XCD, and of those the one that brings the fewest bytes to the
        // XCDs, each its tiles' tokens and its blocks' weights.
        const int blocks = (m.rg + 7) / 8;
        g.xt = 8;
        g.run = 2;
        if (!g.tiles) {
            int64_t least = INT64_MAX;
            for (int xt = 1; xt <= 8; xt *= 2) {
                const int64_t t = (max_tiles + xt - 1) / xt, b = (blocks + 8 / xt - 1) / (8 / xt);
                const int64_t cost = (t * b << 32) + t * xt * kI8Tile * (8 / xt) + b * (8 / xt) * 256 * xt;
                if (cost < least) {
                    least = cost;
                    g.xt = xt;
                    g.run = (int)t;
                }
            }
        }
        g.blocks = (blocks + 8 / g.xt - 1) / (8 / g.xt);
        const int per = g.xt * g.run;
        const dim3 grid((max_tiles + per - 1) / per * g.run * g.blocks * 8), blk(256);
        if (m.paired && g.once) launch(k_i8_tile<true, true, PHX_F32>, grid, blk, 0, st, g);
        else if (m.paired) launch(k_i8_tile<true, false, PHX_F32>, grid, blk, 0, st, g);
        else if (g.once) launch(k_i8_tile<false, true, PHX_F32>, grid, blk, 0, st, g);
        else if (out_type == PHX_F16) launch(k_i8_tile<false, false, PHX_F16>, grid, blk, 0, st, g);
        else if (out_type == PHX_BF16) launch(k_i8_tile<false, false, PHX_BF16>, grid, blk, 0, st, g);
        else launch(k_i8_tile<false, false, PHX_F32>, grid, blk, 0, st, g);
    } else if (!g.tiles && !g.ids) {
        if (g.cap <= 16) rows_dense<8, 1, 1>(st, g, max_tiles, out_type);
        else if (g.cap <= 32) rows_dense<8, 1, 2>(st, g, max_tiles, out_type);
        else {
            // Row tiles of 16 until their workgroups number two per compute unit, of 32 to four, then of 64 where the tokens are
            // past 64 (us by tiles of 16, 32, 64; 2816 columns, T = 96): 4096 outputs 12.7, 13.4, 17.3; 8192 23.6, 13.7, 17.6;
            // 16384 45.0, 25.4, 19.1.  T = 64: 4096 10.6, 11.3; 8192 19.6, 11.6.  In between the rule is not the best: 12288
            // outputs, T = 96, take tiles of 32 and 25.2 us, of 64 18.1.
            const int64_t n = (int64_t)((g.out_cols + 15) / 16) * max_tiles;
            if (g.cap <= 64) {
                if (n < 2 * ncu) rows_dense<8, 1, 4>(st, g, max_tiles, out_type);
                else rows_dense<8, 2, 4>(st, g, max_tiles, out_type);
            } else if (n < 2 * ncu) rows_dense<8, 1, 8>(st, g, max_tiles, out_type);
            else if (n < 4 * ncu) rows_dense<8, 2, 8>(st, g, max_tiles, out_type);
            else rows_dense<8, 4, 8>(st, g, max_tiles, out_type);
        }
    } else if (g.ids) {
        // Single assignments: paired matrices only (launch_i8_down_few takes the others).  8 waves on 16 channels until these
        // workgroups number four per compute unit, then 4 waves on 32 (us, 8 waves first): 128 experts of d = 2816, nf = 704,
        // T = 1 16.0, 15.8; T = 2 22.9, 24.3; T = 4 42.0 either way; 32 of 1024, 512, k = 4: T = 4 11.6, 10.7; T = 8 15.5, 12.7.
        if ((int64_t)((g.out_cols + 15) / 16) * max_tiles < 4 * ncu) rows_float<8, 1, 1, true, false>(st, g, max_tiles);
        else rows_float<4, 2, 1, true, false>(st, g, max_tiles);
    } else if (g.once) rows_by_cap<true>(st, m, g, max_tiles);
    else rows_by_cap<false>(st, m, g, max_tiles);
}

template <int NW>
static void down_few(hipStream_t st, const I8Args& g, int T, int k, int nf, const float* h, const float* weights, int out_type)
{
    const dim3 grid((g.out_cols + 15) / 16, T), blk(64 * NW);
    const uint32_t lds = NW * g.kc * 16;
    if (out_type == PHX_F16) launch(k_i8_down_few<NW, PHX_F16>, grid, blk, lds, st, g, k, nf, h, weights);
    else if (out_type == PHX_BF16) launch(k_i8_down_few<NW, PHX_BF16>, grid, blk, lds, st, g, k, nf, h, weights);
    else launch(k_i8_down_few<NW, PHX_F32>, grid, blk, lds, st, g, k, nf, h, weights);
}

bool i8_down_few_fits(const I8Mat& m) { return 8 * m.kc * 16 <= 61440; }  // its rows and values in 64 KB of LDS

void launch_i8_down_few(hipStream_t st, const I8Mat& m, int T, int k, const float* h, const int* ids, const float* weights,
                        int out_type, void* out)
{
    I8Args g{};
    set_matrix(g, m);
    g.ids = ids;
    g.out = out;
    if (k <= 4) down_few<4>(st, g, T, k, m.cols, h, weights, out_type);
    else down_few<8>(st, g, T, k, m.cols, h, weights, out_type);
}

// ------------------------------------------------------------------------------ experts
// Each expert's assignments as one run of perm and as tiles of up to cap; ids outside [0, E) are in no run.  One workgroup
// takes up to 1024 IPT assignments: an id's place in its run is what its counter's atomic addition returns, kept in a
// register, and the runs are put together in LDS and stored whole.  The order inside a run is the atomics' and no result
// depends on it: a place of the list names its own input and output row.  One compute unit's latency bounds it: 4.5 us to
// 2048 assignments, 8.8 for 16384, whose 16 loads a thread go out in one trip (waited for one by one: 14 us).
template <int IPT>
__global__ __launch_bounds__(1024) void k_i8_lists(int n, int E, int cap, const int* __restrict__ ids, int* __restrict__ perm,
                                                   Tile* __restrict__ tiles, int* __restrict__ ntiles, int* __restrict__ offsets)
{
    __shared__ int count[PHX_MAX_EXPERTS_DEV], start[PHX_MAX_EXPERTS_DEV], first[PHX_MAX_EXPERTS_DEV], total;
    __shared__ uint16_t list[1024 * IPT];
    const int tid = threadIdx.x;
    if (tid < PHX_MAX_EXPERTS_DEV) count[tid] = 0;
    uint32_t place[IPT];  // expert << 16 | place in its run
#pragma unroll
    for (int i = 0; i < IPT; i++) {
        const int a = i * 1024 + tid;
        const uint32_t e = min((unsigned)ids[min(a, n - 1)], 0xFFFFu);  // every load before the first is waited for
        place[i] = (a < n ? e : 0xFFFFu) << 16;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPT; i++)
        if ((place[i] >> 16) < (unsigned)E) place[i] |= (uint32_t)atomicAdd(&count[place[i] >> 16], 1);
    __syncthreads();
    if (tid < 64) {  // prefix sums over the experts, four to a lane
        int c[4], t[4], sc = 0, stl = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[i] = count[4 * tid + i];
            t[i] = (c[i] + cap - 1) / cap;
            sc += c[i];
            stl += t[i];
        }
        int pc = wave_incl_scan_i(sc) - sc, pt = wave_incl_scan_i(stl) - stl;
        if (tid == 63) {
            if (ntiles) *ntiles = pt + stl;
            total = pc + sc;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            start[4 * tid + i] = pc;
            first[4 * tid + i] = pt;
            pc += c[i];
            pt += t[i];
        }
    }
    __syncthreads();
    if (offsets && tid <= E) offsets[tid] = tid < E ? start[tid] : total;
    if (tiles && tid < E) {
        int at = start[tid], left = count[tid];
        for (int i = first[tid]; left > 0; i++, at += cap, left -= cap) tiles[i] = {tid, at, min(cap, left)};
    }
#pragma unroll
    for (int i = 0; i < IPT; i++)
        if ((place[i] >> 16) < (unsigned)E) list[start[place[i] >> 16] + (place[i] & 0xFFFFu)] = (uint16_t)(i * 1024 + tid);
    __syncthreads();
    for (int p = tid; p < total; p += 1024) perm[p] = list[p];
}

void launch_i8_lists(hipStream_t st, int n, int E, int cap, const int* ids, int* perm, Tile* tiles, int* ntiles, int* offsets)
{
    const dim3 one(1), blk(1024);
    if (n <= 2048) launch(k_i8_lists<2>, one, blk, 0, st, n, E, cap, ids, perm, tiles, ntiles, offsets);
    else if (n <= 16384) launch(k_i8_lists<16>, one, blk, 0, st, n, E, cap, ids, perm, tiles, ntiles, offsets);
    else launch(k_i8_lists<64>, one, blk, 0, st, n, E, cap, ids, perm, tiles, ntiles, offsets);
}

// out[t] = sum over the places j, in order, of w[t][j] * y[t k + j]; places without an expert are skipped.  Bound by y's bytes:
// 2048 tokens of 8 x 2816 floats 33 us, 6.2 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void k_i8_combine(int d, int k, int E, const float* __restrict__ y, const int* __restrict__ ids,
                                                    const float* __restrict__ w, void* __restrict__ out)
{
    const int64_t t = blockIdx.y;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= d) return;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j < k; j++) {
        if ((unsigned)ids[t * k + j] >= (unsigned)E) continue;  // uniform
        const float wj = w[t * k + j];
        const f32x4 v = __builtin_nontemporal_load((const f32x4*)(y + (t * k + j) * d + c));  // read once
        acc.x += v.x * wj;
        acc.y += v.y * wj;
        acc.z += v.z * wj;
        acc.w += v.w * wj;
    }
    store_four<DT>(out, t * d + c, acc);
}

void launch_i8_combine(hipStream_t st, int T, int d, int k, int E, const float* y, const int* ids, const float* w, int out_type,
                       void* out)
{
    const dim3 grid((d + 1023) / 1024, T), blk(256);
    if (out_type == PHX_F16) launch(k_i8_combine<PHX_F16>, grid, blk, 0, st, d, k, E, y, ids, w, out);
    else if (out_type == PHX_BF16) launch(k_i8_combine<PHX_BF16>, grid, blk, 0, st, d, k, E, y, ids, w, out);
    else launch(k_i8_combine<PHX_F32>, grid, blk, 0, st, d, k, E, y, ids, w, out);
}

__global__ __launch_bounds__(256) void k_selftest_gated(int act, int n, const float* __restrict__ a, const float* __restrict__ b,
                                                        float* __restrict__ out)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = gated(act, a[i], b[i]);
}

void launch_selftest_gated(hipStream_t st, int act, int n, const float* a, const float* b, float* out)
{
    launch(k_selftest_gated, dim3((n + 255) / 256), dim3(256), 0, st, act, n, a, b, out);
}

}  // namespace phx
