// The residual's addition and the RMS norm of the sum, as int8 rows with a scale per row and as float rows (phx_add_norm_i8).
#include "device_common.h"
#include "i8_rows.h"
#include "rows_io.h"

namespace phx {

// A float as DT holds it.
template <int DT>
__device__ __forceinline__ float held(float v)
{
    if (DT == PHX_F32) return v;
    if (DT == PHX_F16) return h2f(f2h_of(v));
    return bf2f(f2bf_pair(v, 0.0f) & 0xFFFF);
}

template <int DT>
__device__ __forceinline__ void store_eight(void* p, int64_t i, const float (&v)[8])
{
    if constexpr (DT == PHX_F32) {
        store_16<DT>(p, i, {v[0], v[1], v[2], v[3]});
        store_16<DT>(p, i + 4, {v[4], v[5], v[6], v[7]});
    } else store_16<DT>(p, i, v);
}

// NT threads per row, eight consecutive values per thread and step, the row held in registers from its load to its integers: one
// pass over memory, which bounds it (4099 rows of 4096 bf16 values to bf16 and int8: 151 MB in 35 us, 4.3 TB/s where a copy has 4.7,
// and in 27 where they are still in the last cache; one row of 2816 floats 3.9 us, a launch).  Values past the row are zeros and not the row's last again: sum may lie over x,
// and another wave may have stored there.  The mapping of values to threads, and so every rounding of the sum of squares, is
// phx_quant_i8's.
template <int NT, int STEPS, int DT>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_add_norm_i8(int rows, int n, int64_t ld, float eps, const void* x,
                                                                     const void* __restrict__ branch,
                                                                     const float* __restrict__ w, void* sum, int out_type,
                                                                     void* __restrict__ out, int8_t* __restrict__ qs,
                                                                     float* __restrict__ d)
{
    constexpr int RPB = NT < 256 ? 256 / NT : 1, NW = NT / 64;
    constexpr bool EARLY = STEPS * NT <= 2048;
    __shared__ double red[NW];
    __shared__ unsigned redu[NW];
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
    if (NT == 64 && row >= rows) return;  // a whole wave, and no barrier with one wave a row
    const int tid = threadIdx.x % NT, lane = tid & 63, wave = tid >> 6;
    float v[STEPS][8];
    float a[STEPS][8];  // the norm's weights on their way while the row is summed, where registers hold them
    double sq = 0.0;
    constexpr int AT = STEPS < 4 ? STEPS : 4;  // steps whose loads are in flight together: all eight would spill
#pragma unroll
    for (int s0 = 0; s0 < STEPS; s0 += AT) {
        float b[AT][8];
#pragma unroll
        for (int s = s0; s < s0 + AT; s++) {
            const int i = (s * NT + tid) * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) v[s][j] = b[s - s0][j] = 0.0f;
            if (i < n) {
                load_eight<DT>(x, row * n + i, v[s]);
                load_eight<DT>(branch, row * ld + i, b[s - s0]);
            }
        }
        if (EARLY)
#pragma unroll
            for (int s = 0; s < STEPS; s++) load_eight<PHX_F32>(w, min((s * NT + tid) * 8, n - 8), a[s]);
#pragma unroll
        for (int s = s0; s < s0 + AT; s++) {
            const int i = (s * NT + tid) * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) v[s][j] = held<DT>(v[s][j] + b[s - s0][j]);
            if (i < n) {
                store_eight<DT>(sum, row * n + i, v[s]);
#pragma unroll
                for (int j = 0; j < 8; j++) sq += (double)v[s][j] * (double)v[s][j];
            }
        }
    }
    sq = wave_sum_dpp(sq);
    if (NW > 1) {
        if (lane == 0) red[wave] = sq;
        __syncthreads();
        sq = 0.0;
        for (int i = 0; i < NW; i++) sq += red[i];
    }
    const float scale = rms_scale_from_mean((float)(sq / (double)n), eps);
    unsigned am = 0;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int i = (s * NT + tid) * 8;
        if (i >= n) continue;
        if (!EARLY) load_eight<PHX_F32>(w, i, a[s]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[s][j] = v[s][j] * scale * a[s][j];
            am = max(am, __float_as_uint(v[s][j]) & 0x7FFFFFFFu);
        }
    }
    am = wave_max_u32(am);
    if (NW > 1) {
        if (lane == 0) redu[wave] = am;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; i++) am = max(am, redu[i]);
    }
    const RowScale rs = row_scale(am);
    if (tid == 0) d[row] = rs.d;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int i = (s * NT + tid) * 8;
        if (i >= n) continue;
        if (out) {
            if (out_type == PHX_F16) store_eight<PHX_F16>(out, row * n + i, v[s]);
            else if (out_type == PHX_BF16) store_eight<PHX_BF16>(out, row * n + i, v[s]);
            else store_eight<PHX_F32>(out, row * n + i, v[s]);
        }
        int q[8];
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = quant_one(v[s][j], rs.inv);
        *(uint2*)(qs + row * n + i) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    }
}

template <int NT, int STEPS, int DT>
static void add_norm_as(hipStream_t st, const AddNormArgs& a)
{
    constexpr int RPB = NT < 256 ? 256 / NT : 1;
    launch(k_add_norm_i8<NT, STEPS, DT>, dim3((a.rows + RPB - 1) / RPB), dim3(NT * RPB), 0, st, a.rows, a.n, a.ld, a.eps, a.x,
           a.branch, a.w, a.sum, a.out_type, a.out, a.qs, a.d);
}

// phx_quant_i8's sizes, so that the two give the same bits
template <int DT>
static void add_norm_type(hipStream_t st, const AddNormArgs& a)
{
    if (a.n <= 1024) add_norm_as<64, 2, DT>(st, a);
    else if (a.n <= 2048 && a.rows >= 1024) add_norm_as<64, 4, DT>(st, a);
    else if (a.n <= 4096) add_norm_as<256, 2, DT>(st, a);
    else if (a.n <= 8192) add_norm_as<512, 2, DT>(st, a);
    else if (a.n <= 16384) add_norm_as<1024, 2, DT>(st, a);  // the last one's threads and values, and fewer registers
    else if (a.n <= 32768) add_norm_as<1024, 4, DT>(st, a);
    else add_norm_as<1024, 8, DT>(st, a);
}

void launch_add_norm_i8(hipStream_t st, int type, const AddNormArgs& a)
{
    switch (type) {
    case PHX_F16: add_norm_type<PHX_F16>(st, a); break;
    case PHX_BF16: add_norm_type<PHX_BF16>(st, a); break;
    default: add_norm_type<PHX_F32>(st, a);
    }
}

}  // namespace phx
