// Routing to experts (phx_route): scores, balance bias, groups, top-k and weights of a router's logits.
#include "device_common.h"
#include "rows_io.h"

namespace phx {

// Selection keys as unsigned integers in the values' order, 0 for "not a candidate": a double's bits with the sign
// folded (every number but NaN, which no key is, maps above 0).
__device__ __forceinline__ unsigned long long sortable_f64(double v)
{
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

struct RouteArgs {
    int T, E, k, G, used, gs;  // gs = E / G
    bool sigmoid, top2, renorm;
    float scale;
    const void* logits;
    const float* bias;
    int* ids;
    float* w;
};

// One wave per token, lane l holding experts 4 l .. 4 l + 3.  Each round of the choice is a maximum over the wave and
// a ballot: the lowest lane that holds it, and the first of its four, is the lowest index.
template <int DT>
__global__ __launch_bounds__(256) void k_route(RouteArgs R)
{
    constexpr double NINF = -__builtin_inf();
    __shared__ double sel[4][PHX_MAX_EXPERTS_DEV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * 4 + wave;
    if (t >= R.T) return;  // uniform over the wave, and the kernel has no workgroup barrier
    const int e0 = 4 * lane;
    float l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float v = e0 + i < R.E ? load_one<DT>(R.logits, (int64_t)t * R.E + e0 + i) : -INFINITY;
        l[i] = v > -INFINITY ? fminf(v, 3.402823466e38f) : -INFINITY;  // NaN compares false
    }
    // scores, 0 for what is no candidate by its logit
    double s[4];
    if (R.sigmoid) {
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = l[i] > -INFINITY ? 1.0 / (1.0 + exp(-(double)l[i])) : 0.0;
    } else {
        const double m = wave_max_dpp((double)fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])));
        double z = 0.0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[i] = l[i] > -INFINITY ? exp((double)l[i] - m) : 0.0;
            z += s[i];
        }
        z = wave_sum_dpp(z);
        const double rz = z > 0.0 ? 1.0 / z : 0.0;
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] *= rz;
    }
    // c: the score with the bias (what the sums of two take); key: what is compared
    double c[4];
    unsigned long long key[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bool able = l[i] > -INFINITY;
        c[i] = s[i];
        double r = (double)l[i];
        if (R.bias) {
            const float b = e0 + i < R.E ? R.bias[e0 + i] : -INFINITY;
            able = able && b > -INFINITY;
            r = c[i] = s[i] + (double)b;
        }
        if (!able) c[i] = NINF;
        key[i] = able ? sortable_f64(r + 0.0) : 0ull;  // -0 equals 0
    }
    if (R.used < R.G) {
        // a lane per group walks its experts; a group's rank is the number of groups ahead of it
#pragma unroll
        for (int i = 0; i < 4; i++) sel[wave][e0 + i] = R.top2 || R.bias ? c[i] : (double)l[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        double a = NINF, b = NINF;
        if (lane < R.G)
            for (int i = 0; i < R.gs; i++) {
                const double v = sel[wave][lane * R.gs + i];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
        if (R.top2 && b > NINF) a += b;
        int rank = 0;
        for (int g = 0; g < R.G; g++) {
            const double v = readlane_d(a, g);
            rank += v > a || (v == a && g < lane);
        }
        const unsigned long long kept = __ballot(lane < R.G && rank < R.used);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (e0 + i >= R.E || !((kept >> ((e0 + i) / R.gs)) & 1)) key[i] = 0ull;
    }
    int my_id = -1;
    double my_s = 0.0, total = 0.0;
    for (int j = 0; j < R.k; j++) {
        unsigned long long best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < 4; i++)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const unsigned long long top = wave_max_u64(best);
        if (top == 0ull) break;  // no candidate is left; uniform
        const int owner = __builtin_ctzll(__ballot(best == top));
        const double so = at == 0 ? s[0] : at == 1 ? s[1] : at == 2 ? s[2] : s[3];
        const double sv = readlane_d(so, owner);
        const int id = 4 * owner + __builtin_amdgcn_readlane(at, owner);
        total += sv;
        if (lane == j) {
            my_id = id;
            my_s = sv;
        }
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i == at) key[i] = 0ull;
        }
    }
    if (lane < R.k) {
        double w = my_s;
        if (R.renorm) w = total > 0.0 ? w / total : 0.0;
        R.ids[(int64_t)t * R.k + lane] = my_id;
        R.w[(int64_t)t * R.k + lane] = (float)(w * (double)R.scale);
    }
}

void launch_route(hipStream_t st, const phx_route_desc& D, int T, const void* logits, const float* bias, int* ids, float* w)
{
    RouteArgs R;
    R.T = T;
    R.E = D.n_expert;
    R.k = D.n_used;
    R.G = D.n_group;
    R.used = D.n_group_used;
    R.gs = D.n_expert / D.n_group;
    R.sigmoid = D.score == PHX_SCORE_SIGMOID;
    R.top2 = D.group_score == PHX_GROUP_TOP2;
    R.renorm = D.renorm != 0;
    R.scale = D.scale;
    R.logits = logits;
    R.bias = bias;
    R.ids = ids;
    R.w = w;
    const dim3 grid((T + 3) / 4), blk(256);
    switch (D.logits_type) {
    case PHX_F16: launch(k_route<PHX_F16>, grid, blk, 0, st, R); break;
    case PHX_BF16: launch(k_route<PHX_BF16>, grid, blk, 0, st, R); break;
    default: launch(k_route<PHX_F32>, grid, blk, 0, st, R); break;
    }
}

}  // namespace phx
