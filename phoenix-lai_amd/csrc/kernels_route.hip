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
    int T, E, k, G, used, gs, inv_gs;  // gs = E / G; e / gs = e * inv_gs >> 16 for e < 256
    int lpg;                           // lanes that share a group's experts: the largest power of two up to 64 / G
    bool sigmoid, top2, renorm;
    float scale;
    const void* logits;
    const float* bias;
    int* ids;
    float* w;
};

// One wave per token, lane l holding experts V l .. V l + V - 1.  A round of the choice is the wave's maximum of 32-bit
// keys and a ballot: the lowest lane that holds it, and the first of its V, is the lowest index.  The keys are the logits,
// exact in 32 bits, where their order is the scores' (no bias): then only the k chosen scores are ever formed, one per
// lane.  With a bias (WIDE) they are the doubles s + b: the high words decide, and the low words where those are equal.
// One token takes 3.2 us, the latency of its chain of rounds.  Many are bound by instructions, not memory: a round over 64
// lanes serves one token, and 13001 tokens are 13 waves a SIMD: of 128 bf16 logits 8.5 us (4.2 MB); 2048 of 256 with bias and
// groups 7.3 us.  Double scores and 64-bit keys for every expert, each lane four of
// them, took 24.3 and 9.2.
template <int V, bool WIDE, int DT>
__global__ __launch_bounds__(256) void k_route(RouteArgs R)
{
    constexpr double NINF = -__builtin_inf();
    __shared__ double sel[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = blockIdx.x * 4 + wave;
    if (t >= R.T) return;  // uniform over the wave, and the kernel has no workgroup barrier
    const int e0 = V * lane;
    const bool grouped = R.used < R.G, pairs = grouped && R.top2;
    float l[V], bias[V];
    unsigned hi[V], lo[V];
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < V; i++) bias[i] = R.bias[min(e0 + i, R.E - 1)];  // what is past the last expert is no candidate
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float v = load_one<DT>(R.logits, (int64_t)t * R.E + min(e0 + i, R.E - 1));  // every load before a wait
        l[i] = e0 + i < R.E && v > -INFINITY ? fminf(v, 3.402823466e38f) : -INFINITY;  // NaN compares false
        hi[i] = l[i] > -INFINITY ? sortable_f32(l[i] + 0.0f) : 0u;      // -0 equals 0
        lo[i] = 0u;
    }
    // what the softmax needs of the whole row
    const bool soft_row = !R.sigmoid && (WIDE || pairs || !R.renorm);
    double m = 0.0, rz = 0.0, s[V];
    if (soft_row) {
        float mx = l[0];
#pragma unroll
        for (int i = 1; i < V; i++) mx = fmaxf(mx, l[i]);
        m = wave_max_dpp((double)mx);
        double z = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            s[i] = l[i] > -INFINITY ? exp((double)l[i] - m) : 0.0;
            z += s[i];
        }
        z = wave_sum_dpp(z);
        rz = z > 0.0 ? 1.0 / z : 0.0;
    }
    if (WIDE || pairs) {  // every expert's score
#pragma unroll
        for (int i = 0; i < V; i++) {
            if (R.sigmoid) s[i] = l[i] > -INFINITY ? 1.0 / (1.0 + exp(-(double)l[i])) : 0.0;
            else s[i] *= rz;
        }
    }
    double c[V];  // selection scores: what the groups' sums of two take
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float b = bias[i];
            const bool able = l[i] > -INFINITY && b > -INFINITY;
            c[i] = able ? s[i] + (double)b + 0.0 : NINF;
            const unsigned long long key = able ? sortable_f64(c[i]) : 0ull;
            hi[i] = (unsigned)(key >> 32);
            lo[i] = (unsigned)key;
        }
    }
    if (grouped) {
#pragma unroll
        for (int i = 0; i < V; i++)
            sel[wave][e0 + i] = WIDE ? c[i] : !pairs ? (double)l[i] : l[i] > -INFINITY ? s[i] : NINF;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // lpg lanes walk a group's experts and join their two largest; its rank is the number of groups ahead of it
        const int g = lane / R.lpg, sub = lane & (R.lpg - 1);
        double a = NINF, b = NINF;
        if (g < R.G)
            for (int i = sub; i < R.gs; i += R.lpg) {
                const double v = sel[wave][g * R.gs + i];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
        for (int x = 1; x < R.lpg; x <<= 1) {
            const double oa = __shfl_xor(a, x, 64), ob = __shfl_xor(b, x, 64);
            b = fmax(fmin(a, oa), fmax(b, ob));
            a = fmax(a, oa);
        }
        if (pairs && b > NINF) a += b;
        int rank = 0;
        for (int o = 0; o < R.G; o++) {
            const double v = readlane_d(a, o * R.lpg);
            rank += v > a || (v == a && o < g);
        }
        const unsigned long long kept = __ballot(sub == 0 && g < R.G && rank < R.used);
#pragma unroll
        for (int i = 0; i < V; i++)
            if (e0 + i >= R.E || !((kept >> ((((e0 + i) * R.inv_gs) >> 16) * R.lpg)) & 1)) hi[i] = lo[i] = 0u;
    }
    int my_id = -1;
    float my_l = -INFINITY;
    double my_s = 0.0;
    for (int j = 0; j < R.k; j++) {
        unsigned bh = hi[0], bl = lo[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < V; i++)
            if (WIDE ? u64_gt(hi[i], lo[i], bh, bl) : hi[i] > bh) {
                bh = hi[i];
                bl = lo[i];
                at = i;
            }
        const unsigned top = wave_max_u32(bh);
        if (top == 0u) break;  // no candidate is left; uniform
        unsigned long long who = __ballot(bh == top);
        if (WIDE && (who & (who - 1))) {
            const unsigned tl = wave_max_u32(bh == top ? bl : 0u);
            who = __ballot(bh == top && bl == tl);
        }
        const int owner = __builtin_ctzll(who);
        float lv = l[0];
        double sv = WIDE ? s[0] : 0.0;
#pragma unroll
        for (int i = 1; i < V; i++)
            if (at == i) {
                lv = l[i];
                if (WIDE) sv = s[i];
            }
        const int id = V * owner + __builtin_amdgcn_readlane(at, owner);
        if (WIDE) sv = readlane_d(sv, owner);
        else lv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lv), owner));
        if (lane == j) {
            my_id = id;
            my_l = lv;
            my_s = sv;
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (lane == owner && at == i) hi[i] = lo[i] = 0u;
    }
    if (!WIDE && my_id >= 0) {
        if (R.sigmoid) my_s = 1.0 / (1.0 + exp(-(double)my_l));
        else if (soft_row) my_s = exp((double)my_l - m) * rz;
        else my_s = exp((double)my_l - (double)__int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_l), 0)));
    }
    const double total = R.renorm ? wave_sum_dpp(my_s) : 1.0;
    if (lane < R.k) {
        const double w = !R.renorm ? my_s : total > 0.0 ? my_s / total : 0.0;
        R.ids[(int64_t)t * R.k + lane] = my_id;
        R.w[(int64_t)t * R.k + lane] = (float)(w * (double)R.scale);
    }
}

template <int V>
static void route_of(hipStream_t st, int type, const RouteArgs& R)
{
    const dim3 grid((R.T + 3) / 4), blk(256);
#define RT_L(DT)                                                                       \
    if (R.bias) launch(k_route<V, true, DT>, grid, blk, 0, st, R);                     \
    else launch(k_route<V, false, DT>, grid, blk, 0, st, R)
    switch (type) {
    case PHX_F16: RT_L(PHX_F16); break;
    case PHX_BF16: RT_L(PHX_BF16); break;
    default: RT_L(PHX_F32);
    }
#undef RT_L
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
    R.inv_gs = (65536 + R.gs - 1) / R.gs;
    R.lpg = 1;
    while (2 * R.lpg * R.G <= 64) R.lpg *= 2;
    if (R.E <= 64) route_of<1>(st, D.logits_type, R);
    else if (R.E <= 128) route_of<2>(st, D.logits_type, R);
    else route_of<4>(st, D.logits_type, R);
}

}  // namespace phx
