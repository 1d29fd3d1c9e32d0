// The tile kernel of products with fp16 and bf16 matrices in runs of ragged length.  Built apart from the row kernel, since its sums
// need both halves of the register file, for which the matrix instructions' results have to be left in accumulation registers,
// and each type, and the forms with rows in two terms, by themselves, since the widths of a tile are many and long to compile.
#pragma once
#include <algorithm>

#include "half_common.h"

namespace phx {

// k_half_tile: four waves, each 64 stored weight rows (PAIRED: the gate and up rows of 32 channels), by a tile of up to 256 places with
// one workgroup a compute unit, all of whose registers hold sums, or of up to 128 with two (MT 8 and 4: the row tiles of 32 it holds).
// The weights go straight from memory to each wave's registers (the layout has every operand as one run of 1 KB, and no other wave
// of the workgroup wants it), nearly two steps of 64 columns ahead; the places' rows, which all four waves read, go through an LDS
// ring by direct loads three to five steps ahead, row-major runs of 128 bytes with the 16-byte chunks XOR-swizzled by half the row's number
// (16 lanes of a 16-byte read then have 16 distinct bank groups).
// Measured: one 8192 x 8192 matrix by 8192 places 840 us, 1.31 PF (a library product 757), the matrix cores busy in 76% of the cycles: the
// last round and the epilogue of 8 us a tile are the rest.  16384 places in 128 uneven groups of 1408 x 2816 248 us at 5.4 TB/s: 1.33 GB read
// for 1.02 GB, since a group's second tile finds only a part of the weights still in the L2.  Few items are bound by whole rounds:
// 16412 places in 32 groups of 2816 x 4096 380 us, 1.0 PF, 918 items on 256 compute units.
constexpr int TI_WAVE = 32 * (64 * 4 + 16);  // a wave's part of the ring in the epilogue: 32 places' rows of 64 floats
// slots: as many steps as the ring holds, up to six (MT: the row tiles it is made for, 16 KB each)
constexpr int ti_ring(int nt, int mt) { return std::min(mt * 4 / nt, 6); }
// weight loads of group kk of a step, of term t of xt
constexpr int ti_weights(int xt, int t, int kk) { return xt == 1 || (kk == 0) == (t == 0) ? 2 : 0; }
// the loads behind the next step's rows where a step of term t waits for them, in its last group
constexpr int ti_newer(int nt, int ring, int xt, int t)
{
    const int dpg = (nt + 3) / 4, t0 = (t + ring) & 1;  // t0: of the step that issued these rows, ring - 2 before
    int n = std::min(nt, 3 * dpg);
    for (int kk = 0; kk < 3; kk++) n += ti_weights(xt, t, kk);
    for (int kk = (nt - 1) / dpg + 1; kk < 4; kk++) n += ti_weights(xt, t0, kk);  // behind its last row
    for (int j = 1; j <= ring - 3; j++) {
        n += nt;
        for (int kk = 0; kk < 4; kk++) n += ti_weights(xt, (t0 + j) & 1, kk);
    }
    return n;
}

// TERMS: the rows of x, or a paired product's output, are in two terms.  64 columns of x then are two steps, one a term, which
// both take the weights' registers, and the second issues the weights' loads.  16384 rows of two terms by 128 matrices of 2816 x 704
// to float 175 to 193 us, the matrix cores busy in 38% of the cycles, 610 MB read and 184 written (of one term 150 to 160).
template <int NT, int MT, bool PAIRED, bool ONCE, bool BF, bool TERMS>
__device__ __forceinline__ void half_tile_product(const HalfArgs& g, const Tile& tl, int bx, unsigned char* ring, uint32_t* orow)
{
    constexpr int STAGE = NT * 32 * 128, RING = ti_ring(NT, MT), XT = TERMS && !PAIRED ? 2 : 1;
    const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int S = g.kc / 8, Q = S * XT, row_bytes = g.cols * 2;  // steps of the weights and of the rows; bytes of a row's term
    // this lane's rows of the direct loads: one per load, the last row again past the tile's end
    const int chunk = ((lane & 7) ^ (lane >> 4)) * 16;  // of the loads whose first row is a multiple of 16; 4 chunks on for 8
    const __amdgpu_buffer_rsrc_t rsrc = buf_rsrc(g.x + (g.src ? 0 : (int64_t)tl.start * g.cols * XT));
    uint32_t xr[NT];  // rows that src names lie within 2^32 bytes of x, a tile's own of its first
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int at = min(8 * (wave * NT + i) + (lane >> 3), tl.cnt - 1);
        xr[i] = (uint32_t)(g.src ? max(x_row(g, tl.start + at), 0) : at) * (uint32_t)(row_bytes * XT);
        if (XT == 2) xr[i] += chunk ^ (64 * ((wave * NT + i) & 1));
    }
    for (int i = tid; i < NT * 32; i += 256) orow[i] = out_row(g, tl, i);
    int slot = 0;  // the ring's slot of a step; the one before it takes the rows of the step RING - 1 on
    auto after = [&](int at) { return at == (RING - 1) * STAGE ? 0 : at + STAGE; };
    auto before = [&](int at) { return at == 0 ? (RING - 1) * STAGE : at - STAGE; };
    auto column = [&](int s, int i) { return s / XT * 128 + (chunk ^ (64 * ((wave * NT + i) & 1))); };  // the lane's byte of load i's rows
    auto dma = [&](int s, int to, auto I) {          // load I of step s's rows
        constexpr int i = decltype(I)::value;
        const lds_void_t at = (lds_void_t)(ring + to + (wave * NT + i) * 1024);
        if constexpr (XT == 2) {  // columns past the row are what stands behind it, for clear() to remove: 128 bytes more than the rows are there
            const int su = min(s, Q - 1);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, at, 16, xr[i], (su >> 1) * 128 + (su & 1) * row_bytes, 0, 0);
        } else {
            const int off = column(min(s, Q - 1), i);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, at, 16, xr[i] + (off < row_bytes ? off : 0), 0, 0, 0);
        }
    };
    // zeros where a last step's loads, landed, hold columns past the row: against zero weights an infinity is none
    auto clear = [&](int s, int to) {
        if (s / XT != S - 1 || row_bytes == S * 128) return;  // uniform
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
    // slot any more): all at the group's start, the four waves' reads held up each other and the products behind them (an 8192 x
    // 8192 matrix by 8192 places, before the buffers were in scalar registers: 952 us, among the products 928).  Behind the others go
    // the loads: the weights that the group before has just used the registers of, two steps on, and the group's share of the rows
    // RING - 1 steps on.  The order is fixed by scheduling barriers:
    // the wait for the rows counts the loads issued after them.
    constexpr int DPG = (NT + 3) / 4;                                     // direct loads of a group
    constexpr int NEWER[2] = {ti_newer(NT, RING, XT, 0), ti_newer(NT, RING, XT, 1)};
    // the loads behind the first step's rows
    constexpr int NEWER_AT_START = (RING - 2) * NT + 14;
    static_assert(NEWER[0] < 64 && NEWER[1] < 64 && NEWER_AT_START < 64 && RING > 3, "vmcnt's range, and the first step's rows before any weights");
    auto step = [&](int s, auto P, auto TERM) {  // the weights' step and its parity, the rows' term
        constexpr int p = decltype(P)::value, t = decltype(TERM)::value;
        const int r = s * XT + t;
        const int next = after(slot), far = before(slot);
        static_for<4>([&](auto KK) {
            constexpr int kk = decltype(KK)::value;
            static_for<2 * NT>([&](auto M) {
                constexpr int m = decltype(M)::value, j = m / 2, b = m % 2;
                __builtin_amdgcn_sched_barrier(0);
                acc[j][b] = mma32<BF>(wv[p][b][kk], a[kk & 1][j], acc[j][b]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (m == 0 && kk == 3) {
                    __builtin_amdgcn_s_waitcnt(vm_wait(NEWER[t]));
                    clear(r + 1, next);
                    __builtin_amdgcn_s_barrier();
                }
                if constexpr (m < NT) read(kk < 3 ? slot : next, ic<(kk + 1) % 4>{}, ic<(m < NT ? m : 0)>{});
                static_for<2 + DPG>([&](auto I) {
                    constexpr int i = decltype(I)::value, d = kk * DPG + i - 2;
                    if constexpr (m == NT + i * NT / (2 + DPG)) {
                        if constexpr (i < 2 && ti_weights(XT, t, kk) == 0) {
                        } else if constexpr (i < 2 && kk == 0) weight(s + 1, i, ic<1 - p>{}, ic<3>{});
                        else if constexpr (i < 2) weight(s + 2, i, ic<p>{}, ic<(kk + 3) % 4>{});
                        else if constexpr (d < NT) dma(r + RING - 1, far, ic<d>{});
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
    if constexpr (XT == 2)
        static_for<3>([&](auto KK) {
            weight(0, 0, ic<0>{}, KK), weight(0, 1, ic<0>{}, KK);
            __builtin_amdgcn_sched_barrier(0);
        });
    static_for<2>([&](auto P) {
        constexpr int p = decltype(P)::value, r = RING - 3 + p;  // the rows' step p - 2, its loads the rows of step r
        static_for<4>([&](auto KK) {
            constexpr int kk = decltype(KK)::value;
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kk > 0 && (XT == 1 || p == 1)) weight(p, 0, ic<p>{}, ic<(kk + 3) % 4>{}), weight(p, 1, ic<p>{}, ic<(kk + 3) % 4>{});
            else if constexpr (kk == 0 && p == 2 - XT) weight(0, 0, ic<0>{}, ic<3>{}), weight(0, 1, ic<0>{}, ic<3>{});
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
        static_for<XT>([&](auto T) { step(s, ic<0>{}, T); });
        static_for<XT>([&](auto T) { step(s + 1, ic<1>{}, T); });
    }
    if (S & 1) static_for<XT>([&](auto T) { step(S - 1, ic<0>{}, T); });
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
    // the same of a value's two terms, each 32 channels of a place 64 bytes; out_cols is a multiple of 8, as the second product's columns
    auto store_terms = [&](auto J) {
        constexpr int j = decltype(J)::value, PITCH = 2 * 2 * 32 + 16;
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            uint32_t u[2][4];
#pragma unroll
            for (int v = 0; v < 8; v += 2) {
                uint16_t t[2][2];
#pragma unroll
                for (int w = 0; w < 2; w++) split<BF>(gated_half(g.act, acc[j][0][i + v + w], acc[j][1][i + v + w]), t[w]);
#pragma unroll
                for (int z = 0; z < 2; z++) u[z][v / 2] = t[0][z] | (uint32_t)t[1][z] << 16;
            }
#pragma unroll
            for (int z = 0; z < 2; z++) *(uint4*)(mine + r32 * PITCH + z * 64 + (16 * h + i) * 2) = make_uint4(u[z][0], u[z][1], u[z][2], u[z][3]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int c = lane & 7, col = col0 + (c & 3) * 8;  // eight lanes a place, four a term
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const int tok = it * 8 + (lane >> 3);
            const uint32_t o = orow[32 * j + tok];
            const uint4 y = *(const uint4*)(mine + tok * PITCH + c * 16);
            if (o != NO_ROW && col < g.out_cols) *(uint4*)(out + o + (int64_t)((c >> 2) * g.out_cols + col) * 2) = y;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (TERMS && PAIRED) static_for<NT>(store_terms);
    else if constexpr (TERMS) static_for<NT>([&](auto J) { store(ic<4>{}, J); });
    else if (g.type == PHX_F32) static_for<NT>([&](auto J) { store(ic<4>{}, J); });
    else static_for<NT>([&](auto J) { store(ic<2>{}, J); });
}

// Workgroup L runs on XCD L % 8.  The items (a tile's block of 256 stored rows) are in the order of groups, blocks, tiles, and
// each XCD takes an eighth of them as one run: a group's tiles meet a block's weights in one L2 at about one time, and the weights
// leave memory once.
template <int MT, bool PAIRED, bool BF, bool TERMS>
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
    bool alone;
    if (k >= run || item >= all || !G.find(g, item, blocks, &tl, &bx, &alone)) return;  // uniform over the workgroup
    // said once more, so that addresses stay in scalar registers: a buffer in vector ones costs a loop for each load
    tl = {__builtin_amdgcn_readfirstlane(tl.e), __builtin_amdgcn_readfirstlane(tl.start), __builtin_amdgcn_readfirstlane(tl.cnt)};
    bx = __builtin_amdgcn_readfirstlane(bx);
    const int n = (tl.cnt + 31) / 32;
    if constexpr (TERMS && !PAIRED) {  // kHalfTerms
        switch (g.once && alone ? n + 3 : n) {
        case 1: half_tile_product<1, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 2: half_tile_product<2, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 3: half_tile_product<3, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 4: half_tile_product<1, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 5: half_tile_product<2, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow); break;
        default: half_tile_product<3, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow);
        }
    } else if constexpr (MT == 4) {
        // a group's only tile reads its weights alone: past the caches, where the call's are more than they keep to the next (us,
        // through and past them; places in 128 groups of 1408 x 2816: 1624 170, 154; 4000 212, 193; 8000 214, 206; 16384 255, 252;
        // 4000 in 64 of 4096 x 1408 168, 173; past them for every tile, 16384 places: 295)
        switch (g.once && alone ? n + 4 : n) {
        case 1: half_tile_product<1, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 2: half_tile_product<2, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 3: half_tile_product<3, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 4: half_tile_product<4, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 5: half_tile_product<1, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 6: half_tile_product<2, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 7: half_tile_product<3, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow); break;
        default: half_tile_product<4, MT, PAIRED, true, BF, TERMS>(g, tl, bx, ring, orow);
        }
    } else {
        switch (n) {
        case 1: half_tile_product<1, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 2: half_tile_product<2, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 3: half_tile_product<3, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 4: half_tile_product<4, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 5: half_tile_product<5, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 6: half_tile_product<6, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        case 7: half_tile_product<7, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow); break;
        default: half_tile_product<8, MT, PAIRED, false, BF, TERMS>(g, tl, bx, ring, orow);
        }
    }
}

template <int MT, bool PAIRED, bool BF, bool TERMS>
static void half_tiles(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    const dim3 grid((max_tiles * ((m.rg + 7) / 8) + 7) / 8 * 8);
    launch(k_half_tile<MT, PAIRED, BF, TERMS>, grid, dim3(256), 0, st, g);
}

template <bool BF, bool TERMS>
void launch_half_tiles(hipStream_t st, const HalfMat& m, const HalfArgs& g, int max_tiles)
{
    if (g.cap <= kHalfNarrow && m.paired) half_tiles<4, true, BF, TERMS>(st, m, g, max_tiles);
    else if (TERMS ? !m.paired : g.cap <= kHalfNarrow) half_tiles<4, false, BF, TERMS>(st, m, g, max_tiles);
    else if (m.paired) half_tiles<8, true, BF, TERMS>(st, m, g, max_tiles);
    else if constexpr (!TERMS) half_tiles<8, false, BF, TERMS>(st, m, g, max_tiles);
}

}  // namespace phx
