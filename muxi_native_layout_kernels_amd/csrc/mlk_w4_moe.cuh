// Expert layers over 4-bit weights: grouped gate/up product with SiLU(gate) * up, grouped down product, weighted sum.
//
// Several tokens: the routed pairs are brought into expert order in blocks of 16 (moe_align_kernel); a task is a block, or up to two (panels: up to
// eight) of one expert, which share one pass over its weights.  The intermediate is kept row-major [slot][I] in the activations' type (slot = place in the order): the matrix
// instructions take 16 bits, and a second part for the bits below would double the products and the activations' bytes of the down projection, for errors of one rounding in place of 1.4.  The
// weighted products of the down projection are kept in fp32 [pair][slice][H], and a last launch adds a token's pairs in the order of its picks.
// One token: its picks are the tasks, no alignment; the down projection's waves deal the picks among themselves and write the output at once.
#pragma once

#include "mlk_moe_args.cuh"
#include "mlk_w4.cuh"

namespace mlk {

struct W4MoeArgs {
    W4Matrix w1, w2;             // of expert 0
    const uint16_t *X;           // [T][H]
    uint16_t *Y;                 // [T][H]
    const int32_t *ids;          // [T * K]
    const uint16_t *wts;         // [T * K]
    const int32_t *map;          // [id_limit] or null
    int id_limit, T, K, H, I, E, n_pairs;
    int blocks1, blocks2;        // blocks of scales of a row group of w1, of w2
    uint32_t inv;                // w4_inverse() of the tiles of a group
    const int32_t *sorted;
    const MoeTask *tasks;
    const int32_t *n_tasks;
    uint16_t *hbuf;              // [slot][I]
    float *obuf;                 // [pair][slice][H]
    int slices;                  // of the down projection's k
    u32x4 *sums1, *sums2;        // panels: sums of x, of the intermediate (w4_sums_kernel)
};

// Local expert of a pair, -1: dropped.
__device__ __forceinline__ int w4_expert(const W4MoeArgs &p, int pair) {
    int e = p.ids[pair];
    if (e < 0 || e >= p.id_limit) return -1;
    if (p.map) e = p.map[e];
    return e >= 0 && e < p.E ? e : -1;
}
template <int GS>
__device__ __forceinline__ W4Matrix w4_of_expert(const W4Matrix &m, int e, int rows, int k, int blocks) {
    const size_t entries = (size_t)e * rows * blocks * (4 / GS);
    return W4Matrix{m.codes + (size_t)e * rows * (k >> 1), m.scales + entries, m.zeros + entries};
}

__host__ __device__ constexpr int w4_moe_ring(int r) { return r <= 2 ? 4 : 2; }

// Rows of a gate/up workgroup: R / 2 row groups of gate, then the same of up.
template <int GS, int R>
__device__ __forceinline__ void w4_gate_up_rows(W4Rows<R> &rows, const W4MoeArgs &p, int e, int rg0) {
    const W4Matrix m = w4_of_expert<GS>(p.w1, e, 2 * p.I, p.H, p.blocks1);
#pragma unroll
    for (int r = 0; r < R; ++r) w4_row<GS, R>(rows, r, m, rg0 + r % (R / 2) + (r >= R / 2 ? p.I >> 4 : 0), p.H >> 7, p.blocks1);
}

template <int CELLS>
__device__ __forceinline__ void w4_park(f32x4 *red, const f32x4 (&acc)[CELLS], int wave, int lane) {
#pragma unroll
    for (int c = 0; c < CELLS; ++c) red[(wave * CELLS + c) * 64 + lane] = acc[c];
}
template <int CELLS>
__device__ __forceinline__ f32x4 w4_fold(const f32x4 *red, int c, int waves, int lane) {
    f32x4 v = red[c * 64 + lane];
    for (int w = 1; w < waves; ++w) v += red[(w * CELLS + c) * 64 + lane];
    return v;
}

// ---------------------------------------------------------------------------------------------------------- several tokens
// Registers: 128 for four workgroups on a CU (128 experts of 2048 x 768 at 50 tokens, zero points: 58.8 us, without the bound 60.1 with 132); groups of 32 with
// zero points would spill.
template <int GS, bool ZP>
__host__ __device__ constexpr int w4_moe_waves() { return GS == 1 && ZP ? 2 : 4; }

// The 16 slots of a task: expert, place of the first in the order, and the pair in slot lane % 16 (n_pairs: none).  False: no such task.
// FEW, at most 64 pairs: a wave takes them one per lane, goes through the experts in the order of their first pair and counts their blocks: no alignment
// launch (64 experts of 2048 x 1408, top-6, 4 tokens: 39.6 -> 36.4 us).
struct W4MoeBlock {
    int expert, slot0, pair;
};
template <bool FEW>
__device__ __forceinline__ bool w4_moe_block(const W4MoeArgs &p, int task, int lane, W4MoeBlock &b) {
    if constexpr (!FEW) {
        if (task >= *p.n_tasks) return false;
        const MoeTask t = p.tasks[task];
        b.expert = t.expert;
        b.slot0 = t.block0 * 16;
        b.pair = p.sorted[b.slot0 + (lane & 15)];
        return true;
    }
    const int e = lane < p.n_pairs ? w4_expert(p, lane) : -1;
    unsigned long long todo = __ballot(e >= 0);
    int before = 0;
    while (todo) {
        const int first = __builtin_amdgcn_readfirstlane(__ffsll((long long)todo) - 1), expert = __builtin_amdgcn_readlane(e, first);
        const unsigned long long same = __ballot(e == expert);
        const int pairs = __popcll(same), blocks = (pairs + 15) >> 4;
        if (task < before + blocks) {
            const int block = task - before, rank = __popcll(same & ((1ull << lane) - 1ull));
            const bool here = e == expert && rank >> 4 == block;
            // every pair of this block sends its number to the lane of its slot, the others to the last lane
            const int sent = __builtin_amdgcn_ds_permute((here ? rank & 15 : 63) * 4, lane);
            const int got = __shfl(sent, lane & 15);
            b.expert = expert;
            b.slot0 = task * 16;
            b.pair = block * 16 + (lane & 15) < pairs ? got : p.n_pairs;
            return true;
        }
        before += blocks;
        todo &= ~same;
    }
    return false;
}

// One block of 16 tokens a task.  Four waves share the k of R row groups, tile by tile, and add their sums through LDS in wave order.  Small workgroups even out
// over the CUs: with eight waves 128 experts of 2048 x 768 at 50 tokens 87 us, with four 81; 64 of 2048 x 1408 at 4 tokens 35 and 31; 8 of 4096 x 14336 at 16 132
// and 127; two sets of two waves, each on row groups of its own, are between.
constexpr int kW4MoeWaves = 4;

template <class T, int GS, bool ZP, int R, bool FEW>
__global__ void __launch_bounds__(kW4MoeWaves * 64, (w4_moe_waves<GS, ZP>())) w4_moe_gate_up_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    W4MoeBlock task;
    if (!w4_moe_block<FEW>(p, blockIdx.y, threadIdx.x & 63, task)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane >> 4, r16 = lane & 15, rg0 = blockIdx.x * (R / 2);
    W4Rows<R> rows;
    w4_gate_up_rows<GS, R>(rows, p, task.expert, rg0);
    const uint16_t *xrow[1] = {p.X + (size_t)(task.pair < p.n_pairs ? task.pair / p.K : 0) * p.H};
    f32x4 acc[R][1];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_stream<T, GS, ZP, 1, R, w4_moe_ring(R), false>(acc, rows, xrow, nullptr, wave, p.H >> 7, kW4MoeWaves, p.inv, lane, false);
    constexpr int HALF = R / 2;
    w4_park<R>(red, reinterpret_cast<const f32x4(&)[R]>(acc), wave, lane);
    __syncthreads();
    for (int c = wave; c < HALF; c += kW4MoeWaves) {
        const f32x4 g = w4_fold<R>(red, c, kW4MoeWaves, lane), u = w4_fold<R>(red, HALF + c, kW4MoeWaves, lane);
        uint16_t *h = p.hbuf + (size_t)(task.slot0 + o * 4) * p.I + (rg0 + c) * 16 + r16;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[(size_t)i * p.I] = (uint16_t)T::from_f32(silu_mul(g[i], u[i]));
    }
}

template <class T, int GS, bool ZP, int R, bool FEW>
__global__ void __launch_bounds__(kW4MoeWaves * 64, (w4_moe_waves<GS, ZP>())) w4_moe_down_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    W4MoeBlock task;
    if (!w4_moe_block<FEW>(p, blockIdx.y, threadIdx.x & 63, task)) return;
    __shared__ int pairs[16];
    if (threadIdx.x < 16) pairs[threadIdx.x] = task.pair;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane >> 4, r16 = lane & 15, rg0 = blockIdx.x * R;
    const W4Matrix m = w4_of_expert<GS>(p.w2, task.expert, p.H, p.I, p.blocks2);
    W4Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) w4_row<GS, R>(rows, r, m, rg0 + r, p.I >> 7, p.blocks2);
    const uint16_t *xrow[1] = {p.hbuf + (size_t)(task.slot0 + r16) * p.I};
    f32x4 acc[R][1];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_stream<T, GS, ZP, 1, R, w4_moe_ring(R), false>(acc, rows, xrow, nullptr, wave, p.I >> 7, kW4MoeWaves, p.inv, lane, false);
    w4_park<R>(red, reinterpret_cast<const f32x4(&)[R]>(acc), wave, lane);
    __syncthreads();
    for (int c = wave; c < R; c += kW4MoeWaves) {
        const f32x4 v = w4_fold<R>(red, c, kW4MoeWaves, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = pairs[o * 4 + i];
            if (pair < p.n_pairs) p.obuf[(size_t)pair * p.H + (rg0 + c) * 16 + r16] = T::to_f32(p.wts[pair]) * v[i];
        }
    }
}

// More pairs an expert: a task is one or two blocks, and a wave takes eight row groups, so that a workgroup's activations, which it reads whole, come to twice as many
// rows and the weights to twice as many tokens (8 experts of 4096 x 14336, top-2, 64 tokens: 238 -> 159 us).
template <class T, int GS, bool ZP, int TT, int R>
__device__ __forceinline__ void w4_moe_gate_up_blocks(const W4MoeArgs &p, const MoeTask &task, f32x4 *red) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane >> 4, r16 = lane & 15, rg0 = blockIdx.x * (R / 2);
    W4Rows<R> rows;
    w4_gate_up_rows<GS, R>(rows, p, task.expert, rg0);
    const uint16_t *xrow[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int pair = p.sorted[(task.block0 + tt) * 16 + r16];
        xrow[tt] = p.X + (size_t)(pair < p.n_pairs ? pair / p.K : 0) * p.H;
    }
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_stream<T, GS, ZP, TT, R, TT == 1 ? 2 : 1, false>(acc, rows, xrow, nullptr, wave, p.H >> 7, kW4MoeWaves, p.inv, lane, false);
    constexpr int CELLS = R * TT, HALF = CELLS / 2;
    w4_park<CELLS>(red, reinterpret_cast<const f32x4(&)[CELLS]>(acc), wave, lane);
    __syncthreads();
    for (int c = wave; c < HALF; c += kW4MoeWaves) {
        const int r = c / TT, tt = c - r * TT;
        const f32x4 g = w4_fold<CELLS>(red, c, kW4MoeWaves, lane), u = w4_fold<CELLS>(red, HALF + c, kW4MoeWaves, lane);
        uint16_t *h = p.hbuf + (size_t)((task.block0 + tt) * 16 + o * 4) * p.I + (rg0 + r) * 16 + r16;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[(size_t)i * p.I] = (uint16_t)T::from_f32(silu_mul(g[i], u[i]));
    }
}
template <class T, int GS, bool ZP, int TT, int R>
__device__ __forceinline__ void w4_moe_down_blocks(const W4MoeArgs &p, const MoeTask &task, f32x4 *red) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane >> 4, r16 = lane & 15, rg0 = blockIdx.x * R;
    const W4Matrix m = w4_of_expert<GS>(p.w2, task.expert, p.H, p.I, p.blocks2);
    W4Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) w4_row<GS, R>(rows, r, m, rg0 + r, p.I >> 7, p.blocks2);
    const uint16_t *xrow[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) xrow[tt] = p.hbuf + (size_t)((task.block0 + tt) * 16 + r16) * p.I;
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_stream<T, GS, ZP, TT, R, TT == 1 ? 2 : 1, false>(acc, rows, xrow, nullptr, wave, p.I >> 7, kW4MoeWaves, p.inv, lane, false);
    constexpr int CELLS = R * TT;
    w4_park<CELLS>(red, reinterpret_cast<const f32x4(&)[CELLS]>(acc), wave, lane);
    __syncthreads();
    for (int c = wave; c < CELLS; c += kW4MoeWaves) {
        const int r = c / TT, tt = c - r * TT;
        const f32x4 v = w4_fold<CELLS>(red, c, kW4MoeWaves, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = p.sorted[(task.block0 + tt) * 16 + o * 4 + i];
            if (pair < p.n_pairs) p.obuf[(size_t)pair * p.H + (rg0 + r) * 16 + r16] = T::to_f32(p.wts[pair]) * v[i];
        }
    }
}
template <class T, int GS, bool ZP>
__global__ void __launch_bounds__(kW4MoeWaves * 64, 2) w4_moe_gate_up2_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) w4_moe_gate_up_blocks<T, GS, ZP, 1, 8>(p, task, red);
    else w4_moe_gate_up_blocks<T, GS, ZP, 2, 8>(p, task, red);
}
template <class T, int GS, bool ZP>
__global__ void __launch_bounds__(kW4MoeWaves * 64, 2) w4_moe_down2_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) w4_moe_down_blocks<T, GS, ZP, 1, 8>(p, task, red);
    else w4_moe_down_blocks<T, GS, ZP, 2, 8>(p, task, red);
}

// y[t] = T(sum over the token's pairs on this card, in pick order)
template <class T>
__global__ void __launch_bounds__(256) w4_moe_combine_kernel(W4MoeArgs p) {
    const int tok = blockIdx.x;
    for (int n = (blockIdx.y * 256 + threadIdx.x) * 4; n < p.H; n += gridDim.y * 1024) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.K; ++k) {
            const int pair = tok * p.K + k;
            if (w4_expert(p, pair) < 0) continue;
            f32x4 v = *reinterpret_cast<const f32x4 *>(p.obuf + (size_t)pair * p.slices * p.H + n);
            for (int sl = 1; sl < p.slices; ++sl) v += *reinterpret_cast<const f32x4 *>(p.obuf + ((size_t)pair * p.slices + sl) * p.H + n);
            sum += v;
        }
        u32x2 out;
        out[0] = T::from_f32x2(sum[0], sum[1]);
        out[1] = T::from_f32x2(sum[2], sum[3]);
        *reinterpret_cast<u32x2 *>(p.Y + (size_t)tok * p.H + n) = out;
    }
}

// --------------------------------------------------------------------------------------------------------------- one token
template <class T, int GS, bool ZP, int R>
__global__ void __launch_bounds__(512) w4_moe1_gate_up_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    const int e = w4_expert(p, blockIdx.y);
    if (e < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int rg0 = blockIdx.x * (R / 2);
    W4Rows<R> rows;
    w4_gate_up_rows<GS, R>(rows, p, e, rg0);
    u32x4 *xl = reinterpret_cast<u32x4 *>(red);
    for (int i = threadIdx.x; i < p.H >> 3; i += blockDim.x) xl[i] = ld_global_u32x4(p.X + (size_t)i * 8);
    const uint16_t *xrow[1] = {nullptr};
    f32x4 acc[R][1];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    w4_stream<T, GS, ZP, 1, R, 4, true>(acc, rows, xrow, xl, wave, p.H >> 7, waves, p.inv, lane, true);
    __syncthreads();
    // all sixteen tokens of the block are the same one: lanes 0..15 hold the rows
    float *part = reinterpret_cast<float *>(red);
    if (lane < 16)
#pragma unroll
        for (int r = 0; r < R; ++r) part[(wave * R + r) * 16 + lane] = acc[r][0][0];
    __syncthreads();
    const int i = threadIdx.x;
    if (i < R / 2 * 16) {
        float g = 0.f, u = 0.f;
        for (int w = 0; w < waves; ++w) {
            g += part[w * R * 16 + i];
            u += part[w * R * 16 + R / 2 * 16 + i];
        }
        p.hbuf[(size_t)blockIdx.y * p.I + rg0 * 16 + i] = (uint16_t)T::from_f32(silu_mul(g, u));
    }
}

// XL: the intermediates of all picks are staged in LDS, which leaves registers for eight tiles in flight (8 experts of 4096 x 14336: the layer 43.0 -> 41.7 us).
template <class T, int GS, bool ZP, int R, bool XL>
__global__ void __launch_bounds__(512) w4_moe1_down_kernel(W4MoeArgs p) {
    extern __shared__ f32x4 red[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r16 = lane & 15, rg0 = blockIdx.x * R;
    u32x4 *xl = reinterpret_cast<u32x4 *>(red);
    if constexpr (XL)
        for (int i = threadIdx.x; i < p.K * (p.I >> 3); i += blockDim.x) xl[i] = ld_global_u32x4(p.hbuf + (size_t)i * 8);
    // wave w takes picks w % side, w % side + side, ... and of each the tiles of its place among the waves that share it
    const int side = min(p.K, waves), mine = wave % side, place = wave / side, sharing = (waves - mine + side - 1) / side;
    float sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = 0.f;
    for (int k = mine; k < p.K; k += side) {
        const int e = w4_expert(p, k), tiles = p.I >> 7;                  // a dropped pick has no tiles
        const W4Matrix m = w4_of_expert<GS>(p.w2, max(e, 0), p.H, p.I, p.blocks2);
        W4Rows<R> rows;
#pragma unroll
        for (int r = 0; r < R; ++r) w4_row<GS, R>(rows, r, m, rg0 + r, tiles, p.blocks2);
        const uint16_t *xrow[1] = {p.hbuf + (size_t)k * p.I};
        f32x4 acc[R][1];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][0] = f32x4{0.f, 0.f, 0.f, 0.f};
        w4_stream<T, GS, ZP, 1, R, XL ? 8 : w4_moe_ring(R), XL>(acc, rows, xrow, xl + k * (p.I >> 3), place, e < 0 ? 0 : tiles, sharing, p.inv, lane, k == mine);
        const float wt = e < 0 ? 0.f : T::to_f32(p.wts[k]);
#pragma unroll
        for (int r = 0; r < R; ++r) sum[r] = fmaf(wt, acc[r][0][0], sum[r]);
    }
    if constexpr (XL) __syncthreads();                    // the other waves still read the intermediates
    float *part = reinterpret_cast<float *>(red);
    if (lane < 16)
#pragma unroll
        for (int r = 0; r < R; ++r) part[(wave * R + r) * 16 + r16] = sum[r];
    __syncthreads();
    const int i = threadIdx.x;
    if (i < R * 16) {
        float v = 0.f;
        for (int w = 0; w < waves; ++w) v += part[w * R * 16 + i];
        p.Y[rg0 * 16 + i] = (uint16_t)T::from_f32(v);
    }
}

// -------------------------------------------------------------------------------------------------------------------- host
template <class K>
static int w4_moe_lds(K kernel, size_t lds, bool (&ready_on)[64]) {
    if (lds <= 48 * 1024) return MLK_OK;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    if (!ready_on[dev & 63]) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 150 * 1024);
        if (e != hipSuccess) return fail(MLK_ERR_LAUNCH, hipGetErrorString(e));
        ready_on[dev & 63] = true;
    }
    return MLK_OK;
}

struct W4MoePlan {
    int tt;                  // blocks of 16 tokens per task; 0: one token
    int max_tasks;
    bool few;                // at most 64 pairs, no alignment
    bool panels;             // tasks of up to 8 blocks run panels
    int slices;              // of their down projection
};

#define MLK_W4_MOE(KERNEL, GRID, WAVES, LDS, ...)                                          \
    do {                                                                                   \
        static bool ready_on[64] = {};                                                     \
        const int rc = w4_moe_lds(&KERNEL<__VA_ARGS__>, LDS, ready_on);                    \
        if (rc != MLK_OK) return rc;                                                       \
        KERNEL<__VA_ARGS__><<<GRID, (WAVES) * 64, LDS, s>>>(a);                            \
        MLK_LAUNCH_CHECK();                                                                \
    } while (0)

template <class T, int GS, bool ZP, int R, bool FEW>
static int w4_moe_gate_up(const W4MoeArgs &a, int max_tasks, hipStream_t s) {
    MLK_W4_MOE(w4_moe_gate_up_kernel, dim3(a.I / 8 / R, max_tasks), kW4MoeWaves, (size_t)kW4MoeWaves * R * 1024, T, GS, ZP, R, FEW);
    return MLK_OK;
}
template <class T, int GS, bool ZP, int R, bool FEW>
static int w4_moe_down(const W4MoeArgs &a, int max_tasks, hipStream_t s) {
    MLK_W4_MOE(w4_moe_down_kernel, dim3(a.H / 16 / R, max_tasks), kW4MoeWaves, (size_t)kW4MoeWaves * R * 1024, T, GS, ZP, R, FEW);
    return MLK_OK;
}
template <class T, int GS, bool ZP, int R>
static int w4_moe1_gate_up(const W4MoeArgs &a, hipStream_t s) {
    const size_t x = (size_t)a.H * 2, part = (size_t)8 * R * 64;
    MLK_W4_MOE(w4_moe1_gate_up_kernel, dim3(a.I / 8 / R, a.K), 8, (x > part ? x : part), T, GS, ZP, R);
    return MLK_OK;
}
template <class T, int GS, bool ZP, int R>
static int w4_moe1_down(const W4MoeArgs &a, hipStream_t s) {
    const size_t h = (size_t)a.K * a.I * 2;
    const size_t part = (size_t)8 * R * 64;
    if (h <= 128 * 1024) MLK_W4_MOE(w4_moe1_down_kernel, dim3(a.H / 16 / R), 8, (h > part ? h : part), T, GS, ZP, R, true);
    else MLK_W4_MOE(w4_moe1_down_kernel, dim3(a.H / 16 / R), 8, part, T, GS, ZP, R, false);
    return MLK_OK;
}

template <class T, int GS, bool ZP>
int w4_launch_moe(const W4MoeArgs &a, const W4MoePlan &pl, hipStream_t s) {
    int rc = MLK_ERR_INVALID;
    if (pl.tt == 0) {
        // one row group of gate and of up (8 experts of 4096 x 14336: the layer 43.8 us, with two 52.5), one of the down projection (52.4 and 56.6)
        rc = w4_moe1_gate_up<T, GS, ZP, 2>(a, s);
        return rc == MLK_OK ? w4_moe1_down<T, GS, ZP, 1>(a, s) : rc;
    }
    if (pl.tt == 2) {
        MLK_W4_MOE(w4_moe_gate_up2_kernel, dim3(a.I / 64, pl.max_tasks), kW4MoeWaves, (size_t)kW4MoeWaves * 16 * 1024, T, GS, ZP);
        MLK_W4_MOE(w4_moe_down2_kernel, dim3(a.H / 128, pl.max_tasks), kW4MoeWaves, (size_t)kW4MoeWaves * 16 * 1024, T, GS, ZP);
        w4_moe_combine_kernel<T><<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
        return MLK_OK;
    }
    // four row groups a wave: 128 registers (8 experts at 16 tokens: 120 us, with eight 139, with two 129)
    rc = pl.few ? w4_moe_gate_up<T, GS, ZP, 4, true>(a, pl.max_tasks, s) : w4_moe_gate_up<T, GS, ZP, 4, false>(a, pl.max_tasks, s);
    if (rc == MLK_OK) rc = pl.few ? w4_moe_down<T, GS, ZP, 4, true>(a, pl.max_tasks, s) : w4_moe_down<T, GS, ZP, 4, false>(a, pl.max_tasks, s);
    if (rc != MLK_OK) return rc;
    w4_moe_combine_kernel<T><<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // namespace mlk
