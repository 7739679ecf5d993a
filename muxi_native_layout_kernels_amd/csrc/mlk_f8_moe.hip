// Expert layers in e4m3 with block scales: grouped gate/up product with SiLU(gate) * up, grouped down product, weighted sum.
//
// The routed pairs are brought into expert order in blocks of 16, and in the same launch the activations are quantised; a task is one or two blocks of one expert, which share a pass over its
// weights.  The intermediate is quantised from fp32 to [slot][I] and [I / 128][slot] (slot = place in the order).  The weighted products of the down projection are kept in fp32
// [pair][H], and a last launch adds a token's pairs in the order of its picks.  One token needs neither order nor last launch; many pairs an expert go through panels (mlk_f8_moe_panel.cuh).
// Gate and up are sums of exact products in all of them (products that feed codes, mlk_f8.cuh).
#include <algorithm>
#include <cmath>

#include "mlk_f8_moe.cuh"
#include "mlk_panel_lds.cuh"

namespace mlk {

int launch_moe_align_quantize(const int32_t *topk_ids, int n_pairs, int E, const int32_t *experts_map, int id_limit, int32_t *sorted, int32_t *cumsum,
                              int32_t *padded, int32_t *experts_ids, MoeTask *tasks, int32_t *n_tasks, int cb_max, int cb_unit, int32_t *zero, int n_zero, const void *x, int x_kind,
                              bool wide, void *codes, float *scales, int tokens, int k, hipStream_t s);
extern template int f8_launch_moe_panels<F16>(const F8MoeArgs &, int, hipStream_t);
extern template int f8_launch_moe_panels<BF16>(const F8MoeArgs &, int, hipStream_t);

constexpr int kF8MoePairs = 16384;      // routed pairs of a pass: bounds the scratch of long prompts

// Gate/up: the four waves share the windows of two row groups of gate and the same two of up.  Bound by the weights' bytes: workgroups of a quarter of a block of 128 keep the card evenly
// busy, and waves that share windows read far longer pieces than waves with row groups of their own.  The last workgroup of a block to arrive makes the codes, from fp32.
// A workgroup a block, a row group of gate and of up a wave -> this: 64 experts of 2048 x 768 at 50 tokens 47.5 -> 35.9 us (192 MB of weights), 8 of 4096 x 14336 at 16 tokens
// 180 -> 159 (940 MB, 5.9 TB/s), at 2 tokens 89 -> 45.
constexpr int kF8UpWaves = 4, kF8UpGroups = 2, kF8UpParts = 8 / kF8UpGroups;
__device__ __forceinline__ f32x4 *f8_part(const F8MoeArgs &p, int task, int kb, int r, int tt) {
    return p.hpart + ((((size_t)task * (p.I / kF8K) + kb) * 8 + r) * 2 + tt) * 64;
}
// Whether this workgroup is the last of a block's.  Every wave waits for its own stores before the barrier and the arrival is counted behind it: the last one can read them all.
__device__ __forceinline__ bool f8_last_part(const F8MoeArgs &p, int task, int kb, int *last) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        int *at = &p.counters[task * (p.I / kF8K) + kb];
        *last = __hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == kF8UpParts - 1;
    }
    __syncthreads();
    return *last;
}
// Codes and scales of a block of 128 from its values in fp32.
template <int TT>
__device__ __forceinline__ void f8_codes_of_block(const F8MoeArgs &p, int block0, int task, int kb, float *most) {
    constexpr int W = kF8UpWaves, OWN = 8 / W;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t16 = lane & 15;
    f32x4 h[OWN][TT];
#pragma unroll
    for (int j = 0; j < OWN; ++j)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) h[j][tt] = ld_agent_planar(f8_part(p, task, kb, j * W + wave, tt), 64, lane);
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < OWN; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) a = fmaxf(a, f8_magnitude(h[j][tt][i]));
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        if (lane < 16) most[(wave * TT + tt) * 16 + t16] = a;
    }
    __syncthreads();
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        float a = 0.f;
#pragma unroll
        for (int v = 0; v < W; ++v) a = fmaxf(a, most[(v * TT + tt) * 16 + t16]);
        const int e = f8_exponent(a), slot = (block0 + tt) * 16 + t16;
        const float inverse = f8_two_to(-e);
#pragma unroll
        for (int j = 0; j < OWN; ++j)
            *reinterpret_cast<uint32_t *>(p.hbuf + (size_t)slot * p.I + kb * kF8K + (j * W + wave) * 16 + (lane >> 4) * 4) =
                f8_codes(h[j][tt][0], h[j][tt][1], h[j][tt][2], h[j][tt][3], inverse);
        if (wave == 0 && lane < 16) p.hs[(size_t)kb * p.slots + slot] = f8_two_to(e);
    }
}
template <int TT>
__device__ __forceinline__ void f8_gate_up_blocks(const F8MoeArgs &p, const MoeTask &task, f32x4 *red, float *most, int *last) {
    constexpr int G = kF8UpGroups, W = kF8UpWaves, CELLS = G * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t16 = lane & 15;
    const int windows = p.H / kF8K, kb = blockIdx.x / kF8UpParts, rg0 = blockIdx.x * G;
    const uint8_t *w = p.w1 + (size_t)task.expert * 2 * p.I * p.H;
    const float *s = p.s1 + (size_t)task.expert * (p.I / 64) * windows;
    F8Rows<2 * G> rows;
#pragma unroll
    for (int r = 0; r < G; ++r) {
        f8_row(rows, r, w, s, rg0 + r, windows);
        f8_row(rows, G + r, w, s, p.I / 16 + rg0 + r, windows);
    }
    F8Tokens<TT> tokens;
    tokens.step = p.T;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int pair = p.sorted[(task.block0 + tt) * 16 + t16], row = pair < p.n_pairs ? pair / p.K : 0;
        tokens.x[tt] = p.X + (size_t)row * p.H * 2;
        tokens.a[tt] = p.xs + row;
    }
    f32x4 acc[2 * G][TT];
#pragma unroll
    for (int r = 0; r < 2 * G; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    f8_wide_stream<TT, 2 * G, TT == 1 ? 2 : 1>(acc, rows, tokens, wave, windows, W, lane);
#pragma unroll
    for (int c = 0; c < 2 * CELLS; ++c) red[(wave * 2 * CELLS + c) * 64 + lane] = acc[c / TT][c % TT];
    __syncthreads();
    if (wave < CELLS) {
        f32x4 g = red[wave * 64 + lane], u = red[(CELLS + wave) * 64 + lane], h;
        for (int v = 1; v < W; ++v) {
            g += red[(v * 2 * CELLS + wave) * 64 + lane];
            u += red[(v * 2 * CELLS + CELLS + wave) * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = silu_mul(g[i], u[i]);
        st_agent_planar(f8_part(p, blockIdx.y, kb, (rg0 & 7) + wave / TT, wave % TT), 64, lane, h);
    }
    if (!f8_last_part(p, blockIdx.y, kb, last)) return;
    f8_codes_of_block<TT>(p, task.block0, blockIdx.y, kb, most);
}
__global__ void __launch_bounds__(256) f8_moe_gate_up_kernel(F8MoeArgs p) {
    __shared__ f32x4 red[kF8UpWaves * 2 * kF8UpGroups * 2 * 64];
    __shared__ float most[kF8UpWaves * 2 * 16];
    __shared__ int last;
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) f8_gate_up_blocks<1>(p, task, red, most, &last);
    else f8_gate_up_blocks<2>(p, task, red, most, &last);
}

// Down: the four waves share the windows of four row groups and add their sums in wave order.  Waves with row groups of their own read 16 rows each at far places and
// wait longer: 8 experts of 4096 x 14336 at 16 tokens 147 us with two row groups a wave, 72 us shared; 64 of 2048 x 768 at 50 tokens 31.7 and 18.2.
constexpr int kF8DownRows = 4, kF8DownWaves = 4;
template <class T, int TT>
__device__ __forceinline__ void f8_down_blocks(const F8MoeArgs &p, const MoeTask &task, f32x4 *red) {
    constexpr int R = kF8DownRows, W = kF8DownWaves, CELLS = R * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t16 = lane & 15;
    const int windows = p.I / kF8K, rg0 = blockIdx.x * R;
    F8Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) f8_row(rows, r, p.w2 + (size_t)task.expert * p.H * p.I, p.s2 + (size_t)task.expert * (p.H / 128) * windows, rg0 + r, windows);
    F8Tokens<TT> tokens;
    tokens.step = p.slots;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int slot = (task.block0 + tt) * 16 + t16;
        tokens.x[tt] = p.hbuf + (size_t)slot * p.I;
        tokens.a[tt] = p.hs + slot;
    }
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    f8_stream<TT, R, TT == 1 ? 2 : 1>(acc, rows, tokens, wave, windows, W, lane);
#pragma unroll
    for (int c = 0; c < CELLS; ++c) red[(wave * CELLS + c) * 64 + lane] = acc[c / TT][c % TT];
    __syncthreads();
    for (int c = wave; c < CELLS; c += W) {
        const int r = c / TT, tt = c - r * TT;
        f32x4 v = red[c * 64 + lane];
        for (int w = 1; w < W; ++w) v += red[(w * CELLS + c) * 64 + lane];
        const int pair = p.sorted[(task.block0 + tt) * 16 + t16];
        if (pair >= p.n_pairs) continue;
        v *= T::to_f32(p.wts[pair]);
        *reinterpret_cast<f32x4 *>(p.obuf + (size_t)pair * p.H + (rg0 + r) * 16 + (lane >> 4) * 4) = v;
    }
}
template <class T>
__global__ void __launch_bounds__(256) f8_moe_down_kernel(F8MoeArgs p) {
    __shared__ f32x4 red[kF8DownWaves * kF8DownRows * 2 * 64];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) f8_down_blocks<T, 1>(p, task, red);
    else f8_down_blocks<T, 2>(p, task, red);
}

// y[t] = T(sum over the token's pairs on this card, in pick order).  50 tokens of 8 picks, 2048 wide 4.6 us, a launch and two trips to memory; 1000 of 2, 4096 wide 9.0.
template <class T>
__global__ void __launch_bounds__(256) f8_moe_combine_kernel(F8MoeArgs p) {
    const int tok = blockIdx.x, lane = threadIdx.x & 63;
    const size_t step = (size_t)p.slices * p.H;
    const uint64_t here = __ballot(lane < p.K && f8_expert(p, tok * p.K + min(lane, p.K - 1)) >= 0);
    for (int n = (blockIdx.y * 256 + threadIdx.x) * 4; n < p.H; n += gridDim.y * 1024) {
        const float *pair = p.obuf + (size_t)tok * p.K * step + n;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (uint64_t left = here; left != 0;) {
            // the loads of four picks in flight, of the last one again where fewer are left: behind a branch each would wait for the one before
            int k[4];
            bool on[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                on[j] = left != 0;
                k[j] = on[j] ? __builtin_ctzll(left) : k[j == 0 ? 0 : j - 1];
                left &= left - 1;
            }
            f32x4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4 *>(pair + k[j] * step);
            for (int sl = 1; sl < p.slices; ++sl)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += *reinterpret_cast<const f32x4 *>(pair + k[j] * step + (size_t)sl * p.H);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (on[j]) sum += v[j];
        }
        *reinterpret_cast<u32x2 *>(p.Y + (size_t)tok * p.H + n) = u32x2{T::from_f32x2(sum[0], sum[1]), T::from_f32x2(sum[2], sum[3])};
    }
}

// --------------------------------------------------------------------------------------------------------------- one token
// Two launches.  gate/up: a workgroup takes two row groups of gate and of up of a pick, its waves share the windows; every workgroup quantises the token by itself, behind its first loads, and all
// sixteen columns are the token.  The intermediate is left in fp32.
// down: a workgroup takes a row group through all picks, whose intermediates it quantises into LDS; wave w takes picks w % side, w % side + side, ... and of each the
// windows of its place among the waves that share it; the weighted sums are added in wave order.
// 8 experts of 4096 x 14336, two picks: 37.4 us (235 MB of weights at 6.3 TB/s) and 22.8 (117 MB at 5.2); gate/up with a row group of each and eight waves 38 to 43.
constexpr int kF8OneWaves = 8;                   // down
constexpr size_t kF8OneLds = 128 * 1024;         // of the token, of the intermediates

template <class T>
__global__ void __launch_bounds__(256) f8_moe1_gate_up_kernel(F8MoeArgs p) {
    extern __shared__ u32x4 lds[];
    constexpr int G = kF8UpGroups, W = kF8UpWaves;
    const int e = f8_expert(p, blockIdx.y);
    if (e < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), windows = p.H / kF8K, rg0 = blockIdx.x * G;
    F8Rows<2 * G> rows;
    const uint8_t *w = p.w1 + (size_t)e * 2 * p.I * p.H;
    const float *s = p.s1 + (size_t)e * (p.I / 64) * windows;
#pragma unroll
    for (int r = 0; r < G; ++r) {
        f8_row(rows, r, w, s, rg0 + r, windows);
        f8_row(rows, G + r, w, s, p.I / 16 + rg0 + r, windows);
    }
    float *scales = reinterpret_cast<float *>(lds + (size_t)windows * 16);
    f32x4 acc[2 * G][1];
#pragma unroll
    for (int r = 0; r < 2 * G; ++r) acc[r][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    f8_wide_stream_staged<2 * G, 2>(acc, rows, lds, scales, wave, windows, W, lane, [&]() {
        const int l = threadIdx.x & 15;
        for (int b = threadIdx.x >> 4; b < windows; b += W * 4) {
            F8In<T> in;
            in.raw = ld_global_u32x4(reinterpret_cast<const uint16_t *>(p.raw) + (size_t)b * kF8K + l * 8);
            float v[8], scale;
            in.values(v);
            lds[b * 16 + l] = f8_widen(f8_block(v, scale));
            if (l == 0) scales[b] = scale;
        }
        __syncthreads();
    });
    __syncthreads();                             // the other waves still read the token
    f32x4 *red = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int r = 0; r < 2 * G; ++r) red[(wave * 2 * G + r) * 64 + lane] = acc[r][0];
    __syncthreads();
    if (wave < G && (lane & 15) == 0) {
        f32x4 g = red[wave * 64 + lane], u = red[(G + wave) * 64 + lane], h;
        for (int v = 1; v < W; ++v) {
            g += red[(v * 2 * G + wave) * 64 + lane];
            u += red[(v * 2 * G + G + wave) * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = silu_mul(g[i], u[i]);
        *reinterpret_cast<f32x4 *>(p.hraw + (size_t)blockIdx.y * p.I + (rg0 + wave) * 16 + (lane >> 4) * 4) = h;
    }
}
template <class T>
__global__ void __launch_bounds__(512) f8_moe1_down_kernel(F8MoeArgs p) {
    extern __shared__ u32x4 lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), windows = p.I / kF8K, rg = blockIdx.x;
    float *scales = reinterpret_cast<float *>(lds + (size_t)p.K * windows * 8);
    const int side = min(p.K, kF8OneWaves), mine = wave % side, place = wave / side, sharing = (kF8OneWaves - mine + side - 1) / side;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int k = mine; k < p.K; k += side) {
        const int e = f8_expert(p, k);
        F8Rows<1> rows;
        f8_row(rows, 0, p.w2 + (size_t)max(e, 0) * p.H * p.I, p.s2 + (size_t)max(e, 0) * (p.H / 128) * windows, rg, windows);
        F8Staged tokens;
        tokens.x = lds + (size_t)k * windows * 8;
        tokens.a = scales + k * windows;
        tokens.first = 0;
        f32x4 acc[1][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}};
        // a dropped pick has no windows
        f8_stream_staged<1, 8>(acc, rows, tokens, place, e < 0 ? 0 : windows, sharing, lane, [&]() {
            if (k != mine) return;
            const int l = threadIdx.x & 15;
            const int step = kF8OneWaves * 4, blocks = p.K * windows;
            for (int b0 = threadIdx.x >> 4; b0 < blocks; b0 += 4 * step) {
                F8In<float> in[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float *at = p.hraw + (size_t)min(b0 + j * step, blocks - 1) * kF8K + l * 8;
                    in[j].lo = *reinterpret_cast<const f32x4 *>(at);
                    in[j].hi = *reinterpret_cast<const f32x4 *>(at + 4);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = b0 + j * step;
                    if (b >= blocks) break;
                    float v[8], scale;
                    in[j].values(v);
                    reinterpret_cast<u32x2 *>(lds)[b * 16 + l] = f8_block(v, scale);       // of a dropped pick whatever lay there, which is not read
                    if (l == 0) scales[b] = scale;
                }
            }
            __syncthreads();
        });
        const float wt = e < 0 ? 0.f : T::to_f32(p.wts[k]);
        if (e >= 0)
#pragma unroll
            for (int v = 0; v < 4; ++v) sum[v] = fmaf(wt, acc[0][0][v], sum[v]);
    }
    __syncthreads();
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);
    if ((lane & 15) == 0) part[wave * 4 + (lane >> 4)] = sum;
    __syncthreads();
    const int i = threadIdx.x;
    if (i < 16) {
        float v = 0.f;
        for (int w = 0; w < kF8OneWaves; ++w) v += reinterpret_cast<const float *>(part)[w * 16 + i];
        p.Y[rg * 16 + i] = (uint16_t)T::from_f32(v);
    }
}

// -------------------------------------------------------------------------------------------------------------------- host
// Tokens of a pass.  The down panels' offsets of the intermediate's scales [I / 128][slot] are 32 bits: a pass of n pairs has at most n + 15 E + 15 slots (f8_moe_slots), and slots * I / 32 bytes stay
// within 2^32.  With I below 2^23 that leaves 12500 pairs at least.
static int f8_moe_pass_tokens(int n_tokens, int topk, int E, int inter) {
    const int64_t pairs = std::min<int64_t>(kF8MoePairs, (1ll << 37) / inter - 15 * E - 15);
    return (int)std::min<int64_t>(n_tokens, pairs / topk);
}

struct F8MoeWorkspace {
    MoeTask *tasks;
    int32_t *n_tasks, *sorted, *cumsum, *padded, *experts_ids;
    uint8_t *x, *hbuf;
    float *xs, *hs, *hraw, *obuf;
    f32x4 *hpart;
    int32_t *counters;
};
static size_t f8_one_up_lds(int hidden) { return std::max((size_t)hidden * 2 + (size_t)(hidden / kF8K) * 4, (size_t)kF8UpWaves * 2 * kF8UpGroups * 1024); }
static size_t f8_one_down_lds(int topk, int inter) { return std::max((size_t)topk * inter + (size_t)topk * (inter / kF8K) * 4, (size_t)kF8OneWaves * 64); }

struct F8MoePlan {
    bool one;                // one token
    bool panels;
    int blocks;              // of 16 pairs, of a task at most
    int max_tasks, slices;
};
// Experts that get pairs, and how many each: with E of the router's experts here that share of the pairs is expected here.
struct F8MoeLoad {
    int reached, load;
};
static F8MoeLoad f8_moe_load(int tokens, int E, int n_router, int topk) {
    const int pairs = tokens * topk, here = (int)std::max<int64_t>(1, std::min<int64_t>(pairs, (int64_t)pairs * E / n_router));
    const int reached = std::min(here, E);
    return {reached, (here + reached - 1) / reached};
}
// Panels' tasks of an expert with a little more than `load` pairs.
static int f8_moe_tasks(int load) {
    const int width = 16 * kF8PanelBlocks, high = load + (int)std::sqrt((double)load);
    return (high + width - 1) / width;
}
// Slices of the down panels' k: two where k is long and they spare a quarter of the rounds over the card, for the sums of a second slice to be written and read.  One -> two at 8 experts of
// 4096 x 14336 and 64 tokens 109 -> 88 us, 300 198 -> 132, 512 182 -> 167 (through the queues), 2000 379 -> 346 and 9 more to add them; at 1000, where the rounds are the same, 192 -> 210; four 94, 146, 149,
// 342, 193 and up to 35 more.  Of 2048 x 768 two cost 30 %.
static int f8_moe_slices(int load, int reached, int hidden, int inter) {
    if (inter < 64 * kF8K) return 1;
    const int items = (hidden + 255) / 256 * reached * f8_moe_tasks(load), cus = device_cus();
    return (2 * items + cus - 1) / cus * 2 <= (items + cus - 1) / cus * 3 ? 2 : 1;
}
constexpr int kF8MoeStreamed = 18;      // pairs an expert of the streaming kernels
static F8MoePlan f8_moe_plan(int tokens, int E, int n_router, int topk, int hidden, int inter) {
    F8MoePlan pl = {};
    const int pairs = tokens * topk;
    pl.slices = 1;
    if (tokens == 1 && f8_one_up_lds(hidden) <= kF8OneLds && f8_one_down_lds(topk, inter) <= kF8OneLds) {
        pl.one = true;
        return pl;
    }
    // Panels from 19 pairs an expert on: below, tasks of the streaming kernels pass over the weights about as often and start sooner.  The whole layer on the last count of pairs that is streamed and the first
    // of the panels: 8 experts of 4096 x 14336 286 and 277 us, 128 of 2048 x 768 160 and 154.
    // offsets within an expert's weights and of a token are 32 bits
    const F8MoeLoad l = f8_moe_load(tokens, E, n_router, topk);
    pl.panels = l.load > kF8MoeStreamed && (int64_t)hidden * inter < (1ll << 31) && (int64_t)tokens * hidden < (1ll << 31);
    if (pl.panels) pl.slices = f8_moe_slices(l.load, l.reached, hidden, inter);
    pl.blocks = pl.panels ? kF8PanelBlocks : 2;
    pl.max_tasks = std::min(pairs, E + pairs / (16 * pl.blocks));
    return pl;
}
static int f8_moe_slots(int64_t pairs, int E) { return (int)((pairs + E * 15 + 15) / 16 * 16); }
// Counters that the alignment clears: the arrivals of the blocks of 128, or the queues of the panels.
static int f8_moe_counters(const F8MoePlan &pl, int inter) { return pl.panels ? kWideQueues * kWideQueueStep : pl.max_tasks * (inter / kF8K); }
static size_t f8_moe_carve(uint8_t *base, const F8MoePlan &pl, int tokens, int E, int topk, int hidden, int inter, F8MoeWorkspace *ws) {
    const int64_t pairs = (int64_t)tokens * topk, slots = f8_moe_slots(pairs, E), blocks = slots / 16;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        uint8_t *ptr = base ? base + off : nullptr;
        off = (off + bytes + 255) / 256 * 256;
        return ptr;
    };
    F8MoeWorkspace w = {};
    if (pl.one) {
        w.hraw = (float *)take((size_t)topk * inter * 4);
        if (ws) *ws = w;
        return off;
    }
    w.tasks = (MoeTask *)take(sizeof(MoeTask) * (size_t)(blocks + 1));
    w.n_tasks = (int32_t *)take(sizeof(int32_t));
    w.sorted = (int32_t *)take(sizeof(int32_t) * (size_t)slots);
    w.cumsum = (int32_t *)take(sizeof(int32_t) * (size_t)(E + 1));
    w.padded = (int32_t *)take(sizeof(int32_t));
    w.experts_ids = (int32_t *)take(sizeof(int32_t) * (size_t)blocks);
    w.x = take((size_t)tokens * hidden * (pl.panels ? 1 : 2));
    w.xs = (float *)take((size_t)tokens * (hidden / kF8K) * 4);
    w.hbuf = take((size_t)slots * inter);
    w.hs = (float *)take((size_t)slots * (inter / kF8K) * 4);
    w.obuf = (float *)take((size_t)pairs * pl.slices * hidden * 4);
    w.counters = (int32_t *)take((size_t)f8_moe_counters(pl, inter) * 4);
    if (!pl.panels) w.hpart = (f32x4 *)take((size_t)pl.max_tasks * (inter / kF8K) * 16 * 1024);
    if (ws) *ws = w;
    return off;
}

static size_t f8_moe_pass_bytes(int tokens, int E, int n_router, int topk, int hidden, int inter) {
    return f8_moe_carve(nullptr, f8_moe_plan(tokens, E, n_router, topk, hidden, inter), tokens, E, topk, hidden, inter, nullptr);
}
// What the passes of a call take: some of one size, and a shorter last one, whose plan may differ.
static size_t f8_moe_call_bytes(int n_tokens, int E, int n_router, int topk, int hidden, int inter) {
    const int step = f8_moe_pass_tokens(n_tokens, topk, E, inter), rest = n_tokens % step;
    const size_t whole = f8_moe_pass_bytes(step, E, n_router, topk, hidden, inter);
    return rest ? std::max(whole, f8_moe_pass_bytes(rest, E, n_router, topk, hidden, inter)) : whole;
}

template <class T>
static int f8_launch_moe(const F8MoeArgs &a, const F8MoePlan &pl, hipStream_t s) {
    if (pl.one) {
        const size_t up = f8_one_up_lds(a.H), down = f8_one_down_lds(a.K, a.I);
        static bool ready_up[64] = {}, ready_down[64] = {};
        int rc = MLK_OK;
        if (up > 48 * 1024) rc = panel_lds_attribute(&f8_moe1_gate_up_kernel<T>, 150 * 1024, ready_up);
        if (rc == MLK_OK && down > 48 * 1024) rc = panel_lds_attribute(&f8_moe1_down_kernel<T>, 150 * 1024, ready_down);
        if (rc != MLK_OK) return rc;
        f8_moe1_gate_up_kernel<T><<<dim3(a.I / 16 / kF8UpGroups, a.K), kF8UpWaves * 64, up, s>>>(a);
        MLK_LAUNCH_CHECK();
        f8_moe1_down_kernel<T><<<a.H / 16, kF8OneWaves * 64, down, s>>>(a);
        MLK_LAUNCH_CHECK();
        return MLK_OK;
    }
    if (pl.panels) {
        const int rc = f8_launch_moe_panels<T>(a, pl.max_tasks, s);
        if (rc != MLK_OK) return rc;
    } else {
        f8_moe_gate_up_kernel<<<dim3(a.I / 128 * kF8UpParts, pl.max_tasks), kF8UpWaves * 64, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
        f8_moe_down_kernel<T><<<dim3(a.H / 16 / kF8DownRows, pl.max_tasks), kF8DownWaves * 64, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
    }
    f8_moe_combine_kernel<T><<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

size_t mlk_experts_fp8_workspace_bytes(int n_tokens, int n_experts, int n_router_experts, int topk, int hidden, int inter) {
    if (n_tokens <= 0 || n_experts <= 0 || n_experts > 256 || n_router_experts <= 0 || topk <= 0 || topk > 32 || hidden <= 0 || inter <= 0 || hidden >= (1 << 23) || inter >= (1 << 23)) return 0;
    // Enough for every shorter call too, some of whose plans take more (the partial sums of streamed tasks, two slices of the down projection).  Plans follow from the stage of a count of tokens, which
    // never falls; within a stage longer passes take more, so that its last one counts.
    const int longest = f8_moe_pass_tokens(n_tokens, topk, n_experts, inter);
    auto stage = [&](int t) {
        const int load = f8_moe_load(t, n_experts, n_router_experts, topk).load;
        return (int64_t)t * hidden >= (1ll << 31) ? 1 << 20 : load <= kF8MoeStreamed ? 0 : f8_moe_tasks(load);
    };
    size_t most = f8_moe_pass_bytes(1, n_experts, n_router_experts, topk, hidden, inter);
    for (int t = 1; t <= longest; ++t) {
        int high = longest;                                    // the last one of t's stage is in t .. high
        while (t < high) {
            const int mid = t + (high - t + 1) / 2;
            if (stage(mid) == stage(t)) t = mid;
            else high = mid - 1;
        }
        most = std::max(most, f8_moe_pass_bytes(t, n_experts, n_router_experts, topk, hidden, inter));
    }
    return most;
}

int mlk_fused_experts_fp8(const void *w1, const float *w1_scale, const void *w2, const float *w2_scale, const void *x, int n_tokens, int n_experts,
                          int n_router_experts, int topk, int hidden, int inter, int x_kind, const int32_t *topk_ids, const void *topk_weights,
                          const int32_t *experts_map, void *y, void *workspace, size_t workspace_bytes, void *stream) {
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16, "experts fp8: activations must be fp16 or bf16");
    MLK_REQUIRE(n_tokens >= 0, "experts fp8: negative token count");
    MLK_REQUIRE(n_experts >= 1 && n_experts <= 256, "experts fp8: 1..256 experts");
    MLK_REQUIRE(n_router_experts >= 1 && (experts_map || n_router_experts == n_experts), "experts fp8: fewer experts than the router's need an experts_map");
    MLK_REQUIRE(topk >= 1 && topk <= 32, "experts fp8: topk must be in 1..32");
    MLK_REQUIRE(hidden > 0 && inter > 0 && hidden % 128 == 0 && inter % 128 == 0, "experts fp8: hidden and intermediate sizes must be multiples of 128");
    MLK_REQUIRE(hidden < (1 << 23) && inter < (1 << 23), "experts fp8: hidden and intermediate sizes must be below 2^23");
    if (n_tokens == 0) return MLK_OK;
    MLK_REQUIRE(w1 && w1_scale && w2 && w2_scale && x && topk_ids && topk_weights && y && workspace, "experts fp8: null pointer");
    MLK_REQUIRE(aligned16(w1) && aligned16(w2) && aligned16(x) && aligned16(y) && aligned16(workspace),
                "experts fp8: weights, activations, outputs and workspace must lie on 16 bytes");
    if (workspace_bytes < f8_moe_call_bytes(n_tokens, n_experts, n_router_experts, topk, hidden, inter)) return fail(MLK_ERR_WORKSPACE, "experts fp8: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    F8MoeArgs a = {};
    a.w1 = (const uint8_t *)w1;
    a.w2 = (const uint8_t *)w2;
    a.s1 = w1_scale;
    a.s2 = w2_scale;
    a.map = experts_map;
    a.id_limit = n_router_experts;
    a.K = topk;
    a.H = hidden;
    a.I = inter;
    a.E = n_experts;
    const int step = f8_moe_pass_tokens(n_tokens, topk, n_experts, inter);
    for (int t0 = 0; t0 < n_tokens; t0 += step) {
        a.T = std::min(step, n_tokens - t0);
        a.n_pairs = a.T * topk;
        a.Y = (uint16_t *)y + (size_t)t0 * hidden;
        a.ids = topk_ids + (size_t)t0 * topk;
        a.wts = (const uint16_t *)topk_weights + (size_t)t0 * topk;
        const F8MoePlan pl = f8_moe_plan(a.T, n_experts, n_router_experts, topk, hidden, inter);
        a.slots = f8_moe_slots(a.n_pairs, n_experts);
        F8MoeWorkspace ws;
        f8_moe_carve((uint8_t *)workspace, pl, a.T, n_experts, topk, hidden, inter, &ws);
        a.X = ws.x;
        a.xs = ws.xs;
        a.sorted = ws.sorted;
        a.tasks = ws.tasks;
        a.n_tasks = ws.n_tasks;
        a.hbuf = ws.hbuf;
        a.hs = ws.hs;
        a.obuf = ws.obuf;
        a.hraw = ws.hraw;
        a.hpart = ws.hpart;
        a.counters = ws.counters;
        a.raw = (const uint16_t *)x + (size_t)t0 * hidden;
        a.slices = pl.slices;
        int rc = MLK_OK;
        if (!pl.one)
            rc = launch_moe_align_quantize(a.ids, a.n_pairs, n_experts, experts_map, a.id_limit, ws.sorted, ws.cumsum, ws.padded, ws.experts_ids, ws.tasks, ws.n_tasks,
                                           pl.blocks, pl.panels ? 4 : 0, ws.counters, f8_moe_counters(pl, inter), a.raw, x_kind,
                                           !pl.panels, ws.x, ws.xs, a.T, hidden, s);
        if (rc != MLK_OK) return rc;
        rc = x_kind == MLK_F16 ? f8_launch_moe<F16>(a, pl, s) : f8_launch_moe<BF16>(a, pl, s);
        if (rc != MLK_OK) return rc;
    }
    return MLK_OK;
}

}  // extern "C"
