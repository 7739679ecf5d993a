// Expert layers in e4m3 with block scales: grouped gate/up product with SiLU(gate) * up, grouped down product, weighted sum.
//
// The routed pairs are brought into expert order in blocks of 16 (moe_align_kernel); a task is one or two blocks of one expert, which share a pass over its weights.  Activations are
// quantised once.  A gate/up workgroup computes 128 consecutive intermediate values of its tokens, a block of the next product's activations, so it has their
// maximum at hand and leaves codes and scale: [slot][I] and [I / 128][slot] (slot = place in the order).  The weighted products of the down projection are kept in fp32
// [pair][H], and a last launch adds a token's pairs in the order of its picks.
#include <algorithm>
#include <initializer_list>

#include "mlk_f8_moe.cuh"
#include "mlk_panel_lds.cuh"

namespace mlk {

int launch_moe_align_quantize(const int32_t *topk_ids, int n_pairs, int E, const int32_t *experts_map, int id_limit, int32_t *sorted, int32_t *cumsum,
                              int32_t *padded, int32_t *experts_ids, MoeTask *tasks, int32_t *n_tasks, int cb_max, int cb_unit, int32_t *queues, const void *x, int x_kind,
                              bool wide, void *codes, float *scales, int tokens, int k, hipStream_t s);
extern template int f8_launch_moe_panels<F16>(const F8MoeArgs &, int, hipStream_t);
extern template int f8_launch_moe_panels<BF16>(const F8MoeArgs &, int, hipStream_t);

constexpr int kF8MoePairs = 16384;      // routed pairs of a pass: bounds the scratch of long prompts

// Gate/up: wave w of eight streams the w-th row group of gate and the same one of up.
template <int TT>
__device__ __forceinline__ void f8_gate_up_blocks(const F8MoeArgs &p, const MoeTask &task, float *most) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t16 = lane & 15;
    const int windows = p.H / kF8K, rg = blockIdx.x * 8 + wave;
    const uint8_t *w = p.w1 + (size_t)task.expert * 2 * p.I * p.H;
    const float *s = p.s1 + (size_t)task.expert * (p.I / 64) * windows;
    F8Rows<2> rows;
    f8_row(rows, 0, w, s, rg, windows);
    f8_row(rows, 1, w, s, p.I / 16 + rg, windows);
    F8Tokens<TT> tokens;
    tokens.step = p.T;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int pair = p.sorted[(task.block0 + tt) * 16 + t16], row = pair < p.n_pairs ? pair / p.K : 0;
        tokens.x[tt] = p.X + (size_t)row * p.H * 2;
        tokens.a[tt] = p.xs + row;
    }
    f32x4 acc[2][TT];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    f8_wide_stream<TT, 2, TT == 1 ? 2 : 1>(acc, rows, tokens, 0, windows, 1, lane);
    f32x4 h[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[tt][i] = silu_mul(acc[0][tt][i], acc[1][tt][i]);
            a = fmaxf(a, f8_magnitude(h[tt][i]));
        }
        a = fmaxf(a, __shfl_xor(a, 16));
        a = fmaxf(a, __shfl_xor(a, 32));
        if (lane < 16) most[(wave * TT + tt) * 16 + t16] = a;
    }
    __syncthreads();
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        float a = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) a = fmaxf(a, most[(v * TT + tt) * 16 + t16]);
        const int e = f8_exponent(a), slot = (task.block0 + tt) * 16 + t16;
        *reinterpret_cast<uint32_t *>(p.hbuf + (size_t)slot * p.I + rg * 16 + (lane >> 4) * 4) = f8_codes(h[tt][0], h[tt][1], h[tt][2], h[tt][3], f8_two_to(-e));
        if (wave == 0 && lane < 16) p.hs[(size_t)blockIdx.x * p.slots + slot] = f8_two_to(e);
    }
}
__global__ void __launch_bounds__(512, 4) f8_moe_gate_up_kernel(F8MoeArgs p) {
    __shared__ float most[8 * 2 * 16];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) f8_gate_up_blocks<1>(p, task, most);
    else f8_gate_up_blocks<2>(p, task, most);
}

// Down: the waves share the windows of four row groups and add their sums in wave order.
constexpr int kF8DownRows = 4;
template <class T, int TT>
__device__ __forceinline__ void f8_down_blocks(const F8MoeArgs &p, const MoeTask &task, f32x4 *red) {
    constexpr int R = kF8DownRows, CELLS = R * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, t16 = lane & 15;
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
    f8_stream<TT, R, TT == 1 ? 2 : 1>(acc, rows, tokens, wave, windows, waves, lane);
#pragma unroll
    for (int c = 0; c < CELLS; ++c) red[(wave * CELLS + c) * 64 + lane] = acc[c / TT][c % TT];
    __syncthreads();
    for (int c = wave; c < CELLS; c += waves) {
        const int r = c / TT, tt = c - r * TT;
        f32x4 v = red[c * 64 + lane];
        for (int w = 1; w < waves; ++w) v += red[(w * CELLS + c) * 64 + lane];
        const int pair = p.sorted[(task.block0 + tt) * 16 + t16];
        if (pair >= p.n_pairs) continue;
        v *= T::to_f32(p.wts[pair]);
        *reinterpret_cast<f32x4 *>(p.obuf + (size_t)pair * p.H + (rg0 + r) * 16 + (lane >> 4) * 4) = v;
    }
}
template <class T>
__global__ void __launch_bounds__(256) f8_moe_down_kernel(F8MoeArgs p) {
    extern __shared__ f32x4 red[];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks == 1) f8_down_blocks<T, 1>(p, task, red);
    else f8_down_blocks<T, 2>(p, task, red);
}

// y[t] = T(sum over the token's pairs on this card, in pick order)
template <class T>
__global__ void __launch_bounds__(256) f8_moe_combine_kernel(F8MoeArgs p) {
    const int tok = blockIdx.x;
    for (int n = (blockIdx.y * 256 + threadIdx.x) * 4; n < p.H; n += gridDim.y * 1024) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.K; ++k) {
            // loaded whether the pair is here or not: a branch would make every load wait for the one before
            const int pair = tok * p.K + k;
            f32x4 v = *reinterpret_cast<const f32x4 *>(p.obuf + (size_t)pair * p.slices * p.H + n);
            for (int sl = 1; sl < p.slices; ++sl) v += *reinterpret_cast<const f32x4 *>(p.obuf + ((size_t)pair * p.slices + sl) * p.H + n);
            const bool here = f8_expert(p, pair) >= 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += here ? v[i] : 0.f;
        }
        *reinterpret_cast<u32x2 *>(p.Y + (size_t)tok * p.H + n) = u32x2{T::from_f32x2(sum[0], sum[1]), T::from_f32x2(sum[2], sum[3])};
    }
}

// --------------------------------------------------------------------------------------------------------------- one token
// Two launches.  gate/up: a workgroup takes a row group of gate and the one of up of a pick, its waves share the k and add their sums in wave order; every workgroup quantises the
// token by itself, behind its first loads.  The intermediate is left in fp32, as a workgroup has 16 values of a block of 128.
// down: a workgroup takes a row group through all picks, whose intermediates it quantises into LDS; wave w takes picks w % side, w % side + side, ... and of each the
// windows of its place among the waves that share it; the weighted sums are added in wave order.
constexpr int kF8OneWaves = 8;
constexpr size_t kF8OneLds = 128 * 1024;         // of the token, of the intermediates

template <class T>
__global__ void __launch_bounds__(512) f8_moe1_gate_up_kernel(F8MoeArgs p) {
    extern __shared__ u32x4 lds[];
    const int e = f8_expert(p, blockIdx.y);
    if (e < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), windows = p.H / kF8K, rg = blockIdx.x;
    F8Rows<2> rows;
    const uint8_t *w = p.w1 + (size_t)e * 2 * p.I * p.H;
    const float *s = p.s1 + (size_t)e * (p.I / 64) * windows;
    f8_row(rows, 0, w, s, rg, windows);
    f8_row(rows, 1, w, s, p.I / 16 + rg, windows);
    float *scales = reinterpret_cast<float *>(lds + (size_t)windows * 16);
    f32x4 acc[2][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}, {f32x4{0.f, 0.f, 0.f, 0.f}}};
    f8_wide_stream_staged<2, 4>(acc, rows, lds, scales, wave, windows, kF8OneWaves, lane, [&]() {
        const int l = threadIdx.x & 15;
        for (int b = threadIdx.x >> 4; b < windows; b += kF8OneWaves * 4) {
            F8In<T> in;
            in.raw = ld_global_u32x4(reinterpret_cast<const uint16_t *>(p.raw) + (size_t)b * kF8K + l * 8);
            float v[8], scale;
            in.values(v);
            lds[b * 16 + l] = f8_widen(f8_block(v, scale));
            if (l == 0) scales[b] = scale;
        }
        __syncthreads();
    });
    __syncthreads();
    // all columns are the same token: the lanes of column 0 hold four rows each
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);
    if ((lane & 15) == 0) {
        part[(wave * 2) * 4 + (lane >> 4)] = acc[0][0];
        part[(wave * 2 + 1) * 4 + (lane >> 4)] = acc[1][0];
    }
    __syncthreads();
    const int i = threadIdx.x;
    if (i < 16) {
        const float *f = reinterpret_cast<const float *>(part);
        float g = 0.f, u = 0.f;
        for (int v = 0; v < kF8OneWaves; ++v) {
            g += f[v * 32 + i];
            u += f[v * 32 + 16 + i];
        }
        p.hraw[(size_t)blockIdx.y * p.I + rg * 16 + i] = silu_mul(g, u);
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
            for (int b = threadIdx.x >> 4; b < p.K * windows; b += kF8OneWaves * 4) {
                if (f8_expert(p, b / windows) < 0) continue;                  // its intermediate was not written
                F8In<float> in;
                in.lo = *reinterpret_cast<const f32x4 *>(p.hraw + (size_t)b * kF8K + l * 8);
                in.hi = *reinterpret_cast<const f32x4 *>(p.hraw + (size_t)b * kF8K + l * 8 + 4);
                float v[8], scale;
                in.values(v);
                reinterpret_cast<u32x2 *>(lds)[b * 16 + l] = f8_block(v, scale);
                if (l == 0) scales[b] = scale;
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
static int f8_moe_pass_tokens(int n_tokens, int topk) { return n_tokens < kF8MoePairs / topk ? n_tokens : kF8MoePairs / topk; }

struct F8MoeWorkspace {
    MoeTask *tasks;
    int32_t *n_tasks, *sorted, *cumsum, *padded, *experts_ids;
    uint8_t *x, *hbuf;
    float *xs, *hs, *hraw, *obuf;
};
static size_t f8_one_lds(int picks, int k, bool wide) { return (size_t)picks * k * (wide ? 2 : 1) + (size_t)picks * (k / kF8K) * 4 + 64; }

struct F8MoePlan {
    bool one;                // one token
    bool panels;
    int blocks;              // of 16 pairs, of a task at most
    int max_tasks, slices;
};
static F8MoePlan f8_moe_plan(int tokens, int E, int n_router, int topk, int hidden, int inter) {
    F8MoePlan pl = {};
    const int pairs = tokens * topk;
    pl.slices = 1;
    if (tokens == 1 && f8_one_lds(1, hidden, true) <= kF8OneLds && f8_one_lds(topk, inter, false) <= kF8OneLds) {
        pl.one = true;
        return pl;
    }
    // with E of the router's experts here that share of the pairs is expected here
    const int here = (int)std::max<int64_t>(1, std::min<int64_t>(pairs, (int64_t)pairs * E / n_router));
    const int reached = std::min(here, E), load = (here + reached - 1) / reached;
    // offsets within an expert's weights and of a token are 32 bits
    pl.panels = load > 32 && (int64_t)hidden * inter < (1ll << 31) && (int64_t)tokens * hidden < (1ll << 31);
    pl.blocks = pl.panels ? kF8PanelBlocks : 2;
    pl.max_tasks = std::min(pairs, E + pairs / (16 * pl.blocks));
    return pl;
}
static int f8_moe_slots(int64_t pairs, int E) { return (int)((pairs + E * 15 + 15) / 16 * 16); }
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
    } else {
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
    }
    if (ws) *ws = w;
    return off;
}

template <class T>
static int f8_launch_moe(const F8MoeArgs &a, const F8MoePlan &pl, hipStream_t s) {
    if (pl.one) {
        const size_t up = std::max(f8_one_lds(1, a.H, true), (size_t)kF8OneWaves * 128), down = std::max(f8_one_lds(a.K, a.I, false), (size_t)kF8OneWaves * 64);
        static bool ready_up[64] = {}, ready_down[64] = {};
        int rc = MLK_OK;
        if (up > 48 * 1024) rc = panel_lds_attribute(&f8_moe1_gate_up_kernel<T>, 150 * 1024, ready_up);
        if (rc == MLK_OK && down > 48 * 1024) rc = panel_lds_attribute(&f8_moe1_down_kernel<T>, 150 * 1024, ready_down);
        if (rc != MLK_OK) return rc;
        f8_moe1_gate_up_kernel<T><<<dim3(a.I / 16, a.K), kF8OneWaves * 64, up, s>>>(a);
        MLK_LAUNCH_CHECK();
        f8_moe1_down_kernel<T><<<a.H / 16, kF8OneWaves * 64, down, s>>>(a);
        MLK_LAUNCH_CHECK();
        return MLK_OK;
    }
    if (pl.panels) {
        const int rc = f8_launch_moe_panels<T>(a, pl.max_tasks, s);
        if (rc != MLK_OK) return rc;
    } else {
        f8_moe_gate_up_kernel<<<dim3(a.I / 128, pl.max_tasks), 512, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
        f8_moe_down_kernel<T><<<dim3(a.H / 16 / kF8DownRows, pl.max_tasks), 256, 4 * kF8DownRows * 2 * 1024, s>>>(a);
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
    if (n_tokens <= 0 || n_experts <= 0 || n_experts > 256 || n_router_experts <= 0 || topk <= 0 || topk > 32 || hidden <= 0 || inter <= 0) return 0;
    // a long call goes in passes of one size and a shorter last one, whose plan may differ
    const int step = f8_moe_pass_tokens(n_tokens, topk), rest = n_tokens % step;
    size_t most = 0;
    for (int t : {step, rest})
        if (t > 0) most = std::max(most, f8_moe_carve(nullptr, f8_moe_plan(t, n_experts, n_router_experts, topk, hidden, inter), t, n_experts, topk, hidden, inter, nullptr));
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
    if (workspace_bytes < mlk_experts_fp8_workspace_bytes(n_tokens, n_experts, n_router_experts, topk, hidden, inter)) return fail(MLK_ERR_WORKSPACE, "experts fp8: workspace too small");
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
    const int step = f8_moe_pass_tokens(n_tokens, topk);
    for (int t0 = 0; t0 < n_tokens; t0 += step) {
        a.T = std::min(step, n_tokens - t0);
        a.n_pairs = a.T * topk;
        a.slots = f8_moe_slots(a.n_pairs, n_experts);
        a.Y = (uint16_t *)y + (size_t)t0 * hidden;
        a.ids = topk_ids + (size_t)t0 * topk;
        a.wts = (const uint16_t *)topk_weights + (size_t)t0 * topk;
        const F8MoePlan pl = f8_moe_plan(a.T, n_experts, n_router_experts, topk, hidden, inter);
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
        a.raw = (const uint16_t *)x + (size_t)t0 * hidden;
        a.slices = pl.slices;
        int rc = MLK_OK;
        if (!pl.one)
            rc = launch_moe_align_quantize(a.ids, a.n_pairs, n_experts, experts_map, a.id_limit, ws.sorted, ws.cumsum, ws.padded, ws.experts_ids, ws.tasks, ws.n_tasks,
                                           pl.blocks, pl.panels ? 4 : 0, nullptr, a.raw, x_kind, !pl.panels, ws.x, ws.xs, a.T, hidden, s);
        if (rc != MLK_OK) return rc;
        rc = x_kind == MLK_F16 ? f8_launch_moe<F16>(a, pl, s) : f8_launch_moe<BF16>(a, pl, s);
        if (rc != MLK_OK) return rc;
    }
    return MLK_OK;
}

}  // extern "C"
