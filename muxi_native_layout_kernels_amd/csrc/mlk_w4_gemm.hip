// Linear layers over 4-bit weights: one token (GeMV) to prefill-sized batches.
#include <algorithm>

#include "mlk_w4_panel_gemm.cuh"

namespace mlk {

#define MLK_W4_EXTERN(T, GS)                                                                          \
    extern template int w4_launch_stream<T, GS, false>(const W4GemmArgs &, int, int, int, int, hipStream_t); \
    extern template int w4_launch_stream<T, GS, true>(const W4GemmArgs &, int, int, int, int, hipStream_t);  \
    extern template int w4_launch_panel<T, GS, false>(const W4PanelArgs &, int, hipStream_t);           \
    extern template int w4_launch_panel<T, GS, true>(const W4PanelArgs &, int, hipStream_t);
MLK_W4_EXTERN(F16, 4)
MLK_W4_EXTERN(F16, 2)
MLK_W4_EXTERN(F16, 1)
MLK_W4_EXTERN(BF16, 4)
MLK_W4_EXTERN(BF16, 2)
MLK_W4_EXTERN(BF16, 1)
#undef MLK_W4_EXTERN

struct W4Plan {
    int r, tt, wgs, waves;  // streaming kernels: row groups and blocks of 16 tokens of a workgroup
    int tb;                 // panels: blocks of 32 tokens; 0: streaming kernels
    int slices;             // of K
};

// Up to 32 tokens.  Microseconds on weights from memory, groups of 128, bf16 (r row groups a workgroup, s slices of K):
//   one to four tokens   one workgroup per CU as far as r <= 4 goes, K whole: 4096 x 4096 r = 1 4.7 (s = 2: 6.3), 4096 x 14336 r = 1 9.8, r = 2 s = 2 10.7; 28672 x 8192 one
//                        token r = 2 25.7, r = 4 27.5, two tokens r = 4 24.9, r = 2 31.6.  So, with m * tiles up to 600, where that gives between half of the CUs and all
//                        a workgroup: 4096 x 4096 at 8 tokens 7.1 in slices, 5.7 whole, at 16 7.2 and 7.0, at 24 8.2 and 8.6; 8192 x 8192 at 8 11.3 and 10.8, at 16 12.1 and
//                        12.8; 7168 x 2304 at 32 8.5 and 7.7
//   more                 the activations weigh more (every workgroup reads all of them): r = 8 where that many row groups each, in slices of 48 tiles at least, leave
//                        three quarters of the CUs a workgroup: 28672 x 8192 at 32 tokens r = 4 45.7, r = 8 32.6,
//                        at 16 31.2 and 28.8; 27648 x 5120 at 32 30.0 and 22.8; 28672 x 4096 at 16 16.6 and 17.3; not 13824 x 5120 at 32, r = 4 18.8, r = 8 s = 2 19.1.
//                        Else r = 4, and slices bring the workgroups back: 4096 x 14336 at 16 tokens r = 1
//                        16.7, r = 2 s = 2 13.6, r = 4 s = 4 11.6.  At least six tiles a slice
//                        (1280 x 5120 at 16 tokens r = 2 s = 4 6.3, s = 8 9).  More workgroups than CUs have four waves (57344 x 2048 at 32 tokens r = 8 25.0, with four
//                        22.2; fewer eight: 28672 x 8192 32.9, with four 37.8)
static W4Plan w4_plan_stream(int m, int n, int k) {
    const int groups = n / 16, tiles = k / 128, cus = device_cus();
    W4Plan pl = {};
    pl.tb = 0;
    pl.slices = pl.r = 1;
    pl.tt = (m + 15) / 16;
    if (m <= 4 || (m * tiles <= 600 && 2 * groups > cus && groups <= 4 * cus)) {
        while (pl.r < 4 && groups > pl.r * cus) pl.r *= 2;
        if (m == 1 && pl.r == 4 && groups > 4 * cus) pl.r = 2;
        pl.wgs = (groups + pl.r - 1) / pl.r;
        pl.waves = m == 1 && pl.r == 1 && groups <= cus && tiles >= 16 && tiles * 256 <= kW4TokenLds ? 16 : 8;      // 16: only with the token in LDS
        return pl;
    }
    auto slices_of = [&](int wgs, int most) { return std::max(1, std::min(cus / wgs, most)); };
    const int wide = (groups + 7) / 8;
    if (4 * wide * slices_of(wide, tiles / 48) >= 3 * cus) {
        pl.r = 8;
        pl.slices = slices_of(wide, tiles / 48);
    } else {
        const int most = std::max(1, std::min(tiles / 6, 8));
        pl.r = 4;
        while (pl.r > 1 && (groups + pl.r - 1) / pl.r * most < 128) pl.r /= 2;
        pl.slices = slices_of((groups + pl.r - 1) / pl.r, most);
    }
    pl.wgs = (groups + pl.r - 1) / pl.r;
    pl.waves = pl.wgs > cus ? 4 : 8;
    return pl;
}

// A fitted cost of panels of 32 tb tokens in `slices` slices of K, in microseconds: rounds of one panel per CU; a window of 128 k takes 0.82 (tb = 2) or 1.18 us
// (tb = 4) with few panels on the chip and 0.2 or 0.5 more with one on every CU; three windows go to the start and the end, one for every 16 groups to the
// sums of x; launches and sums 6 us, the fold 2 us and its bytes.  Smaller groups cost more vector instructions a window.
static double w4_panel_cost(int m, int n, int k, int group, int tb, int slices, int cus) {
    const int64_t panels = ((int64_t)n + 255) / 256 * (((int64_t)m + 32 * tb - 1) / (32 * tb)), rounds = (panels * slices + cus - 1) / cus;
    const int windows = (k / 128 + slices - 1) / slices, g = group < 128 ? 128 / group : 1;
    const double full = rounds > 1 ? 1.0 : (double)panels * slices / cus;
    const double window = (tb == 2 ? 0.82 + 0.2 * full : 1.18 + 0.5 * full) * (g == 1 ? 1.0 : (g == 2 ? 1.15 : 1.45));
    return rounds * (windows + (windows * g + 15) / 16 + 3) * window + 6 + (slices > 1 ? 2 + (double)slices * m * n * 8 / 5e6 : 0);
}
// And of the streaming kernels with tt blocks of 16 tokens and r row groups a workgroup: a tile of 128 k takes 0.05 us and 0.027 for every block and row group (r = 8
// 0.0235), or what the workgroups on the chip read of the activations for it at 9.2 TB/s, which L2 gives, or what one reads at 48 GB/s; a round of workgroups 1.4,
// slices 2.5 (r = 8 3.5) and their bytes.
// 256 workgroups each: 4096 x 4096 at 100 tokens tt = 2 r = 4 12.8 us, at 160 tt = 3 16.2, at 256 tt = 4 20.8; 1280 x 5120 at 100 tt = 3 r = 1 16.6, tt = 3 r = 4 in four slices 10.8.
static double w4_stream_cost(int m, int n, int k, int group, int tt, int r, int slices, int cus) {
    const int64_t wgs = ((int64_t)n / 16 + r - 1) / r * (((int64_t)m + 16 * tt - 1) / (16 * tt)) * slices, rounds = (wgs + cus - 1) / cus;
    const double work = (r == 8 ? 0.06 + 0.0235 * tt * r : 0.05 + 0.0268 * tt * r) * (group == 32 ? 1.2 : (group == 64 ? 1.05 : 1.0));
    const double tile = std::max({work, 4096.0 * tt * std::min<int64_t>(wgs, cus) / 9.2e6, (4096.0 * tt + 1024.0 * r) / 48e3});
    return 2.6 + rounds * (1.4 + (k / 128 + slices - 1) / slices * tile) + (slices > 1 ? (r == 8 ? 3.5 : 2.5) + (double)slices * n * ((m + 15) / 16 * 16) * 8 / 5e6 : 0);
}

// Above 32 tokens the cheaper of panels and streaming kernels by those costs (512 x 7168 at 100 tokens panels 17.9, streaming 8.7; 1024 x 1024 at 256 14.8 and 5.1;
// 4096 x 4096 at 160 23.8 and 16.2, at 500 32.0 and 39.8; 11008 x 4096 at 100 26.9 and 34.4).
static W4Plan w4_plan(int m, int n, int k, int group) {
    if (m <= 32) return w4_plan_stream(m, n, k);
    const int cus = device_cus(), groups = n / 16, tiles = k / 128;
    W4Plan best = {};
    double least = 1e300;
    auto panels = [&](int tb, int slices) {
        const double c = w4_panel_cost(m, n, k, group, tb, slices, cus);
        if (c < least) {
            least = c;
            best = W4Plan{0, 0, 0, 0, tb, slices};
        }
    };
    for (int tb = 2; tb <= 4; tb += 2) {
        panels(tb, 1);
        for (int slices = 2; slices <= 16 && slices * 2 <= tiles; ++slices) panels(tb, slices);
    }
    for (int tt = 2; tt <= 4; ++tt)
        for (int r = tt == 2 ? 1 : (tt == 3 ? 2 : 4); r <= (tt < 4 ? 8 : 4); r *= 2) {            // others are the cheapest for one shape in thousands
            const int64_t blocks = ((int64_t)m + 16 * tt - 1) / (16 * tt), wgs = (groups + r - 1) / r;
            for (int slices = 1; slices == 1 || (slices <= 8 && slices * 6 <= tiles && wgs * blocks * slices <= 2 * cus); ++slices) {
                const double c = w4_stream_cost(m, n, k, group, tt, r, slices, cus);
                if (c < least && blocks <= 65535) {
                    least = c;
                    best = W4Plan{r, tt, (int)wgs, wgs * blocks * slices > cus ? 4 : 8, 0, slices};
                }
            }
        }
    return best;
}
static size_t w4_sums_bytes(int m, int k, int group) {
    return ((size_t)m * w4_sum_pitch(k, group < 128 ? group / 32 : 4) * 16 + 255) / 256 * 256;
}
static size_t w4_partial_bytes(const W4Plan &pl, int m, int n, int k, int group) {
    if (pl.tb) return w4_sums_bytes(m, k, group) + (pl.slices > 1 ? (size_t)pl.slices * m * n * 4 : 0);
    if (pl.slices <= 1) return 0;
    return (size_t)pl.slices * pl.wgs * pl.r * ((m + 16 * pl.tt - 1) / (16 * pl.tt) * pl.tt) * 1024;
}

template <class T, int GS>
static int w4_stream_of(const W4GemmArgs &a, const W4Plan &pl, hipStream_t s) {
    return a.A.zeros ? w4_launch_stream<T, GS, true>(a, pl.r, pl.tt, pl.wgs, pl.waves, s) : w4_launch_stream<T, GS, false>(a, pl.r, pl.tt, pl.wgs, pl.waves, s);
}

static int w4_stream(const W4GemmArgs &a, const W4Plan &pl, int x_kind, int group, hipStream_t s) {
    const bool f16 = x_kind == MLK_F16;
    if (group == 32) return f16 ? w4_stream_of<F16, 1>(a, pl, s) : w4_stream_of<BF16, 1>(a, pl, s);
    if (group == 64) return f16 ? w4_stream_of<F16, 2>(a, pl, s) : w4_stream_of<BF16, 2>(a, pl, s);
    return f16 ? w4_stream_of<F16, 4>(a, pl, s) : w4_stream_of<BF16, 4>(a, pl, s);
}

template <class T, int GS>
static int w4_panel_of(const W4PanelArgs &a, int tb, hipStream_t s) {
    return a.A.zeros ? w4_launch_panel<T, GS, true>(a, tb, s) : w4_launch_panel<T, GS, false>(a, tb, s);
}

static int w4_panel(const W4PanelArgs &a, int tb, int x_kind, int group, hipStream_t s) {
    const bool f16 = x_kind == MLK_F16;
    if (group == 32) return f16 ? w4_panel_of<F16, 1>(a, tb, s) : w4_panel_of<BF16, 1>(a, tb, s);
    if (group == 64) return f16 ? w4_panel_of<F16, 2>(a, tb, s) : w4_panel_of<BF16, 2>(a, tb, s);
    return f16 ? w4_panel_of<F16, 4>(a, tb, s) : w4_panel_of<BF16, 4>(a, tb, s);
}

// ------------------------------------------------------------------------------------------------------------ relayout
// Codes: a thread makes one dword of the layout.  Both sides are read and written in runs of 64 bytes at least (a tile row of 128 codes).
template <bool PACK>
__global__ void __launch_bounds__(256) w4_codes_kernel(const uint32_t *__restrict__ src, uint32_t *__restrict__ dst, int64_t total, int tiles) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        // i counts the layout's dwords: [row group][tile][lane = 16 o + r][j]; the row-major dword is 16 tile + 4 j + o of the row
        const int j = (int)i & 3, r = (int)(i >> 2) & 15, o = (int)(i >> 6) & 3;
        const int64_t tile = i >> 8, rg = tile / tiles;
        const int64_t at = (rg * 16 + r) * tiles * 16 + (tile - rg * tiles) * 16 + 4 * j + o;
        const uint32_t d = src[PACK ? at : i];
        uint32_t out = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int nib = (c >> 1) + 4 * (c & 1);            // of code c in the layout
            out |= PACK ? ((d >> (4 * c)) & 15u) << (4 * nib) : ((d >> (4 * nib)) & 15u) << (4 * c);
        }
        dst[PACK ? i : at] = out;
    }
}

// Scales and zero points: [rows][K / G] -> [row group][K / max(G, 128)][16][per], per = max(1, 128 / G).
template <typename E, bool PACK>
__global__ void __launch_bounds__(256) w4_scales_kernel(const E *__restrict__ src, E *__restrict__ dst, int64_t total, int groups, int per) {
    const int blocks = groups / per;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int g = (int)(i % per);
        const int64_t a = i / per, b = a >> 4, rg = b / blocks;
        const int64_t at = (rg * 16 + (a & 15)) * groups + (b - rg * blocks) * per + g;
        dst[PACK ? i : at] = src[PACK ? at : i];
    }
}

static int w4_grid(int64_t total) {
    const int64_t wgs = (total + 255) / 256;
    return (int)(wgs < 16384 ? wgs : 16384);
}

static bool w4_group_ok(int k, int group) { return group == 32 || group == 64 || (group >= 128 && group % 128 == 0 && k % group == 0); }

static int w4_codes(const void *src, void *dst, int64_t batch, int n, int k, void *stream, bool pack) {
    MLK_REQUIRE(batch >= 0 && n >= 0 && k >= 0, "w4 layout: negative size");
    MLK_REQUIRE(n % 16 == 0 && k % 128 == 0, "w4 layout: N % 16 and K % 128 must be 0");
    const int64_t total = batch * n * (k / 8);
    if (total == 0) return MLK_OK;
    MLK_REQUIRE(src && dst && (((uintptr_t)src | (uintptr_t)dst) & 3) == 0, "w4 layout: codes must lie on 4 bytes");
    if (pack) w4_codes_kernel<true><<<w4_grid(total), 256, 0, (hipStream_t)stream>>>((const uint32_t *)src, (uint32_t *)dst, total, k / 128);
    else w4_codes_kernel<false><<<w4_grid(total), 256, 0, (hipStream_t)stream>>>((const uint32_t *)src, (uint32_t *)dst, total, k / 128);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

static int w4_scales(const void *src, void *dst, int64_t batch, int n, int k, int group, int elem_size, void *stream, bool pack) {
    MLK_REQUIRE(batch >= 0 && n >= 0 && k >= 0, "w4 layout: negative size");
    MLK_REQUIRE(n % 16 == 0 && k % 128 == 0, "w4 layout: N % 16 and K % 128 must be 0");
    MLK_REQUIRE(w4_group_ok(k, group), "w4 layout: the group must be 32, 64 or a multiple of 128 that divides K");
    MLK_REQUIRE(elem_size == 1 || elem_size == 2, "w4 layout: scales have 2 bytes, zero points 1");
    const int groups = k / group, per = group < 128 ? 128 / group : 1;
    const int64_t total = batch * n * groups;
    if (total == 0) return MLK_OK;
    MLK_REQUIRE(src && dst, "w4 layout: null pointer");
    const int grid = w4_grid(total);
    hipStream_t s = (hipStream_t)stream;
    if (elem_size == 2 && pack) w4_scales_kernel<uint16_t, true><<<grid, 256, 0, s>>>((const uint16_t *)src, (uint16_t *)dst, total, groups, per);
    else if (elem_size == 2) w4_scales_kernel<uint16_t, false><<<grid, 256, 0, s>>>((const uint16_t *)src, (uint16_t *)dst, total, groups, per);
    else if (pack) w4_scales_kernel<uint8_t, true><<<grid, 256, 0, s>>>((const uint8_t *)src, (uint8_t *)dst, total, groups, per);
    else w4_scales_kernel<uint8_t, false><<<grid, 256, 0, s>>>((const uint8_t *)src, (uint8_t *)dst, total, groups, per);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

int mlk_pack_layout_a_w4(const void *src, void *dst, int64_t batch, int n, int k, void *stream) { return w4_codes(src, dst, batch, n, k, stream, true); }
int mlk_unpack_layout_a_w4(const void *src, void *dst, int64_t batch, int n, int k, void *stream) { return w4_codes(src, dst, batch, n, k, stream, false); }
int mlk_pack_scales_w4(const void *src, void *dst, int64_t batch, int n, int k, int group, int elem_size, void *stream) {
    return w4_scales(src, dst, batch, n, k, group, elem_size, stream, true);
}
int mlk_unpack_scales_w4(const void *src, void *dst, int64_t batch, int n, int k, int group, int elem_size, void *stream) {
    return w4_scales(src, dst, batch, n, k, group, elem_size, stream, false);
}

int mlk_gemm_layout_a_w4(const void *a, const void *scale, const void *zero, const void *b, void *c, int m, int n, int k, int group, int x_kind,
                         float alpha, const void *bias, void *workspace, size_t workspace_bytes, void *stream) {
    MLK_REQUIRE(m >= 0 && n >= 0 && k > 0, "w4 gemm: negative size");
    MLK_REQUIRE(n % 16 == 0 && k % 128 == 0, "w4 gemm: N % 16 and K % 128 must be 0");
    MLK_REQUIRE(w4_group_ok(k, group), "w4 gemm: the group must be 32, 64 or a multiple of 128 that divides K");
    MLK_REQUIRE(k < (1 << 23), "w4 gemm: K must be below 2^23");
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16, "w4 gemm: activations must be fp16 or bf16");
    if (m == 0 || n == 0) return MLK_OK;
    MLK_REQUIRE(a && scale && b && c, "w4 gemm: null pointer");
    MLK_REQUIRE(aligned16(a) && aligned16(b) && aligned16(c) && aligned16(workspace), "w4 gemm: weights, activations, outputs and workspace must lie on 16 bytes");
    MLK_REQUIRE(((uintptr_t)scale & 7) == 0 && ((uintptr_t)zero & 3) == 0, "w4 gemm: scales must lie on 8 bytes, zero points on 4");
    const W4Plan pl = w4_plan(m, n, k, group);
    const size_t part = w4_partial_bytes(pl, m, n, k, group);
    if (part && (!workspace || workspace_bytes < kCounterBytes + part)) return fail(MLK_ERR_WORKSPACE, "w4 gemm: workspace too small");
    const W4Matrix w = {(const uint8_t *)a, (const uint16_t *)scale, (const uint8_t *)zero};
    const int blocks = k / (group > 128 ? group : 128);
    const uint32_t inv = w4_inverse(group > 128 ? group / 128 : 1);
    if (pl.tb) {
        W4PanelArgs p = {};
        p.A = w;
        p.X = (const uint16_t *)b;
        p.C = (uint16_t *)c;
        p.bias = (const uint16_t *)bias;
        p.alpha = alpha;
        p.M = m;
        p.N = n;
        p.K = k;
        p.blocks = blocks;
        p.inv = inv;
        p.slices = pl.slices;
        p.sums = (u32x4 *)((uint8_t *)workspace + kCounterBytes);
        p.partial = (float *)((uint8_t *)workspace + kCounterBytes + w4_sums_bytes(m, k, group));
        return w4_panel(p, pl.tb, x_kind, group, (hipStream_t)stream);
    }
    W4GemmArgs p = {};
    p.A = w;
    p.bias = (const uint16_t *)bias;
    p.alpha = alpha;
    p.N = n;
    p.K = k;
    p.blocks = blocks;
    p.inv = inv;
    p.slices = pl.slices;
    p.counters = part ? (int *)workspace : nullptr;
    p.partial = part ? (f32x4 *)((uint8_t *)workspace + kCounterBytes) : nullptr;
    p.M = m;
    p.X = (const uint16_t *)b;
    p.C = (uint16_t *)c;
    return w4_stream(p, pl, x_kind, group, (hipStream_t)stream);
}

size_t mlk_gemm_w4_workspace_bytes(int m, int n, int k, int group) {
    if (m <= 0 || n <= 0 || k <= 0 || !w4_group_ok(k, group)) return 0;
    const size_t part = w4_partial_bytes(w4_plan(m, n, k, group), m, n, k, group);
    return part ? kCounterBytes + part : 0;
}

}  // extern "C"
