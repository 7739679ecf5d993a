// Linear layers over 4-bit weights: one token (GeMV) to prefill-sized batches.
#include "mlk_w4_gemm.cuh"

namespace mlk {

#define MLK_W4_EXTERN(T, GS)                                                                          \
    extern template int w4_launch_stream<T, GS, false>(const W4GemmArgs &, int, int, int, hipStream_t); \
    extern template int w4_launch_stream<T, GS, true>(const W4GemmArgs &, int, int, int, hipStream_t);
MLK_W4_EXTERN(F16, 4)
MLK_W4_EXTERN(F16, 2)
MLK_W4_EXTERN(F16, 1)
MLK_W4_EXTERN(BF16, 4)
MLK_W4_EXTERN(BF16, 2)
MLK_W4_EXTERN(BF16, 1)
#undef MLK_W4_EXTERN

struct W4Plan {
    int r, wgs, waves;
};

// Up to 64 tokens.
static W4Plan w4_plan_stream(int m, int n) {
    const int groups = n / 16, cus = device_cus(), most = m <= 16 ? 8 : 4;
    W4Plan pl;
    pl.r = 1;
    while (pl.r < most && groups > pl.r * cus) pl.r *= 2;
    pl.wgs = groups <= cus ? groups : (groups + pl.r * cus - 1) / (pl.r * cus) * cus;
    if (pl.wgs > groups) pl.wgs = groups;
    pl.waves = m == 1 && pl.r <= 2 ? 16 : 8;
    return pl;
}

template <class T, int GS>
static int w4_stream_of(const W4GemmArgs &a, hipStream_t s) {
    const W4Plan pl = w4_plan_stream(a.M, a.N);
    return a.A.zeros ? w4_launch_stream<T, GS, true>(a, pl.r, pl.wgs, pl.waves, s) : w4_launch_stream<T, GS, false>(a, pl.r, pl.wgs, pl.waves, s);
}

static int w4_stream(const W4GemmArgs &a, int x_kind, int group, hipStream_t s) {
    const bool f16 = x_kind == MLK_F16;
    if (group == 32) return f16 ? w4_stream_of<F16, 1>(a, s) : w4_stream_of<BF16, 1>(a, s);
    if (group == 64) return f16 ? w4_stream_of<F16, 2>(a, s) : w4_stream_of<BF16, 2>(a, s);
    return f16 ? w4_stream_of<F16, 4>(a, s) : w4_stream_of<BF16, 4>(a, s);
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
    MLK_REQUIRE(aligned16(a) && aligned16(b), "w4 gemm: weights and activations must lie on 16 bytes");
    MLK_REQUIRE(((uintptr_t)scale & 7) == 0 && ((uintptr_t)zero & 3) == 0, "w4 gemm: scales must lie on 8 bytes, zero points on 4");
    W4GemmArgs p;
    p.A = W4Matrix{(const uint8_t *)a, (const uint16_t *)scale, (const uint8_t *)zero};
    p.bias = (const uint16_t *)bias;
    p.alpha = alpha;
    p.N = n;
    p.K = k;
    p.blocks = k / (group > 128 ? group : 128);
    p.inv = w4_inverse(group > 128 ? group / 128 : 1);
    p.slices = 1;
    p.partial = nullptr;
    p.counters = nullptr;
    for (int m0 = 0; m0 < m; m0 += 64) {
        p.M = m - m0 < 64 ? m - m0 : 64;
        p.X = (const uint16_t *)b + (size_t)m0 * k;
        p.C = (uint16_t *)c + (size_t)m0 * n;
        const int rc = w4_stream(p, x_kind, group, (hipStream_t)stream);
        if (rc != MLK_OK) return rc;
    }
    return MLK_OK;
}

size_t mlk_gemm_w4_workspace_bytes(int m, int n, int k) { return 0; }

}  // extern "C"
