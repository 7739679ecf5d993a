// Quantising activations to e4m3, and the linear layers in e4m3: one token to prefill-sized batches.
#include <algorithm>

#include "mlk_f8_panel.cuh"

namespace mlk {

// ---------------------------------------------------------------------------------------------------------------- quantising
// Sixteen lanes take a block of 128, so the maximum is four exchanges within 16 lanes; a workgroup takes 16 tokens and NB consecutive blocks of each, whose loads
// are in flight together: runs of 256 NB bytes, and the scales of 16 tokens side by side.
template <class T, int NB>
__global__ void __launch_bounds__(256) f8_quantize_kernel(const void *__restrict__ x, uint8_t *__restrict__ codes, float *__restrict__ scales, int64_t scale_t,
                                                          int64_t scale_k, int64_t tokens, int blocks) {
    const int64_t token = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int l = threadIdx.x & 15, kb0 = blockIdx.y * NB;
    if (token >= tokens) return;
    const size_t row = (size_t)token * blocks * kF8K;
    F8In<T> in[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (kb0 + b < blocks) in[b].load(x, row + (size_t)(kb0 + b) * kF8K + l * 8);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (kb0 + b >= blocks) break;
        float v[8], scale;
        in[b].values(v);
        const u32x2 q = f8_block(v, scale);
        *reinterpret_cast<u32x2 *>(codes + row + (size_t)(kb0 + b) * kF8K + l * 8) = q;
        if (l == 0) scales[token * scale_t + (kb0 + b) * scale_k] = scale;
    }
}

int launch_quantize_fp8(const void *x, int x_kind, uint8_t *codes, float *scales, int64_t scale_t, int64_t scale_k, int64_t T, int K, hipStream_t s) {
    constexpr int NB = 4;
    const int blocks = K / kF8K;
    const dim3 grid((unsigned)((T + 15) / 16), (blocks + NB - 1) / NB);
    if (x_kind == MLK_F32) f8_quantize_kernel<float, NB><<<grid, 256, 0, s>>>(x, codes, scales, scale_t, scale_k, T, blocks);
    else if (x_kind == MLK_F16) f8_quantize_kernel<F16, NB><<<grid, 256, 0, s>>>(x, codes, scales, scale_t, scale_k, T, blocks);
    else f8_quantize_kernel<BF16, NB><<<grid, 256, 0, s>>>(x, codes, scales, scale_t, scale_k, T, blocks);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

// ---------------------------------------------------------------------------------------------------------------- streaming
struct F8GemmArgs {
    const uint8_t *A;
    const float *a_scale;        // [ceil(N / 128)][K / 128]
    const uint8_t *X;            // [M][K]
    const float *x_scale;        // token t's window kb at t xs_t + kb xs_k
    int64_t xs_t, xs_k;
    uint16_t *C;
    const uint16_t *bias;
    float alpha;
    int M, N, K;
};

// A workgroup owns up to R consecutive row groups and TT blocks of 16 tokens (blockIdx.y); its waves deal the windows of 128 k among themselves (window t to wave
// t mod waves, so that together they read each row group front to back) and add their sums through LDS in wave order.
constexpr int kF8Waves = 8;
template <class T, int TT, int R>
__global__ void __launch_bounds__(kF8Waves * 64) f8_stream_kernel(F8GemmArgs p) {
    extern __shared__ f32x4 red[];
    constexpr int CELLS = R * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int windows = p.K / kF8K, groups = p.N / 16, rg0 = blockIdx.x * R, m0 = blockIdx.y * (TT * 16);
    F8Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) f8_row(rows, r, p.A, p.a_scale, min(rg0 + r, groups - 1), windows);
    F8Tokens<TT> tokens;
    tokens.step = p.xs_k;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
        const int64_t t = min(m0 + tt * 16 + (lane & 15), p.M - 1);
        tokens.x[tt] = p.X + t * p.K;
        tokens.a[tt] = p.x_scale + t * p.xs_t;
    }
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    f8_stream<TT, R, (CELLS <= 2 ? 4 : 2)>(acc, rows, tokens, wave, windows, kF8Waves, lane);
#pragma unroll
    for (int c = 0; c < CELLS; ++c) red[(wave * CELLS + c) * 64 + lane] = acc[c / TT][c % TT];
    __syncthreads();
    for (int c = wave; c < CELLS; c += kF8Waves) {
        const int r = c / TT, token = m0 + (c - r * TT) * 16 + (lane & 15), n = (rg0 + r) * 16 + (lane >> 4) * 4;
        f32x4 v = red[c * 64 + lane];
        for (int w = 1; w < kF8Waves; ++w) v += red[(w * CELLS + c) * 64 + lane];
        if (rg0 + r >= groups || token >= p.M) continue;
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = p.alpha * v[i] + (p.bias ? T::to_f32(p.bias[n + i]) : 0.f);
        *reinterpret_cast<u32x2 *>(p.C + (size_t)token * p.N + n) = u32x2{T::from_f32x2(o[0], o[1]), T::from_f32x2(o[2], o[3])};
    }
}

template <class T, int TT, int R>
static int f8_launch_stream(const F8GemmArgs &a, hipStream_t s) {
    f8_stream_kernel<T, TT, R><<<dim3((a.N / 16 + R - 1) / R, (a.M + TT * 16 - 1) / (TT * 16)), kF8Waves * 64, (size_t)kF8Waves * R * TT * 1024, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

// Panels move and multiply like those of a 16-bit product of half the k: as many bytes, and the matrix cores take twice as many k in the time.
extern template int f8_launch_panel<F16>(const F8PanelArgs &, int, int, hipStream_t);
extern template int f8_launch_panel<BF16>(const F8PanelArgs &, int, int, hipStream_t);
size_t panel8_arguments(Panel8Args &p, int m, int n, int k, int pr, int tb, int p3);
void gemm_plan(int m, int n, int k, bool fp8, bool b_native, int32_t *out);

struct F8Plan {
    bool panels;
    int pr, tb, p3;
};
static F8Plan f8_plan(int m, int n, int k) {
    F8Plan pl = {};
    // offsets within a panel are 32 bits
    if (m <= 64 || k >= 1 << 23) return pl;
    int32_t out[4];
    gemm_plan(m, n, k / 2, false, false, out);
    pl.panels = true;
    pl.pr = out[1] / 2;
    pl.tb = out[2];
    pl.p3 = out[3];
    return pl;
}
template <class T>
static int f8_launch_gemm(const F8GemmArgs &a, const F8Plan &pl, void *partial, size_t partial_bytes, hipStream_t s) {
    if (pl.panels) {
        F8PanelArgs g = {};
        g.p.A = a.A;
        g.p.B = reinterpret_cast<const uint16_t *>(a.X);
        g.p.C = a.C;
        g.p.bias = a.bias;
        g.p.scale = a.a_scale;
        g.p.partial = (f32x4 *)partial;
        g.p.alpha = a.alpha;
        if (panel8_arguments(g.p, a.M, a.N, a.K / 2, pl.pr, pl.tb, pl.p3) > partial_bytes) return fail(MLK_ERR_WORKSPACE, "gemm fp8: workspace too small");
        g.x_scale = a.x_scale;
        g.xs_t = (uint32_t)a.xs_t;
        g.xs_k = (uint32_t)a.xs_k;
        return f8_launch_panel<T>(g, pl.pr, pl.tb, s);
    }
    if (a.M <= 16) return f8_launch_stream<T, 1, 2>(a, s);
    return f8_launch_stream<T, 2, 2>(a, s);
}

struct F8Scratch {
    uint8_t *codes;
    float *scales;
    void *partial;
    size_t partial_bytes;
};
static size_t f8_carve(uint8_t *base, int m, int n, int k, bool quantize, F8Scratch *out) {
    const F8Plan pl = f8_plan(m, n, k);
    Panel8Args p = {};
    const size_t partial = pl.panels ? panel8_arguments(p, m, n, k / 2, pl.pr, pl.tb, pl.p3) : 0;
    if (!quantize && partial == 0) {
        if (out) *out = F8Scratch{};
        return 0;
    }
    size_t off = kCounterBytes;
    auto take = [&](size_t bytes) {
        uint8_t *ptr = base ? base + off : nullptr;
        off = (off + bytes + 255) / 256 * 256;
        return ptr;
    };
    F8Scratch w;
    w.codes = take(quantize ? (size_t)m * k : 0);
    w.scales = (float *)take(quantize ? (size_t)m * (k / kF8K) * 4 : 0);
    w.partial = take(partial);
    w.partial_bytes = partial;
    if (out) *out = w;
    return off;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

int mlk_quantize_fp8(const void *x, int x_kind, void *codes, float *scales, int64_t scale_t, int64_t scale_k, int64_t n_tokens, int k, void *stream) {
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16 || x_kind == MLK_F32, "quantize_fp8: activations must be fp16, bf16 or fp32");
    MLK_REQUIRE(n_tokens >= 0 && n_tokens <= (1ll << 27), "quantize_fp8: 0..2^27 rows");
    MLK_REQUIRE(k >= 0 && k % 128 == 0 && k / 512 < 65535, "quantize_fp8: K % 128 must be 0, K below 2^25");
    if (n_tokens == 0 || k == 0) return MLK_OK;
    MLK_REQUIRE(x && codes && scales, "quantize_fp8: null pointer");
    MLK_REQUIRE(aligned16(x) && aligned16(codes), "quantize_fp8: activations and codes must lie on 16 bytes");
    return launch_quantize_fp8(x, x_kind, (uint8_t *)codes, scales, scale_t, scale_k, n_tokens, k, (hipStream_t)stream);
}

size_t mlk_gemm_fp8_workspace_bytes(int m, int n, int k, int b_kind) {
    if (m <= 0 || n <= 0 || k <= 0 || k % 128 != 0) return 0;
    return f8_carve(nullptr, m, n, k, b_kind != MLK_FP8_E4M3, nullptr);
}

int mlk_gemm_layout_a_fp8(const void *a, const float *a_scale, const void *b, int b_kind, const float *b_scale, int64_t b_scale_t, int64_t b_scale_k, void *c,
                          int c_kind, int m, int n, int k, float alpha, const void *bias, void *workspace, size_t workspace_bytes, void *stream) {
    MLK_REQUIRE(c_kind == MLK_F16 || c_kind == MLK_BF16, "gemm fp8: outputs must be fp16 or bf16");
    MLK_REQUIRE(b_kind == MLK_FP8_E4M3 || b_kind == c_kind, "gemm fp8: activations must be e4m3 codes or of the output's kind");
    MLK_REQUIRE(m >= 0, "gemm fp8: negative token count");
    MLK_REQUIRE(n > 0 && k > 0 && n % 16 == 0 && k % 128 == 0 && k < (1 << 25), "gemm fp8: N % 16 and K % 128 must be 0, K below 2^25");
    if (m == 0) return MLK_OK;
    MLK_REQUIRE(a && a_scale && b && c && (b_kind != MLK_FP8_E4M3 || b_scale), "gemm fp8: null pointer");
    MLK_REQUIRE(aligned16(a) && aligned16(b) && aligned16(c), "gemm fp8: weights, activations and outputs must lie on 16 bytes");
    if (workspace_bytes < mlk_gemm_fp8_workspace_bytes(m, n, k, b_kind)) return fail(MLK_ERR_WORKSPACE, "gemm fp8: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    F8GemmArgs p = {};
    p.A = (const uint8_t *)a;
    p.a_scale = a_scale;
    p.X = (const uint8_t *)b;
    p.x_scale = b_scale;
    p.xs_t = b_scale_t;
    p.xs_k = b_scale_k;
    p.C = (uint16_t *)c;
    p.bias = (const uint16_t *)bias;
    p.alpha = alpha;
    p.M = m;
    p.N = n;
    p.K = k;
    F8Scratch w;
    if (f8_carve((uint8_t *)workspace, m, n, k, b_kind != MLK_FP8_E4M3, &w) > 0)
        MLK_REQUIRE(workspace && aligned16(workspace), "gemm fp8: workspace off 16 bytes");
    F8Plan pl = f8_plan(m, n, k);
    if (b_kind != MLK_FP8_E4M3) {
        const int rc = launch_quantize_fp8(b, b_kind, w.codes, w.scales, 1, m, m, k, s);
        if (rc != MLK_OK) return rc;
        p.X = w.codes;
        p.x_scale = w.scales;
        p.xs_t = 1;
        p.xs_k = m;
    } else if (b_scale_t < 0 || b_scale_k < 0 || b_scale_t >= 1 << 21 || b_scale_k >= (1ll << 29) / (k / kF8K)) {
        pl.panels = false;                                     // scales that far apart: the panels' offsets of them are 32 bits
    }
    return c_kind == MLK_F16 ? f8_launch_gemm<F16>(p, pl, w.partial, w.partial_bytes, s) : f8_launch_gemm<BF16>(p, pl, w.partial, w.partial_bytes, s);
}

}  // extern "C"
