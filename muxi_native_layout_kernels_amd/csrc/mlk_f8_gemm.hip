// Quantising activations to e4m3, and the linear layers in e4m3: one token to prefill-sized batches.
#include <algorithm>

#include "mlk_f8_panel.cuh"

namespace mlk {

// ---------------------------------------------------------------------------------------------------------------- quantising
// Sixteen lanes take a block of 128, so the maximum is four exchanges within 16 lanes; a workgroup takes 16 tokens and NB consecutive blocks of each, whose loads
// are in flight together: runs of 256 NB bytes, and the scales of 16 tokens side by side.  Bound by the bytes: 8191 x 14336 of fp16 60 us, 356 MB at 5.9 TB/s; 32 x 7168 3.1 us, the launch.
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

constexpr int kF8MostK = 65535 * 512;   // of the quantising kernel's grid, whose workgroups take 512 k
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
    const uint8_t *X;            // [M][K] codes
    const float *x_scale;        // token t's window kb at t xs_t + kb xs_k
    int64_t xs_t, xs_k;
    const void *raw;             // [M][K] activations that the kernel quantises by itself, or null
    uint16_t *C;
    const uint16_t *bias;
    float alpha;
    int M, N, K;
    int slices;
    int rg_each, rg_more;        // row groups of a workgroup; the first rg_more workgroups have one more
    f32x4 *partial;              // [workgroup (x, z)][slice][cell][two planes of 64 x 8 bytes]
    int *counters;               // [workgroup (x, z)], zero between calls
};

// Bytes of LDS that `m` staged tokens of `windows` windows take: 16 bytes between the rows, so that tokens read different banks, and their scales.
__host__ __device__ constexpr int f8_staged_pitch(int windows) { return windows * 8 + 1; }      // in pieces of 16 bytes
__host__ __device__ constexpr size_t f8_staged_bytes(int m, int windows) { return ((size_t)m * f8_staged_pitch(windows) * 16 + (size_t)m * windows * 4 + 15) / 16 * 16; }

// Windows t0 .. t0 + n - 1 of all tokens, up to four (of codes one, f8_plan), into LDS, from codes or (raw) from activations, which are quantised on the way: 16 lanes a block of 128.
template <class T>
__device__ __forceinline__ void f8_stage(const F8GemmArgs &p, u32x4 *lds, int t0, int n) {
    float *scales = reinterpret_cast<float *>(lds + (size_t)p.M * f8_staged_pitch(n));
    uint8_t *codes = reinterpret_cast<uint8_t *>(lds);
    const int l = threadIdx.x & 15, lanes = blockDim.x >> 4;
    for (int b = threadIdx.x >> 4; b < p.M * n; b += lanes) {
        const int token = b / n, t = b - token * n;
        const size_t at = (size_t)token * p.K + (size_t)(t0 + t) * kF8K + l * 8;
        u32x2 q;
        float scale;
        if (p.raw) {
            F8In<T> in;
            float v[8];
            in.raw = ld_global_u32x4(reinterpret_cast<const uint16_t *>(p.raw) + at);
            in.values(v);
            q = f8_block(v, scale);
        } else {
            q = *reinterpret_cast<const u32x2 *>(p.X + at);
            scale = p.x_scale[token * p.xs_t + (t0 + t) * p.xs_k];
        }
        *reinterpret_cast<u32x2 *>(codes + (size_t)token * f8_staged_pitch(n) * 16 + t * kF8K + l * 8) = q;
        if (l == 0) scales[token * n + t] = scale;
    }
}

// Where a workgroup has its tokens from: codes, up to four tokens in LDS (codes of one, or activations that the workgroup quantises), activations that each wave quantises for its own windows.
enum F8Feed { kF8Codes, kF8InLds, kF8Quantise };

// Bound by the weights' bytes, with more tokens by what the workgroups read of the activations.  A workgroup owns up to R consecutive row groups, which are dealt out evenly over the
// grid, and TT blocks of 16 tokens (blockIdx.z); its waves deal the windows of 128 k among themselves (window t to wave t mod waves, so that together they read each row
// group front to back) and add their sums through LDS in wave order.  `slices` workgroups may share a set of row groups, each on its own range of k: the last one to arrive adds their
// fp32 sums in the order of k.  28672 x 8192 at 16 tokens 40.6 us (5.8 TB/s; a large read reaches 6.9; 38.3 from codes), 512 x 7168 at one token 5.9 (launch, first loads and the fold of four
// slices).
template <class T, int TT, int R, int U, int FEED>
__global__ void __launch_bounds__(512) f8_stream_kernel(F8GemmArgs p) {
    extern __shared__ u32x4 lds[];
    __shared__ int s_last;
    constexpr int CELLS = R * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int windows = p.K / kF8K, b = blockIdx.x, sl = blockIdx.y, m0 = blockIdx.z * (TT * 16);
    const int rg0 = b * p.rg_each + min(b, p.rg_more), nr = p.rg_each + (b < p.rg_more ? 1 : 0);
    const int t0 = (int)((long long)windows * sl / p.slices), t1 = (int)((long long)windows * (sl + 1) / p.slices);
    F8Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) f8_row(rows, r, p.A, p.a_scale, rg0 + min(r, nr - 1), windows);
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (FEED == kF8InLds) {
        const int n = t1 - t0, token = min(lane & 15, p.M - 1);
        F8Staged tokens;
        tokens.x = lds + (size_t)token * f8_staged_pitch(n);
        tokens.a = reinterpret_cast<const float *>(lds + (size_t)p.M * f8_staged_pitch(n)) + token * n;
        tokens.first = t0;
        f8_stream_staged<R, U>(acc, rows, tokens, t0 + wave, t1, waves, lane, [&]() {
            f8_stage<T>(p, lds, t0, n);
            __syncthreads();
        });
    } else if constexpr (FEED == kF8Quantise) {
        F8RawTokens<TT> tokens;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) tokens.x[tt] = reinterpret_cast<const uint16_t *>(p.raw) + (size_t)min(m0 + tt * 16 + (lane & 15), p.M - 1) * p.K;
        f8_stream_raw<T, TT, R, U>(acc, rows, tokens, t0 + wave, t1, waves, lane);
    } else {
        F8Tokens<TT> tokens;
        tokens.step = p.xs_k;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int64_t t = min(m0 + tt * 16 + (lane & 15), p.M - 1);
            tokens.x[tt] = p.X + t * p.K;
            tokens.a[tt] = p.x_scale + t * p.xs_t;
        }
        f8_stream<TT, R, U>(acc, rows, tokens, t0 + wave, t1, waves, lane);
    }
    auto store = [&](int c, f32x4 v) {
        const int r = c / TT, token = m0 + (c - r * TT) * 16 + (lane & 15), n = (rg0 + r) * 16 + (lane >> 4) * 4;
        if (r >= nr || token >= p.M) return;
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = p.alpha * v[i] + (p.bias ? T::to_f32(p.bias[n + i]) : 0.f);
        *reinterpret_cast<u32x2 *>(p.C + (size_t)token * p.N + n) = u32x2{T::from_f32x2(o[0], o[1]), T::from_f32x2(o[2], o[3])};
    };
    const int set = blockIdx.z * gridDim.x + blockIdx.x;
    auto part = [&](int s, int c) { return p.partial + (((size_t)set * p.slices + s) * CELLS + c) * 64; };
    f32x4 *red = reinterpret_cast<f32x4 *>(lds);
    if constexpr (FEED == kF8InLds) __syncthreads();                     // the other waves still read the tokens
#pragma unroll
    for (int c = 0; c < CELLS; ++c) red[(wave * CELLS + c) * 64 + lane] = acc[c / TT][c % TT];
    __syncthreads();
    for (int c = wave; c < CELLS; c += waves) {
        f32x4 v = red[c * 64 + lane];
        for (int w = 1; w < waves; ++w) v += red[(w * CELLS + c) * 64 + lane];
        if (p.slices == 1) store(c, v);
        else st_agent_planar(part(sl, c), 64, lane, v);
    }
    if (p.slices == 1) return;
    // every wave waits for its own stores before the barrier and the arrival is counted behind it: whoever sees all the others can read their sums
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        const int before = __hip_atomic_fetch_add(&p.counters[set], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = before == p.slices - 1;
        if (s_last) __hip_atomic_store(&p.counters[set], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int c = wave; c < CELLS; c += waves)
        store(c, fold_agent_planar([&](int s) { return part(s, c); }, p.slices, 64, lane));
}

struct F8Plan {
    bool panels;
    int pr, tb, p3;              // of the panels
    int r, tt, waves, slices;    // of the streaming kernel: row groups and blocks of tokens of a workgroup
    F8Feed feed;
};

template <class T, int TT, int R, int U, int FEED>
static int f8_launch_stream_one(F8GemmArgs a, const F8Plan &pl, hipStream_t s) {
    const int groups = a.N / 16, wgs = (groups + R - 1) / R, per_slice = (a.K / kF8K + pl.slices - 1) / pl.slices;
    a.slices = pl.slices;
    a.rg_each = groups / wgs;
    a.rg_more = groups % wgs;
    size_t lds = (size_t)pl.waves * R * TT * 1024;
    if (FEED == kF8InLds) lds = std::max(lds, f8_staged_bytes(a.M, per_slice));
    if (lds > 48 * 1024) {
        static bool ready_on[64] = {};
        const int rc = panel_lds_attribute(&f8_stream_kernel<T, TT, R, U, FEED>, 150 * 1024, ready_on);
        if (rc != MLK_OK) return rc;
    }
    f8_stream_kernel<T, TT, R, U, FEED><<<dim3(wgs, pl.slices, (a.M + TT * 16 - 1) / (TT * 16)), pl.waves * 64, lds, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}
// Windows in flight: as many as fit the registers of eight waves a CU.
__host__ __device__ constexpr int f8_ring(int tt, int r) { return r == 1 && tt == 1 ? 8 : r * tt <= 2 ? 4 : (r + tt < 8 ? 2 : 1); }
__host__ __device__ constexpr int f8_raw_ring(int tt, int r) { return r * tt == 1 ? 2 : 1; }       // more registers than workgroups pay for: 4096 x 14336 at 4 tokens, two rows, two windows 15.5 us, one 14.6
template <class T>
static int f8_launch_stream(const F8GemmArgs &a, const F8Plan &pl, hipStream_t s) {
    // what f8_plan() picks
#define MLK_F8_S(R) if (pl.feed == kF8InLds && pl.r == R) return f8_launch_stream_one<T, 1, R, f8_ring(1, R), kF8InLds>(a, pl, s)
#define MLK_F8_Q(TT, R) if (pl.feed == kF8Quantise && pl.tt == TT && pl.r == R) return f8_launch_stream_one<T, TT, R, f8_raw_ring(TT, R), kF8Quantise>(a, pl, s)
#define MLK_F8_R(TT, R) if (pl.feed == kF8Codes && pl.tt == TT && pl.r == R) return f8_launch_stream_one<T, TT, R, f8_ring(TT, R), kF8Codes>(a, pl, s)
    MLK_F8_S(1);
    MLK_F8_S(2);
    MLK_F8_S(4);
    MLK_F8_Q(1, 1);
    MLK_F8_Q(1, 2);
    MLK_F8_Q(1, 4);
    MLK_F8_Q(1, 8);
    MLK_F8_Q(2, 1);
    MLK_F8_Q(2, 2);
    MLK_F8_Q(2, 4);
    MLK_F8_R(1, 1);
    MLK_F8_R(1, 2);
    MLK_F8_R(1, 4);
    MLK_F8_R(1, 8);
    MLK_F8_R(2, 1);
    MLK_F8_R(2, 2);
    MLK_F8_R(2, 4);
    MLK_F8_R(3, 2);
    MLK_F8_R(4, 2);
#undef MLK_F8_S
#undef MLK_F8_Q
#undef MLK_F8_R
    return fail(MLK_ERR_INVALID, "gemm fp8: launch parameters");
}

// Panels move and multiply like those of a 16-bit product of half the k: as many bytes, and the matrix cores take twice as many k in the time.
extern template int f8_launch_panel<F16>(const F8PanelArgs &, int, int, hipStream_t);
extern template int f8_launch_panel<BF16>(const F8PanelArgs &, int, int, hipStream_t);
size_t panel8_arguments(Panel8Args &p, int m, int n, int k, int pr, int tb, int p3);
void gemm_plan(int m, int n, int k, bool fp8, bool b_native, int32_t *out);

constexpr size_t kF8StagedLds = 140 * 1024;     // of staged tokens

// Launches that are fastest, timed in graphs on weights from memory (us; g r, tt, waves, slices of the streaming kernel, s: tokens staged in LDS, q: quantised by
// the waves that multiply them, p: panels of 128 rows x 64 tokens).  Quantised by the workgroups, activations save a launch.
//   few row groups       512 x 7168 codes g1,1,4,4 5.5, g1,1,4,1 7 and more; at 16 tokens 6.0; 1280 x 5120 g1,1,8,1 5.8, at 32 tokens g2,2,8,4 7.2, at 64 g2,4,8,4 8.8, p 10.9
//   one a CU             4096 x 4096 g1,1,8,1 5.7, g2 7.2; at 64 tokens g2,2,8,1 10.1; 4096 x 14336 at 16 tokens g4,1,4,8 14.3, g1,1,8,1 16.3; at 32 g4,2,8,4 16.4, p in eight slices 18.1; at 64 p 19.7, g 21.7
//   up to two            7168 x 2048 g2,1,4,1 5.5, 8192 x 3584 g2,1,8,1 7.5, w4 8.3; at 64 tokens g4,2,8,1 8.7; 5120 x 13824 at 8 g4,1,4,8 17.5, g2,1,8,1 19.4; at 24 p in six slices 20.0, g2,2,8,4 20.8
//   up to four           13824 x 5120 at 4 tokens g4,1,8,1 15.2, g2 15.7; at 32 g4,2,8,1 18.0, p in two slices 19.8; at 64 p 21.0, g4,4,8,1 23.7
//   more                 28672 x 8192 at 8 tokens g8,1,4,1 40.5, g2 41.8, g4 42.0; 37888 x 3584 at 8 g2,1,4,1 27.7, g8 32 and more; 28672 x 8192 at 17 p 43.2, g4,2,4,1 43.9, at 64 p 44.4, g 59.9
//   64, long k           8192 x 8192 p in four slices 24.8, g4,4,8,1 27.6, both with quantising; 4608 x 7168 in seven 19.8 and 23.4
//   quantising, s or q   512 x 7168 one token s1,1,8,4 6.0, q1,1,4,8 6.7; at 8 tokens 7.3 and 6.8; 4096 x 4096 at 2 s1,1,8,1 7.2, q2,1,8,4 7.7; at 4 8.0 and 7.7; 4608 x 7168 at 2 s2,1,8,1 11.1, q 11.9; 8192 x 8192 at
//                        2 15.6 and 14.3; 37888 x 3584 at 2 s2,1,4,1 24.9, q4,1,8,1 26.9; 28672 x 8192 at 2 39.4, q8,1,4,1 41.1; at 4 43.3 and 41.0; 16000 x 1024 at 2 s4,1,8,1 5.8, q 6.3
//   quantising, q or a launch ahead of g or p    512 x 7168 at 16 tokens q1,1,4,8 7.1, g 9.1; at 32 q1,2,4,8 8.2, g 10.0; 4096 x 4096 at 16 q2,1,8,4 8.2, g 10.7; at 32 q4,2,8,4 10.0, g 11.7; 4096 x 14336 at 8 q4,1,8,4 14.5,
//                        g 17.9; at 32 19.3 and 21.3; 3584 x 18944 at 32 25.0 and 23.6; 2048 x 2048 at 7 q1,1,8,1 5.3, in two slices of two rows 6.1, s and g 5.5; 7168 x 2048 at 16 q2,1,8,1 6.5, g 9.0; at 24 8.1 and
//                        10.2; 8192 x 8192 at 32 23.9 and 21.8; 5120 x 13824 at 16 q4,1,8,4 21.9, q2,1,8,1 23.5, g 21.2; at 32 35 and 23.5; 13824 x 5120 at 8 q4,1,8,1 15.7, g 19.2; at 24 20.5 and 22.1, at 32 24.3 and 22.8;
//                        22016 x 4096 at 7 q2,1,4,1 20.2, q4,1,8,1 22.0, g 21.1; 28672 x 8192 at 16 q8,1,4,1 40.7, g 44.0; at 24 q4,2,4,1 54.8, p 49.6
//   staged codes         one token of large weights only: 28672 x 8192 38.1, g 40.8; 4096 x 14336 13.1, g 14.1; 4096 x 4096 6.2, g 5.7
static bool f8_panels_fit(int k) { return k < 1 << 23; }            // offsets within a panel are 32 bits
static bool f8_deep(int k) { return k / kF8K >= 96; }                // slices bring workgroups of a few row groups back
// Whether the panels' own plan is taken: from some number of tokens on, 257 at the latest.
static bool f8_wide(int m, int n, int k) {
    const int groups = n / 16, cus = device_cus();
    // up to 256 tokens through few rows: 512 x 7168 at 200 tokens g4,2,8,4 9.4, panels 12.2; at 300 12.5; 4096 x 4096 at 100 g4,2,8,1 12.6, panels 14.9; at 200 16.5
    const bool narrow = m <= 64 || (m <= 128 && groups <= cus && !f8_deep(k)) || (m <= 256 && groups <= cus / 4);
    return !narrow && f8_panels_fit(k);
}
static F8Plan f8_plan(int m, int n, int k, bool raw) {
    F8Plan pl = {};
    const int groups = n / 16, windows = k / kF8K, cus = device_cus();
    const bool panels_fit = f8_panels_fit(k), deep = f8_deep(k);
    const int rows = (n + 127) / 128;
    auto panels = [&](int pr, int tb, int p3) {
        pl.panels = true;
        pl.pr = pr;
        pl.tb = tb;
        pl.p3 = std::max(1, p3);
        return pl;
    };
    if (f8_wide(m, n, k)) {
        int32_t out[4];
        gemm_plan(m, n, k / 2, false, false, out);
        return panels(out[1] / 2, out[2], out[3]);
    }
    auto stream = [&](int r, int tt, int waves, int slices) {
        pl.r = r;
        pl.tt = tt;
        pl.waves = waves;
        pl.slices = std::max(1, std::min(slices, windows / waves));
    };
    const int blocks = std::min((m + 15) / 16, 4), thin = windows >= 32 ? 4 : 1, many = windows >= 16 ? 8 : 4;
    // in LDS
    const bool lds = raw ? m <= 4 && (groups <= cus / 4 || (m <= 2 && groups <= cus && !deep) || (m <= 2 && groups <= cus * 3 / 2) || (m == 1 && groups <= 2 * cus) ||
                                      (m <= 2 && (groups > 4 * cus || (groups > 2 * cus && windows < 16))))
                         : m == 1 && (int64_t)n * k >= 50000000;
    if (lds) {
        if (groups <= cus / 4) stream(1, 1, 8, thin);
        else if (groups <= cus) stream(m * windows > 200 ? 2 : 1, 1, 8, m * windows > 200 ? 4 : 1);
        else if (groups <= 2 * cus) stream(2, 1, deep ? 4 : 8, deep ? 4 : 1);
        else if (groups <= 3 * cus) stream(4, 1, 8, 1);
        else stream(2, 1, 4, 1);
        if (f8_staged_bytes(m, (windows + pl.slices - 1) / pl.slices) <= kF8StagedLds) {
            pl.feed = kF8InLds;
            return pl;
        }
    }
    // quantised by the waves
    const bool two = m > 16 && m <= 32 && (groups <= cus ? m * windows <= 4096 : groups <= 2 * cus ? windows <= 32 : groups <= 4 * cus && m * windows <= 1000);
    if (raw && (m <= 16 || two)) {
        const int tt = two ? 2 : 1;
        pl.feed = kF8Quantise;
        if (groups <= cus / 4) stream(1, tt, 4, windows >= 16 ? 8 : 1);
        else if (groups <= cus && windows < 32) stream(1, tt, many, 1);
        else if (groups <= cus) stream(two || deep ? 4 : 2, tt, 8, 4);
        else if (groups <= 2 * cus && deep) stream(4, tt, 8, 4);
        else if (groups <= 2 * cus) stream(2, tt, many, 1);
        else if (groups <= 4 * cus) stream(4, tt, many, 1);
        else if (windows < 48) stream(groups < 6 * cus ? 2 : 4, tt, groups < 6 * cus ? 4 : many, 1);
        else stream(8, tt, 4, 1);
        return pl;
    }
    if (panels_fit && ((m > 16 && (groups > 4 * cus || (deep && groups > cus))) || (m > 32 && m <= 64 && (groups > 2 * cus || (windows >= 48 && groups > cus) || (deep && groups > cus / 2)))))
        return panels(1, 1, std::min(cus / rows, windows / 12));
    if (m <= 16) {
        if (groups <= cus / 4) stream(1, 1, 4, thin);
        else if (groups <= 2 * cus && deep) stream(4, 1, 4, 8);
        else if (groups <= cus) stream(1, 1, 8, 1);
        else if (groups <= 2 * cus) stream(2, 1, windows >= 24 ? 8 : 4, 1);
        else if (groups <= 4 * cus) stream(4, 1, 8, 1);
        else stream(windows >= 48 ? 8 : 2, 1, 4, 1);
    } else {
        if (groups <= cus / 4 && m <= 64) stream(1, 2, 8, thin);
        // more than 256 tokens come here only with k that the panels do not take: whole, as arrivals of any number of tokens do not fit the counters
        else if (m > 64) stream(m > 128 || groups > cus / 2 ? 4 : 2, 2, 8, groups <= cus / 4 && m <= 256 ? thin : 1);
        else if (groups <= cus / 2) stream(2, blocks, 8, 4);
        else if (groups <= cus && deep) stream(4, 2, 8, 4);
        else if (groups <= cus) stream(m <= 32 ? 1 : 2, 2, 8, 1);
        else if (groups <= 2 * cus && m <= 48) stream(2, blocks, 8, 1);
        else stream(4, 2, 8, 1);
    }
    return pl;
}

static size_t f8_partial_bytes(const F8Plan &pl, int m, int n, int k) {
    Panel8Args p = {};
    if (pl.panels) return panel8_arguments(p, m, n, k / 2, pl.pr, pl.tb, pl.p3);
    if (pl.slices == 1) return 0;
    const size_t sets = (size_t)((n / 16 + pl.r - 1) / pl.r) * ((m + pl.tt * 16 - 1) / (pl.tt * 16));
    return sets * pl.slices * pl.r * pl.tt * 1024;
}
struct F8Scratch {
    uint8_t *codes;
    float *scales;
    void *partial;
    size_t partial_bytes;
};
// quantize: activations that the call quantises with a launch of its own
static size_t f8_carve(uint8_t *base, size_t partial, int m, int k, bool quantize, F8Scratch *out) {
    F8Scratch w = {};
    size_t off = 0;
    if (quantize || partial > 0) {
        off = kCounterBytes;
        auto take = [&](size_t bytes) {
            uint8_t *ptr = base ? base + off : nullptr;
            off = (off + bytes + 255) / 256 * 256;
            return ptr;
        };
        w.codes = take(quantize ? (size_t)m * k : 0);
        w.scales = (float *)take(quantize ? (size_t)m * (k / kF8K) * 4 : 0);
        w.partial = take(partial);
        w.partial_bytes = partial;
    }
    if (out) *out = w;
    return off;
}
static bool f8_quantises(const F8Plan &pl, bool raw) { return raw && pl.feed == kF8Codes; }
static size_t f8_call_bytes(const F8Plan &pl, int m, int n, int k, bool raw) { return f8_carve(nullptr, f8_partial_bytes(pl, m, n, k), m, k, f8_quantises(pl, raw), nullptr); }
// The most that a call of 1 .. m tokens takes.  The panels' plan follows from the tokens' number of blocks of 64, and within one the last count takes most.  Above 16384 tokens the
// bound of all plans: a slot of at most 256 x 256 sums a CU where panels are cut in slices, two where they are dealt.
static size_t f8_most_bytes(int m, int n, int k, bool raw) {
    size_t most = 0, partial = 0;
    int t = 1;
    for (; t <= m && t <= 257 && !f8_wide(t, n, k); ++t) most = std::max(most, f8_call_bytes(f8_plan(t, n, k, raw), t, n, k, raw));
    if (t > m) return most;
    if (!f8_wide(t, n, k)) return std::max(most, f8_call_bytes(f8_plan(m, n, k, raw), m, n, k, raw));            // the panels do not take this k
    for (int end = (t + 63) / 64 * 64; t <= m && t <= 16384; t = end + 1, end += 64) {
        const int last = std::min(end, m);
        partial = std::max(partial, f8_partial_bytes(f8_plan(last, n, k, raw), last, n, k));
    }
    if (m > 16384) partial = std::max(partial, (size_t)device_cus() * 2 * 256 * 256 * 4);
    return std::max(most, f8_carve(nullptr, partial, m, k, raw, nullptr));
}

template <class T>
static int f8_launch_gemm(F8GemmArgs a, const F8Plan &pl, const F8Scratch &w, uint8_t *workspace, hipStream_t s) {
    if (pl.panels) {
        F8PanelArgs g = {};
        g.p.A = a.A;
        g.p.B = reinterpret_cast<const uint16_t *>(a.X);
        g.p.C = a.C;
        g.p.bias = a.bias;
        g.p.scale = a.a_scale;
        g.p.partial = (f32x4 *)w.partial;
        g.p.alpha = a.alpha;
        if (panel8_arguments(g.p, a.M, a.N, a.K / 2, pl.pr, pl.tb, pl.p3) > w.partial_bytes) return fail(MLK_ERR_WORKSPACE, "gemm fp8: workspace too small");
        g.x_scale = a.x_scale;
        g.xs_t = (uint32_t)a.xs_t;
        g.xs_k = (uint32_t)a.xs_k;
        return f8_launch_panel<T>(g, pl.pr, pl.tb, s);
    }
    a.partial = (f32x4 *)w.partial;
    a.counters = (int *)workspace;
    return f8_launch_stream<T>(a, pl, s);
}

}  // namespace mlk

using namespace mlk;

extern "C" {

int mlk_quantize_fp8(const void *x, int x_kind, void *codes, float *scales, int64_t scale_t, int64_t scale_k, int64_t n_tokens, int k, void *stream) {
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16 || x_kind == MLK_F32, "quantize_fp8: activations must be fp16, bf16 or fp32");
    MLK_REQUIRE(n_tokens >= 0 && n_tokens <= (1ll << 27), "quantize_fp8: 0..2^27 rows");
    MLK_REQUIRE(k >= 0 && k % 128 == 0 && k <= kF8MostK, "quantize_fp8: K % 128 must be 0, K at most 33553920");
    if (n_tokens == 0 || k == 0) return MLK_OK;
    MLK_REQUIRE(x && codes && scales, "quantize_fp8: null pointer");
    MLK_REQUIRE(aligned16(x) && aligned16(codes), "quantize_fp8: activations and codes must lie on 16 bytes");
    return launch_quantize_fp8(x, x_kind, (uint8_t *)codes, scales, scale_t, scale_k, n_tokens, k, (hipStream_t)stream);
}

size_t mlk_gemm_fp8_workspace_bytes(int m, int n, int k, int b_kind) {
    if (m <= 0 || n <= 0 || k <= 0 || k % 128 != 0) return 0;
    const bool raw = b_kind != MLK_FP8_E4M3;
    return f8_most_bytes(m, n, k, raw);
}

int mlk_gemm_fp8_needs_workspace(int m, int n, int k, int b_kind) {
    if (m <= 0 || n <= 0 || k <= 0 || k % 128 != 0) return 0;
    const bool raw = b_kind != MLK_FP8_E4M3;
    return f8_call_bytes(f8_plan(m, n, k, raw), m, n, k, raw) > 0;
}

int mlk_gemm_layout_a_fp8(const void *a, const float *a_scale, const void *b, int b_kind, const float *b_scale, int64_t b_scale_t, int64_t b_scale_k, void *c,
                          int c_kind, int m, int n, int k, float alpha, const void *bias, void *workspace, size_t workspace_bytes, void *stream) {
    MLK_REQUIRE(c_kind == MLK_F16 || c_kind == MLK_BF16, "gemm fp8: outputs must be fp16 or bf16");
    MLK_REQUIRE(b_kind == MLK_FP8_E4M3 || b_kind == c_kind, "gemm fp8: activations must be e4m3 codes or of the output's kind");
    MLK_REQUIRE(m >= 0 && m <= (1 << 21), "gemm fp8: 0..2^21 tokens");
    MLK_REQUIRE(n > 0 && k > 0 && n % 16 == 0 && k % 128 == 0 && k <= kF8MostK, "gemm fp8: N % 16 and K % 128 must be 0, K at most 33553920");
    // a launch has fewer than 2^32 threads, and the streaming kernels use up to 16 a row
    MLK_REQUIRE(n <= (1 << 27), "gemm fp8: at most 2^27 rows of weights");
    if (m == 0) return MLK_OK;
    MLK_REQUIRE(a && a_scale && b && c && (b_kind != MLK_FP8_E4M3 || b_scale), "gemm fp8: null pointer");
    MLK_REQUIRE(aligned16(a) && aligned16(b) && aligned16(c), "gemm fp8: weights, activations and outputs must lie on 16 bytes");
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
    const bool raw = b_kind != MLK_FP8_E4M3;
    F8Plan pl = f8_plan(m, n, k, raw);
    if (!raw && pl.panels && (b_scale_t < 0 || b_scale_k < 0 || b_scale_t >= 1 << 21 || b_scale_k >= (1ll << 29) / (k / kF8K))) {
        pl = F8Plan{};                                         // scales that far apart: the panels' offsets of them are 32 bits
        pl.r = 2;
        pl.tt = 4;                                             // 2^21 tokens are 2^15 workgroups side by side
        pl.waves = 8;
        pl.slices = 1;
    }
    F8Scratch w;
    const size_t need = f8_carve((uint8_t *)workspace, f8_partial_bytes(pl, m, n, k), m, k, f8_quantises(pl, raw), &w);
    if (workspace_bytes < need) return fail(MLK_ERR_WORKSPACE, "gemm fp8: workspace too small");
    MLK_REQUIRE(need == 0 || (workspace && aligned16(workspace)), "gemm fp8: workspace off 16 bytes");
    if (raw && pl.feed != kF8Codes) {
        p.raw = b;
    } else if (raw) {
        const int rc = launch_quantize_fp8(b, b_kind, w.codes, w.scales, 1, m, m, k, s);
        if (rc != MLK_OK) return rc;
        p.X = w.codes;
        p.x_scale = w.scales;
        p.xs_t = 1;
        p.xs_k = m;
    }
    return c_kind == MLK_F16 ? f8_launch_gemm<F16>(p, pl, w, (uint8_t *)workspace, s) : f8_launch_gemm<BF16>(p, pl, w, (uint8_t *)workspace, s);
}

}  // extern "C"
