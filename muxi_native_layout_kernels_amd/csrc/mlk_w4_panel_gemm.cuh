// The 4-bit linear layers with many tokens: panels (mlk_w4_panel.cuh), whole or in K slices that a second launch adds.
#pragma once

#include "mlk_w4_gemm.cuh"
#include "mlk_w4_panel.cuh"

namespace mlk {

struct W4PanelArgs {
    W4Matrix A;
    const uint16_t *X;
    uint16_t *C;
    const uint16_t *bias;
    float alpha;
    int M, N, K, blocks;
    uint32_t inv;
    int row_tiles, token_tiles, slices;
    u32x4 *sums;           // [M][w4_sum_pitch()]
    float *partial;        // [slice][M][N]
};

template <class T, int GS, bool ZP, int TB>
__global__ void __launch_bounds__(512, 2) w4_panel_kernel(W4PanelArgs p) {
    using P = W4Panel<T, GS, ZP, TB>;
    extern __shared__ u32x4 win[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, i32 = lane & 31;
    // workgroups go to the XCDs in turn: an XCD gets a contiguous run of panels, the token tiles of a row tile side by side
    const int total = p.row_tiles * p.token_tiles * p.slices, xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
    const int u = (blockIdx.x >> 3) + xcd * each + min(xcd, more);
    const int sl = u % p.slices, v = u / p.slices, tt0 = v % p.token_tiles, rt = v / p.token_tiles;
    const int tiles = p.K >> 7, groups = p.N >> 4;
    const int t0 = (int)((unsigned)tiles * sl / p.slices), t1 = (int)((unsigned)tiles * (sl + 1) / p.slices);
    const int rg0 = rt * 16 + wave * 2, m0 = tt0 * P::TOK;

    const typename P::Rows rows = P::rows_of(p.A, min(rg0, groups - 1), min(rg0 + 1, groups - 1), tiles, p.blocks, lane);
    typename P::Tokens tk;
    tk.x = p.X + (size_t)m0 * p.K;
    tk.c = p.sums + (size_t)m0 * w4_sum_pitch(p.K, GS);
#pragma unroll
    for (int i = 0; i < P::NLOAD; ++i) tk.row[i] = (uint32_t)min(P::load_token(i, tid), p.M - 1 - m0);
    f32x16 acc[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[tb][i] = 0.f;
    P::run(acc, rows, tk, p.K, t0, t1 - t0, p.inv, win);

    const int row = rg0 * 16 + i32;
    if (p.slices > 1) {
        if (row < p.N)
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int token = m0 + tb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
                    if (token < p.M) p.partial[((size_t)sl * p.M + token) * p.N + row] = acc[tb][i];
                }
        return;
    }
    // 32 rows x 32 tokens at a time through the wave's own part of LDS: a token's 32 outputs are stored in one piece of 64 bytes
    constexpr int PITCH = 40;
    uint16_t *mine = reinterpret_cast<uint16_t *>(win) + wave * (32 * PITCH);
    const float b = p.bias && row < p.N ? T::to_f32(p.bias[row]) : 0.f;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[(8 * (i >> 2) + 4 * h + (i & 3)) * PITCH + i32] = (uint16_t)T::from_f32(p.alpha * acc[tb][i] + b);
        wave_lds_sync();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int tk = c * 16 + (lane >> 2), piece = lane & 3, token = m0 + tb * 32 + tk;
            if (token < p.M && rg0 * 16 + piece * 8 < p.N)
                *reinterpret_cast<u32x4 *>(p.C + (size_t)token * p.N + rg0 * 16 + piece * 8) = *reinterpret_cast<const u32x4 *>(mine + tk * PITCH + piece * 8);
        }
        wave_lds_sync();
    }
}

// C = T(alpha * (sum of the slices in the order of k) + bias), four outputs a thread.
template <class T>
__global__ void __launch_bounds__(256) w4_panel_fold_kernel(W4PanelArgs p) {
    const size_t cells = (size_t)p.M * p.N / 4;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (size_t)gridDim.x * 256) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.slices; ++s) v += *reinterpret_cast<const f32x4 *>(p.partial + ((size_t)s * cells + i) * 4);
        const int n = (int)(i * 4 % p.N);
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.bias)
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = T::to_f32(p.bias[n + j]);
        u32x2 q;
        q[0] = T::from_f32x2(p.alpha * v[0] + b[0], p.alpha * v[1] + b[1]);
        q[1] = T::from_f32x2(p.alpha * v[2] + b[2], p.alpha * v[3] + b[3]);
        *reinterpret_cast<u32x2 *>(p.C + i * 4) = q;
    }
}

template <class T, int GS, bool ZP, int TB>
static int w4_launch_panel_one(W4PanelArgs a, hipStream_t s) {
    using P = W4Panel<T, GS, ZP, TB>;
    a.row_tiles = (a.N + P::ROWS - 1) / P::ROWS;
    a.token_tiles = (a.M + P::TOK - 1) / P::TOK;
    static bool ready_on[64] = {};
    const int rc = panel_lds_attribute(&w4_panel_kernel<T, GS, ZP, TB>, P::lds_bytes, ready_on);
    if (rc != MLK_OK) return rc;
    const int rc2 = w4_launch_sums<T, GS>(a.X, a.sums, a.M, a.K, s);
    if (rc2 != MLK_OK) return rc2;
    w4_panel_kernel<T, GS, ZP, TB><<<a.row_tiles * a.token_tiles * a.slices, 512, P::lds_bytes, s>>>(a);
    MLK_LAUNCH_CHECK();
    if (a.slices > 1) {
        const size_t wgs = ((size_t)a.M * a.N / 4 + 255) / 256;
        w4_panel_fold_kernel<T><<<(int)(wgs < 2048 ? wgs : 2048), 256, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
    }
    return MLK_OK;
}

// tb: token blocks of 32 of a panel, 2 or 4
template <class T, int GS, bool ZP>
int w4_launch_panel(const W4PanelArgs &a, int tb, hipStream_t s) {
    return tb == 2 ? w4_launch_panel_one<T, GS, ZP, 2>(a, s) : w4_launch_panel_one<T, GS, ZP, 4>(a, s);
}

}  // namespace mlk
