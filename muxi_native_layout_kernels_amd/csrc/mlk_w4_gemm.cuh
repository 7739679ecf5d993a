// Streaming kernel of the 4-bit linear layers, for few tokens or little weight: bound by the weights' bytes, with more tokens by what the workgroups read of
// the activations.
//
// A workgroup owns up to R consecutive row groups (of 16 rows); its waves deal the tiles of 128 k among themselves (tile t to wave t mod waves, so
// that together they read each row group front to back) and add their sums through LDS in wave order.  The row groups are dealt out evenly over the
// grid; `slices` workgroups may share a set of row groups, each on its own range of k: the last one to arrive adds their fp32 sums in the
// order of k.  Workgroups take up to 64 tokens (blockIdx.z).
#pragma once

#include "mlk_w4.cuh"

namespace mlk {

struct W4GemmArgs {
    W4Matrix A;
    const uint16_t *X;
    uint16_t *C;
    const uint16_t *bias;
    float alpha;
    int M, N, K;
    int blocks;            // blocks of scales of a row group (K / max(group, 128)), and w4_inverse() of the tiles of each
    uint32_t inv;
    int slices;
    int rg_each, rg_more;  // row groups of a workgroup; the first rg_more workgroups have one more
    int t_each, t_more;    // tiles of a slice, likewise
    f32x4 *partial;        // [workgroup][slice][cell][two planes of 64 x 8 bytes]
    int *counters;         // [workgroup (x, z)], zero between calls
};

constexpr int kW4TokenLds = 128 * 1024;      // bytes of LDS that one token may take

// Waves a workgroup may have, so that the ring fits the registers.
__host__ __device__ constexpr int w4_stream_waves(int tt, int r, bool xl) { return xl ? 16 : 8; }
__host__ __device__ constexpr int w4_ring(int tt, int r, bool xl) {
    return xl ? (r == 1 ? 8 : 4) : (tt == 1 ? (r <= 2 ? 4 : 2) : (tt * r <= 8 && tt < 4 ? 2 : 1));
}

// Cells that the waves add at a time: eight waves of 16 take 128 KiB of LDS.
__host__ __device__ constexpr int w4_fold_cells(int cells) { return cells > 16 ? cells / 2 : cells; }

template <class T, int GS, bool ZP, int TT, int R, bool XL>
__global__ void __launch_bounds__(w4_stream_waves(TT, R, XL) * 64) w4_stream_kernel(W4GemmArgs p) {
    extern __shared__ u32x4 lds[];
    __shared__ int s_last;
    constexpr int CELLS = R * TT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int o = lane >> 4, r16 = lane & 15;
    const int tiles = p.K >> 7, b = blockIdx.x, sl = blockIdx.y;
    const int rg0 = b * p.rg_each + min(b, p.rg_more), nr = p.rg_each + (b < p.rg_more ? 1 : 0);
    const int t0 = sl * p.t_each + min(sl, p.t_more), t1 = t0 + p.t_each + (sl < p.t_more ? 1 : 0);

    W4Rows<R> rows;
#pragma unroll
    for (int r = 0; r < R; ++r) w4_row<GS, R>(rows, r, p.A, rg0 + min(r, nr - 1), tiles, p.blocks);
    const int m0 = blockIdx.z * (TT * 16);
    const uint16_t *xrow[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) xrow[tt] = p.X + (size_t)min(m0 + tt * 16 + r16, p.M - 1) * p.K;
    f32x4 acc[R][TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) acc[r][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (XL)
        for (int i = t0 * 16 + threadIdx.x; i < t1 * 16; i += blockDim.x) lds[i - t0 * 16] = ld_global_u32x4(p.X + (size_t)i * 8);
    w4_stream<T, GS, ZP, TT, R, w4_ring(TT, R, XL), XL>(acc, rows, xrow, lds - t0 * 16, t0 + wave, t1, waves, p.inv, lane, true);

    auto store = [&](int c, f32x4 v) {
        const int r = c / TT, tt = c - r * TT;
        if (r >= nr) return;
        const int row = (rg0 + r) * 16 + r16;
        const float b = p.bias ? T::to_f32(p.bias[row]) : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int token = m0 + tt * 16 + o * 4 + i;
            if (token < p.M) p.C[(size_t)token * p.N + row] = (uint16_t)T::from_f32(p.alpha * v[i] + b);
        }
    };
    const int set = blockIdx.z * gridDim.x + blockIdx.x;
    auto part = [&](int s, int c) { return p.partial + (((size_t)set * p.slices + s) * CELLS + c) * 64; };
    f32x4 *red = reinterpret_cast<f32x4 *>(lds);
    constexpr int FOLD = w4_fold_cells(CELLS);
#pragma unroll
    for (int c0 = 0; c0 < CELLS; c0 += FOLD) {
        if (XL || c0 > 0) __syncthreads();                // the other waves still read the token, or the cells before
#pragma unroll
        for (int c = c0; c < c0 + FOLD; ++c) red[(wave * FOLD + c - c0) * 64 + lane] = acc[c / TT][c % TT];
        __syncthreads();
        for (int c = c0 + wave; c < c0 + FOLD; c += waves) {
            f32x4 v = red[(c - c0) * 64 + lane];
            for (int w = 1; w < waves; ++w) v += red[(w * FOLD + c - c0) * 64 + lane];
            if (p.slices == 1) store(c, v);
            else st_agent_planar(part(blockIdx.y, c), 64, lane, v);
        }
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

template <class T, int GS, bool ZP, int TT, int R, bool XL>
static int w4_launch_stream_one(W4GemmArgs a, int wgs, int waves, hipStream_t s) {
    const int groups = a.N / 16, t = a.K / kW4TileK, per_slice = (t + a.slices - 1) / a.slices;
    a.rg_each = groups / wgs;
    a.rg_more = groups % wgs;
    a.t_each = t / a.slices;
    a.t_more = t % a.slices;
    size_t lds = (size_t)waves * w4_fold_cells(R * TT) * 1024;
    if (XL && (size_t)per_slice * 256 > lds) lds = (size_t)per_slice * 256;
    if (waves > w4_stream_waves(TT, R, XL) || lds > 150 * 1024) return fail(MLK_ERR_INVALID, "w4 gemm: launch parameters");
    if (lds > 48 * 1024) {
        static bool ready_on[64] = {};                     // the attribute belongs to a device
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess) dev = 0;
        if (!ready_on[dev & 63]) {
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&w4_stream_kernel<T, GS, ZP, TT, R, XL>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 150 * 1024);
            if (e != hipSuccess) return fail(MLK_ERR_LAUNCH, hipGetErrorString(e));
            ready_on[dev & 63] = true;
        }
    }
    w4_stream_kernel<T, GS, ZP, TT, R, XL><<<dim3(wgs, a.slices, XL ? 1 : (a.M + TT * 16 - 1) / (TT * 16)), waves * 64, lds, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

// r = row groups per workgroup, tt = blocks of 16 tokens: what w4_plan() picks of them; wgs * r >= N / 16.  One token is staged in LDS (r = 1, 2; a slice of 64 K at most): 4096 x 4096
// 4.7 us against 5.1.
template <class T, int GS, bool ZP>
int w4_launch_stream(const W4GemmArgs &a, int r, int tt, int wgs, int waves, hipStream_t s) {
    if ((int64_t)r * wgs < a.N / 16 || wgs > a.N / 16) return fail(MLK_ERR_INVALID, "w4 gemm: launch parameters");
#define MLK_W4_R(TT, R) if (tt == TT && r == R) return w4_launch_stream_one<T, GS, ZP, TT, R, false>(a, wgs, waves, s)
    if (a.M == 1 && (a.K / kW4TileK + a.slices - 1) / a.slices * 256 <= kW4TokenLds) {
        if (r == 1) return w4_launch_stream_one<T, GS, ZP, 1, 1, true>(a, wgs, waves, s);
        if (r == 2) return w4_launch_stream_one<T, GS, ZP, 1, 2, true>(a, wgs, waves, s);
    }
    MLK_W4_R(1, 1);
    MLK_W4_R(1, 2);
    MLK_W4_R(1, 4);
    MLK_W4_R(1, 8);
    MLK_W4_R(2, 1);
    MLK_W4_R(2, 2);
    MLK_W4_R(2, 4);
    MLK_W4_R(2, 8);
    MLK_W4_R(3, 2);
    MLK_W4_R(3, 4);
    MLK_W4_R(3, 8);
    MLK_W4_R(4, 4);
#undef MLK_W4_R
    return fail(MLK_ERR_INVALID, "w4 gemm: launch parameters");
}

}  // namespace mlk
