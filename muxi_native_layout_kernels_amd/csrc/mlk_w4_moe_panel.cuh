// The expert layers over 4-bit weights with many tokens per expert: panels (mlk_w4_panel.cuh) of one expert's rows and up to 32 TB of its tokens.
//
// gate/up  a workgroup computes 128 intermediate values of its tokens: each wave a row group of gate and the same one of up.  The exchange of 16 lanes that
//          brought the two into one operand brings gate and up of a value into one lane again.  They go to the intermediate through LDS, 256 bytes of
//          a slot in one piece, and the sums of their groups with them (in a launch of their own 12.8 us of 851 for 2000 pairs of 14336).
// down     256 outputs; `slices` workgroups share the k of one panel, the weighted sums of each go to obuf [pair][slice][H] in fp32.
#pragma once

#include "mlk_w4_moe.cuh"
#include "mlk_w4_panel.cuh"

namespace mlk {

template <class T, int GS, bool ZP, int TB>
__device__ __forceinline__ void w4_gate_up_panel(const W4MoeArgs &p, const MoeTask &task, u32x4 *win) {
    using P = W4Panel<T, GS, ZP, TB>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, i32 = lane & 31, tiles = p.H >> 7, rg = blockIdx.x * 8 + wave;
    const int slot0 = task.block0 * 16, slots = task.nblocks * 16;
    const W4Matrix m = w4_of_expert<GS>(p.w1, task.expert, 2 * p.I, p.H, p.blocks1);
    const typename P::Rows rows = P::rows_of(m, rg, (p.I >> 4) + rg, tiles, p.blocks1, lane);
    typename P::Tokens tk;
    tk.x = p.X;
    tk.c = p.sums1;
#pragma unroll
    for (int i = 0; i < P::NLOAD; ++i) {
        const int pair = p.sorted[slot0 + min(P::load_token(i, tid), slots - 1)];
        tk.row[i] = (uint32_t)(pair < p.n_pairs ? pair / p.K : 0);
    }
    f32x16 acc[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[tb][i] = 0.f;
    P::run(acc, rows, tk, p.H, 0, tiles, p.inv, win);

    constexpr int PITCH = 128 + 8;
    uint16_t *out = reinterpret_cast<uint16_t *>(win);
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // lanes 0..15 of a half: value i, lanes 16..31: value i + 8
            auto gu = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[tb][i]), __float_as_uint(acc[tb][i + 8]), false, false);
            const int v = i + (i32 >> 4) * 8, token = tb * 32 + 8 * (v >> 2) + 4 * h + (v & 3);
            out[token * PITCH + wave * 16 + (i32 & 15)] = (uint16_t)T::from_f32(silu_mul(__uint_as_float(gu[0]), __uint_as_float(gu[1])));
        }
    __syncthreads();
    const int pitch = w4_sum_pitch(p.I, GS);
    for (int c = tid; c < slots * 16; c += 512) {                         // sixteen lanes a slot
        const u32x4 v = *reinterpret_cast<const u32x4 *>(out + (c >> 4) * PITCH + (c & 15) * 8);
        const size_t slot = slot0 + (c >> 4);
        *reinterpret_cast<u32x4 *>(p.hbuf + slot * p.I + blockIdx.x * 128 + (c & 15) * 8) = v;
        const float s = w4_group_sum<T, GS>(v);
        if ((c & 15) % (4 * GS) == 0) p.sums2[slot * pitch + blockIdx.x * (4 / GS) + (c & 15) / (4 * GS)] = w4_sum_parts(s);
        if (blockIdx.x == 0 && (c & 15) == 0) p.sums2[slot * pitch + pitch - 1] = u32x4{0u, 0u, 0u, 0u};
    }
}

template <class T, int GS, bool ZP, int TB>
__device__ __forceinline__ void w4_down_panel(const W4MoeArgs &p, const MoeTask &task, u32x4 *win) {
    using P = W4Panel<T, GS, ZP, TB>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, i32 = lane & 31, tiles = p.I >> 7, groups = p.H >> 4, rg = blockIdx.x * 16 + wave * 2, sl = blockIdx.z;
    const int slot0 = task.block0 * 16, slots = task.nblocks * 16;
    const int t0 = tiles * sl / p.slices, t1 = tiles * (sl + 1) / p.slices;
    const W4Matrix m = w4_of_expert<GS>(p.w2, task.expert, p.H, p.I, p.blocks2);
    const typename P::Rows rows = P::rows_of(m, min(rg, groups - 1), min(rg + 1, groups - 1), tiles, p.blocks2, lane);
    typename P::Tokens tk;
    tk.x = p.hbuf + (size_t)slot0 * p.I;
    tk.c = p.sums2 + (size_t)slot0 * w4_sum_pitch(p.I, GS);
#pragma unroll
    for (int i = 0; i < P::NLOAD; ++i) tk.row[i] = (uint32_t)min(P::load_token(i, tid), slots - 1);
    f32x16 acc[TB];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[tb][i] = 0.f;
    P::run(acc, rows, tk, p.I, t0, t1 - t0, p.inv, win);

    const int row = rg * 16 + i32;
    if (row >= p.H) return;
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int token = tb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
            const int pair = token < slots ? p.sorted[slot0 + token] : p.n_pairs;
            if (pair < p.n_pairs) p.obuf[((size_t)pair * p.slices + sl) * p.H + row] = T::to_f32(p.wts[pair]) * acc[tb][i];
        }
}

// Panels of 128 tokens; an expert's last one is a panel of 64 where its tokens fit in that (8 experts of 4096 x 14336, top-2, at 1000 tokens 890 -> 815 us).
// Panels of 64 for all lose from 50 tokens an expert on, up to 25 %, and gain at most 5 % below.
template <class T, int GS, bool ZP>
__global__ void __launch_bounds__(512, 2) w4_moe_gate_up_panel_kernel(W4MoeArgs p) {
    extern __shared__ u32x4 win[];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks <= 4) w4_gate_up_panel<T, GS, ZP, 2>(p, task, win);
    else w4_gate_up_panel<T, GS, ZP, 4>(p, task, win);
}
template <class T, int GS, bool ZP>
__global__ void __launch_bounds__(512, 2) w4_moe_down_panel_kernel(W4MoeArgs p) {
    extern __shared__ u32x4 win[];
    if ((int)blockIdx.y >= *p.n_tasks) return;
    const MoeTask task = p.tasks[blockIdx.y];
    if (task.nblocks <= 4) w4_down_panel<T, GS, ZP, 2>(p, task, win);
    else w4_down_panel<T, GS, ZP, 4>(p, task, win);
}

template <class T, int GS, bool ZP>
int w4_launch_moe_panel(const W4MoeArgs &a, const W4MoePlan &pl, hipStream_t s) {
    constexpr size_t lds = W4Panel<T, GS, ZP, 4>::lds_bytes;
    int rc = w4_launch_sums<T, GS>(a.X, a.sums1, a.T, a.H, s);
    if (rc != MLK_OK) return rc;
    static bool ready1[64] = {}, ready2[64] = {};
    rc = panel_lds_attribute(&w4_moe_gate_up_panel_kernel<T, GS, ZP>, lds, ready1);
    if (rc == MLK_OK) rc = panel_lds_attribute(&w4_moe_down_panel_kernel<T, GS, ZP>, lds, ready2);
    if (rc != MLK_OK) return rc;
    w4_moe_gate_up_panel_kernel<T, GS, ZP><<<dim3(a.I / 128, pl.max_tasks), 512, lds, s>>>(a);
    MLK_LAUNCH_CHECK();
    w4_moe_down_panel_kernel<T, GS, ZP><<<dim3((a.H + 255) / 256, pl.max_tasks, a.slices), 512, lds, s>>>(a);
    MLK_LAUNCH_CHECK();
    w4_moe_combine_kernel<T><<<dim3(a.T, (a.H + 1023) / 1024), 256, 0, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // namespace mlk
