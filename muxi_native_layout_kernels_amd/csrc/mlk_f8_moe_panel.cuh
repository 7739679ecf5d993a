// The expert layers in e4m3 with many pairs an expert: panels (mlk_f8_panel.cuh) of 256 rows and up to 256 pairs of one expert.
//
// gate/up  128 intermediate values: the four row quarters of a panel hold 32 gate rows and the up rows with the same index, so that gate and up of a value sit in the same lane and
//          register of a wave.  The largest of a token's 128 goes around the waves through LDS, the codes are turned around there, 128 bytes of a slot in a row.
// down     256 outputs; `slices` workgroups share the k of a panel, the weighted sums of each go to obuf [pair][slice][H] in fp32.
//
// Order of the work: (expert, row tile, task of the expert) with tasks fastest, one line cut into eight equal runs, one per XCD: the tasks of an expert share a row tile's weights in one L2.
//
// gate/up multiplies codes as 16-bit numbers (products that feed codes, mlk_f8.cuh), in panels of up to 128 pairs: the registers of larger ones go to the widened weights, and a task of more takes
// its row tile twice.
//
// 8 experts of 4096 x 14336, two picks, 1000 tokens: gate/up 509 us (470 GFLOP, 0.92 PFLOP/s), down 210 (235 GFLOP).  The down loop runs as fast as in the linear layers' panels (1.7 to 1.9 us a window of 256 x 256); what is
// missing to their rate are columns that pad a task to 64, an item's first loads and its epilogue, beside which the CU has nothing else, and the 16 x 11 panels for 256 CUs.  gate/up takes 1.6 times what
// 8-bit products in panels of 256 pairs take (317 us; 64 experts of 2048 x 1408 at 2000 tokens 210 and 127): each half of a task reads its weights from LDS and widens them again, in both token halves of the
// workgroup.  16-bit panels of 256 tokens reach 1.2 PFLOP/s on products of this kind (mlk_moe_wide.cuh).
#pragma once

#include "mlk_f8_moe.cuh"
#include "mlk_f8_panel.cuh"
#include "mlk_moe_wide.cuh"

namespace mlk {

constexpr int kF8OutPitch = 128 + 16;                          // gate/up turn-around buffer: bytes per token

// The arguments and the place in the workgroup, taken afresh for every item of a kernel that loops over them (as wide_args does).
__device__ __forceinline__ const F8MoeArgs &f8_moe_args(int &lane, int &wave) {
    auto at = __builtin_amdgcn_kernarg_segment_ptr();
    int tid = threadIdx.x;
    asm volatile("" : "+s"(at), "+v"(tid));
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    return *(const F8MoeArgs *)at;
}

// Both panels return a ticket of the next item (QUEUE, wave 0).
template <bool QUEUE, int TB>
__device__ __forceinline__ int f8_moe_gate_up_panel(const F8MoeArgs &p, const MoeTask &tk, int rt, int wave, int lane) {
    extern __shared__ u32x4 win[];
    using Loop = F8PanelLoop<2, TB, 2, true>;
    const int wr = wave & 3, wt = wave >> 2, groups_i = p.I >> 4, windows = p.H >> 7, slots = tk.nblocks * 16;
    const uint32_t tile_row = (uint32_t)p.H * 16u;             // bytes of a row group
    const int32_t *sorted = p.sorted + tk.block0 * 16;
    // slots without a routed pair read token 0: their columns of the product are never used
    auto row_of = [&](int slot) {
        const int id = slot < slots ? sorted[slot] : p.n_pairs;
        return id < p.n_pairs ? id / p.K : 0;
    };
    F8PanelSrc src;
    src.p.a = p.w1 + (size_t)tk.expert * 2 * p.I * p.H + (size_t)rt * 8 * tile_row;
    src.w_off = Loop::weight_offset(lane);
    // tiles 2 wave, 2 wave + 1 of the panel: of quarter wave / 2 its gate rows (even waves) or its up rows
    src.p.a_off[0] = (uint32_t)((wave & 1) * groups_i + (wave >> 1) * 2) * tile_row;
    src.p.a_off[1] = src.p.a_off[0] + tile_row;
    src.p.b = reinterpret_cast<const uint16_t *>(p.X);
    p8_token_rows<Loop>(src.p, (uint32_t)p.H, wave, lane, row_of);
    if (wave < 4) {
        src.scales = reinterpret_cast<const uint8_t *>(p.xs);
        src.s_off = (uint32_t)row_of(wave * 64 + lane) * 4u;
        src.s_step = (uint32_t)p.T * 4u;
    } else {
        src.scales = reinterpret_cast<const uint8_t *>(p.s1 + ((size_t)tk.expert * (p.I >> 6) + rt) * windows);
        src.s_off = (uint32_t)((lane & 1) * (p.I >> 7) * windows) * 4u;
        src.s_step = 4;
    }
    typename Loop::Acc acc;
    Loop::run(acc, src, 0, windows, wave, lane);
    const int ticket = QUEUE && wave == 0 ? wide_ticket(p.counters, blockIdx.x & 7, lane) : 0;
    __syncthreads();
    float *most = reinterpret_cast<float *>(win);              // [4][64 TB]
    uint8_t *out = reinterpret_cast<uint8_t *>(win) + 4 * 256 * 4;
    const int t16 = lane & 15;
#pragma unroll
    for (int j = 0; j < 2 * TB; ++j) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc.acc[i][j][e] = silu_mul(acc.acc[i][j][e], acc.acc[2 + i][j][e]);
                m = fmaxf(m, f8_magnitude(acc.acc[i][j][e]));
            }
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        if (lane < 16) most[wr * 256 + wt * TB * 32 + 16 * j + t16] = m;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2 * TB; ++j) {
        const int slot = wt * TB * 32 + 16 * j + t16;
        const int e = f8_exponent(fmaxf(fmaxf(most[slot], most[256 + slot]), fmaxf(most[512 + slot], most[768 + slot])));
        const float inverse = f8_two_to(-e);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 h = acc.acc[i][j];
            *reinterpret_cast<uint32_t *>(out + slot * kF8OutPitch + wr * 32 + i * 16 + 4 * (lane >> 4)) = f8_codes(h[0], h[1], h[2], h[3], inverse);
        }
        if (wr == 0 && lane < 16 && slot < slots) p.hs[(size_t)rt * p.slots + tk.block0 * 16 + slot] = f8_two_to(e);
    }
    __syncthreads();
    // eight lanes store the 128 bytes of a slot; slots without a routed pair are stored too (nobody reads them)
    const int tid = wave * 64 + lane, q = tid & 7;
    uint8_t *dst = p.hbuf + (size_t)tk.block0 * 16 * p.I + rt * 128 + q * 16;
#pragma unroll
    for (int it = 0; it < TB; ++it) {
        const int slot = it * 64 + (tid >> 3);
        if (slot < slots) *reinterpret_cast<u32x4 *>(dst + (size_t)slot * p.I) = *reinterpret_cast<const u32x4 *>(out + slot * kF8OutPitch + q * 16);
    }
    return ticket;
}

template <class T, bool QUEUE, int TB>
__device__ __forceinline__ int f8_moe_down_panel(const F8MoeArgs &p, const MoeTask &tk, int rt, int sk, int wave, int lane) {
    extern __shared__ u32x4 win[];
    using Loop = F8PanelLoop<2, TB>;
    const int wr = wave & 3, wt = wave >> 2, groups = p.H >> 4, rgp = rt * 16, windows = p.I >> 7, slots = tk.nblocks * 16;
    const uint32_t tile_row = (uint32_t)p.I * 16u;
    F8PanelSrc src;
    src.p.a = p.w2 + (size_t)tk.expert * p.H * p.I + (size_t)rgp * tile_row;
    src.w_off = Loop::weight_offset(lane);
    // rows past H: a copy of the last row group, never stored
#pragma unroll
    for (int i = 0; i < 2; ++i) src.p.a_off[i] = (uint32_t)(min(rgp + Loop::tile(wave, i), groups - 1) - rgp) * tile_row;
    src.p.b = reinterpret_cast<const uint16_t *>(p.hbuf + (size_t)tk.block0 * 16 * p.I);
    p8_token_rows<Loop>(src.p, (uint32_t)p.I, wave, lane, [&](int slot) { return slot < slots ? slot : 0; });
    if (wave < 4) {
        const int slot = wave * 64 + lane;
        src.scales = reinterpret_cast<const uint8_t *>(p.hs + tk.block0 * 16);
        src.s_off = (uint32_t)(slot < slots ? slot : 0) * 4u;
        src.s_step = (uint32_t)p.slots * 4u;
    } else {
        src.scales = reinterpret_cast<const uint8_t *>(p.s2 + ((size_t)tk.expert * (p.H >> 7) + rt * 2) * windows);
        src.s_off = (uint32_t)(min(rt * 2 + (lane & 1), (p.H >> 7) - 1) - rt * 2) * windows * 4u;
        src.s_step = 4;
    }
    const int w0 = (int)((long long)sk * windows / p.slices), w1 = (int)((long long)(sk + 1) * windows / p.slices);
    typename Loop::Acc acc;
    Loop::run(acc, src, w0, w1 - w0, wave, lane);
    const int ticket = QUEUE && wave == 0 ? wide_ticket(p.counters + 8 * kWideQueueStep, blockIdx.x & 7, lane) : 0;
    __syncthreads();
    // every wave turns its 32 rows x 32 TB tokens around in its own part of LDS, one row pair after the other, and stores 128 bytes of a pair with eight lanes
    uint8_t *out = reinterpret_cast<uint8_t *>(win) + (size_t)wave * 128 * kWideDownPitch;
    const int t8 = lane >> 3, q = lane & 7, n0 = (rgp + wr * 4) * 16;
    if (n0 >= p.H) return ticket;
    const int32_t *sorted = p.sorted + tk.block0 * 16;
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
        acc.each(lane, [](int) {}, [&](int row, int token, f32x4 v) {
            if (row >> 5 == pr) *reinterpret_cast<f32x4 *>(out + token * kWideDownPitch + (row & 31) * 4) = v;
        });
        wave_lds_sync();
#pragma unroll 4
        for (int it = 0; it < 4 * TB; ++it) {
            const int slot = wt * TB * 32 + it * 8 + t8, id = slot < slots ? sorted[slot] : p.n_pairs;
            if (id < p.n_pairs) {
                f32x4 v = *reinterpret_cast<const f32x4 *>(out + (it * 8 + t8) * kWideDownPitch + q * 16);
                v *= T::to_f32(p.wts[id]);
                *reinterpret_cast<f32x4 *>(p.obuf + ((size_t)id * p.slices + sk) * p.H + n0 + pr * 32 + q * 4) = v;
            }
        }
        wave_lds_sync();
    }
    return ticket;
}

// Task of an item: items of an expert are (rest, task) with tasks fastest, `rest` of `per_task`.
__device__ __forceinline__ MoeTask f8_moe_item(const F8MoeArgs &p, int item, int per_task, int &rest) {
    const MoeTask t0 = p.tasks[item / per_task];               // some task of the item's expert
    const int local = item - (int)t0.first * per_task;
    rest = local / t0.count;
    return p.tasks[t0.first + local % t0.count];
}

template <bool QUEUE>
__device__ __forceinline__ int f8_moe_gate_up_item(const F8MoeArgs &p, int item, int wave, int lane) {
    int rt;
    const MoeTask tk = f8_moe_item(p, item, p.I >> 7, rt);
    MoeTask half = tk;
    half.nblocks = min(tk.nblocks, 8);
    if (tk.nblocks > 8) {
        f8_moe_gate_up_panel<false, 2>(p, half, rt, wave, lane);
        __syncthreads();
        half.block0 += 8;
        half.nblocks = tk.nblocks - 8;
    }
    if (half.nblocks <= 4) return f8_moe_gate_up_panel<QUEUE, 1>(p, half, rt, wave, lane);
    return f8_moe_gate_up_panel<QUEUE, 2>(p, half, rt, wave, lane);
}
template <class T, bool QUEUE>
__device__ __forceinline__ int f8_moe_down_item(const F8MoeArgs &p, int item, int wave, int lane) {
    int rest;
    const int row_tiles = (p.H + 255) >> 8;
    const MoeTask tk = f8_moe_item(p, item, row_tiles * p.slices, rest);
    const int sk = rest / row_tiles, rt = rest - sk * row_tiles;             // slices slowest: workgroups that run together share a window of k
    switch ((tk.nblocks + 3) >> 2) {
        case 1: return f8_moe_down_panel<T, QUEUE, 1>(p, tk, rt, sk, wave, lane);
        case 2: return f8_moe_down_panel<T, QUEUE, 2>(p, tk, rt, sk, wave, lane);
        case 3: return f8_moe_down_panel<T, QUEUE, 3>(p, tk, rt, sk, wave, lane);
        default: return f8_moe_down_panel<T, QUEUE, 4>(p, tk, rt, sk, wave, lane);
    }
}
__device__ __forceinline__ int f8_moe_up_items(const F8MoeArgs &p) { return (p.I >> 7) * p.n_tasks[0]; }
__device__ __forceinline__ int f8_moe_down_items(const F8MoeArgs &p) { return ((p.H + 255) >> 8) * p.slices * p.n_tasks[0]; }

__global__ void __launch_bounds__(512) f8_moe_gate_up_panel_kernel(F8MoeArgs p) {
    const int n = f8_moe_up_items(p), item = wide_item(blockIdx.x, n);
    if (item >= n) return;
    f8_moe_gate_up_item<false>(p, item, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), threadIdx.x & 63);
}
template <class T>
__global__ void __launch_bounds__(512) f8_moe_down_panel_kernel(F8MoeArgs p) {
    const int n = f8_moe_down_items(p), item = wide_item(blockIdx.x, n);
    if (item >= n) return;
    f8_moe_down_item<T, false>(p, item, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), threadIdx.x & 63);
}
__global__ void __launch_bounds__(512) f8_moe_gate_up_queue_kernel(F8MoeArgs) {
    __shared__ int s_item;
    int ticket = blockIdx.x >> 3;
    for (;;) {
        int lane, wave;
        const F8MoeArgs &p = f8_moe_args(lane, wave);
        if (wave == 0) s_item = wide_next(p.counters, f8_moe_up_items(p), blockIdx.x & 7, ticket, lane);
        __syncthreads();                                       // also: LDS is free again
        const int item = __builtin_amdgcn_readfirstlane(s_item);
        if (item < 0) return;
        ticket = f8_moe_gate_up_item<true>(p, item, wave, lane);
    }
}
template <class T>
__global__ void __launch_bounds__(512) f8_moe_down_queue_kernel(F8MoeArgs) {
    __shared__ int s_item;
    int ticket = blockIdx.x >> 3;
    for (;;) {
        int lane, wave;
        const F8MoeArgs &p = f8_moe_args(lane, wave);
        if (wave == 0) s_item = wide_next(p.counters + 8 * kWideQueueStep, f8_moe_down_items(p), blockIdx.x & 7, ticket, lane);
        __syncthreads();                                       // also: LDS is free again
        const int item = __builtin_amdgcn_readfirstlane(s_item);
        if (item < 0) return;
        ticket = f8_moe_down_item<T, true>(p, item, wave, lane);
    }
}

constexpr size_t f8_most(size_t a, size_t b) { return a > b ? a : b; }
constexpr size_t f8_moe_up_ring() { return f8_most(F8PanelLoop<2, 1, 2, true>::lds_bytes, F8PanelLoop<2, 2, 2, true>::lds_bytes); }
constexpr size_t f8_moe_down_ring() {
    return f8_most(f8_most(F8PanelLoop<2, 1>::lds_bytes, F8PanelLoop<2, 2>::lds_bytes), f8_most(F8PanelLoop<2, 3>::lds_bytes, F8PanelLoop<2, 4>::lds_bytes));
}
// Do at most n items of `windows` each go through the queues (wide_queue_pays)?  They cost 1 to 4 us a kernel and win where tasks differ in width: gate/up of 8 experts of 4096 x 14336 at 300
// tokens 263 -> 262 us, at 512 402 -> 331, at 1000 581 -> 505, at 2000 916 -> 906 (down in two slices 342 -> 331, at 512 115 -> 117, at 1000 in one 208 -> 212), at 128 206 -> 203, at 100 214 -> 225; of 64 experts
// of 2048 x 1408 at 500 86 -> 85, at 2000 215 -> 214.
static inline bool f8_queue_pays(const F8MoeArgs &a, int n, int windows) {
    const double mean = (double)a.n_pairs / a.id_limit, spread = 3 * sqrt(mean);
    if (ceil(fmax(mean - spread, 1) / 64) == ceil((mean + spread) / 64)) return false;
    return n > device_cus() && (double)n / device_cus() * windows >= 80;
}
template <class T>
int f8_launch_moe_panels(const F8MoeArgs &a, int max_tasks, hipStream_t s) {
    constexpr size_t lds_up = f8_most(f8_moe_up_ring(), 4096 + 256 * kF8OutPitch), lds_down = f8_most(f8_moe_down_ring(), kWideDownOut);
    static bool ready_up[2][64] = {}, ready_down[2][64] = {};
    const int items_up = (a.I >> 7) * max_tasks, items_down = ((a.H + 255) >> 8) * a.slices * max_tasks;
    const bool queue_up = f8_queue_pays(a, items_up, a.H >> 7), queue_down = f8_queue_pays(a, items_down, (a.I >> 7) / a.slices);
    const auto up = queue_up ? &f8_moe_gate_up_queue_kernel : &f8_moe_gate_up_panel_kernel;
    const auto down = queue_down ? &f8_moe_down_queue_kernel<T> : &f8_moe_down_panel_kernel<T>;
    int rc = panel_lds_attribute(up, lds_up, ready_up[queue_up]);
    if (rc == MLK_OK) rc = panel_lds_attribute(down, lds_down, ready_down[queue_down]);
    if (rc != MLK_OK) return rc;
    up<<<queue_up ? device_cus() : (items_up + 7) / 8 * 8, 512, lds_up, s>>>(a);
    MLK_LAUNCH_CHECK();
    down<<<queue_down ? device_cus() : (items_down + 7) / 8 * 8, 512, lds_down, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // namespace mlk
