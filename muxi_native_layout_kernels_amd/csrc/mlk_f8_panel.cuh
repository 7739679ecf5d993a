// Panels of the e4m3 products: 128 PR weight rows x 64 TB tokens a workgroup (PR = 1, 2; TB = 1..4), eight waves of 32 PR rows x 32 TB tokens.
//
// A window of 128 k is, byte for byte, two k32 slabs of the 16-bit panels (mlk_panel8.cuh): a weight tile of 16 rows is two runs of 1 KiB, a token's piece one line of 128
// bytes.  So tokens come in the same chunks of eight with the same swizzle (P8TokenPairs), and what comes out goes through the same stores and the same fold.
//
// What bounds it: the matrix cores and the reads from LDS about alike.  A window of 256 x 256 keeps a SIMD's matrix core busy for 2048 cycles and LDS for 2000 (192 KB read, 64 written), and takes 3000 with its share
// of first loads and stores (8192 x 8192 at 4000 tokens: a CU is busy for 383 thousand cycles in two rounds of 64 windows, at 1.7 GHz, the clock that power holds): 222 to 256 us by card (2.1 to 2.4 PFLOP/s), the matrix
// cores busy 67 % of the cycles.  A panel of 128 x 64 takes 700 cycles of LDS for 256 of products:
// 13824 x 5120 at 100 tokens 22 us, the matrix cores busy 24 %.
#pragma once

#include "mlk_f8.cuh"
#include "mlk_panel8_gemm.cuh"

namespace mlk {

// Where a wave's loads come from, beside P8Src: the scales.  Waves 0..3 fetch those of the tokens (64 a wave), waves 4..7 those of the weights.
struct F8PanelSrc {
    P8Src p;
    uint32_t w_off;             // this lane's byte of a slab of a weight tile
    const uint8_t *scales;      // base of this wave's scales
    uint32_t s_off;             // this lane's byte offset at window 0
    uint32_t s_step;            // bytes from one window to the next
};

// NS = 2: the first half of a wave's row tiles and the second have scales of their own, of which waves 4..7 fetch one each in lanes 0 and 1.
// EXACT: products of 16 bits of the same codes (products that feed codes, mlk_f8.cuh).  A wave widens a window's weights once, each block of tokens ahead of its products.
template <int PR, int TB, int NS = 1, bool EXACT = false>
struct F8PanelLoop : P8TokenPairs<TB, true> {
    using Tok = P8TokenPairs<TB, true>;          // its NB: chunks of tokens a wave fetches
    using Acc = P8Acc16<PR, TB>;
    static constexpr int RT = 2 * PR, TT = 2 * TB;                          // row tiles and token blocks of a wave
    static constexpr int A_WIN = 1024 * PR, B_WIN = Tok::B_PAIR, S_WIN = 128;       // granules of 16 bytes: weights, tokens, scales (256 of tokens, 256 of weights)
    static constexpr int WIN = A_WIN + B_WIN + S_WIN;
    // Three windows where they fit: 28672 x 8192 at 300 tokens in panels of 256 x 128 158 us with two, 117; 13824 x 5120 at 100 in 128 x 64 34.0, 23.5.  Four and five bring 3 % at most there, and
    // two workgroups of 128 x 64 no longer share a CU (20480 x 5120 at 700 tokens 123 us, 136).
    static constexpr int RING = 3 * WIN * 16 <= (int)kP8MostLds ? 3 : 2;
    static constexpr size_t lds_bytes = (size_t)RING * WIN * 16;
    static constexpr int LOADS = 2 * PR + TB + 1;                           // of a wave and window
    // They go out behind the barrier that frees their buffer: FIRST in the last step of a window, EACH in the steps that follow.  All at once in the last step they hold up every wave of the
    // workgroup in the same place: 8192 x 8192 at 4096 tokens 278 us, two a step 254, three 258, four 259.
    static constexpr int FIRST = 2, EACH = TT == 2 ? LOADS : 2;
    static_assert(FIRST + (TT - 1) * EACH >= LOADS, "all loads of a window go out in one");
    static_assert(lds_bytes <= kP8MostLds, "the ring has to fit");

    __device__ static __forceinline__ int tile(int wave, int i) { return PR * wave + i; }
    // Octets of 8 k of a slab lie in LDS in the order 0 2 1 3 4 6 5 7: the 32 lanes that a read serves together take two octets of equal parity, and these then are 256 bytes in a row,
    // every bank once.
    __device__ static __forceinline__ uint32_t weight_offset(int lane) {
        const int at = lane >> 3, octet = (at & 4) | ((at & 1) << 1) | ((at >> 1) & 1);
        return (octet * 8 + (lane & 7)) * 16;
    }

    // Load l < LOADS of a wave and window: its weight tiles by slabs, its chunks of tokens, its scales.
    __device__ static __forceinline__ void issue(const F8PanelSrc &src, int wave, int window, int buf, int l) {
        extern __shared__ u32x4 win[];
        u32x4 *at = win + buf * WIN;
        if (l < 2 * PR) {
            __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)src.p.a, 0, 0xffffffffu, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at + tile(wave, l >> 1) * 128 + (l & 1) * 64, 16, src.w_off, src.p.a_off[l >> 1] + window * 2048 + (l & 1) * 1024, 0, 0);
        } else if (l < 2 * PR + TB) {
            Tok::issue1(src.p, wave, at + A_WIN, window, l - 2 * PR);
        } else {
            __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)src.scales, 0, 0xffffffffu, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, at + A_WIN + B_WIN + wave * 16, 4, src.s_off, window * src.s_step, 0, 0);
        }
    }

    // Windows w0 .. w0 + n - 1.  On return nothing is in flight and LDS is free once the workgroup has met at a barrier.
    //
    // A step multiplies the wave's row tiles with one block of 16 tokens.  While it does, the block of the next step is read, and the sums of the step before, whose products have
    // ended by then, are scaled and added.  The barrier of a window stands ahead of its last step, when all its operands are in registers: behind it the first operands of the next window are
    // read into those that the last step leaves, and the loads of window w + RING go out into the buffer.
    __device__ static __forceinline__ void run(Acc &out, const F8PanelSrc &src, int w0, int n, int wave, int lane) {
        extern __shared__ u32x4 win[];
        const int wr = wave & 3, wt = wave >> 2;
        const int last = w0 + n - 1;
        auto fetch = [&](int w, int buf, int l) { issue(src, wave, min(w0 + w, last), buf, l); };        // windows past the end: copies of the last one
        const int q = lane >> 4, a_idx = wr * RT * 256 + ((q & 1) + (q & 2) * 2) * 16 + (lane & 15);       // in units of 8 bytes: octets 2 q, and 2 q + 1 at + 32
        const int b0 = A_WIN + Tok::operand16(src.p, 0, lane) + wt * TT * 128, b1 = A_WIN + Tok::operand16(src.p, 1, lane) + wt * TT * 128;
        const int s_idx = (A_WIN + B_WIN) * 4 + wt * TT * 16 + (lane & 15), ws_idx = (A_WIN + B_WIN + 64) * 4 + (NS == 2 ? 0 : (wr * PR) / 4);
        F8Operand a[RT], b[2];
        F8WideOperand wide[EXACT ? RT : 1];
        f32x4 d[2][RT];
        float s[2], sw[NS], scale[NS];
        auto read_a = [&](int buf, int i) {
            const u32x2 *at = reinterpret_cast<const u32x2 *>(win + buf * WIN) + a_idx + i * 256;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x2 x = at[h * 128], y = at[h * 128 + 32];
                a[i].v[h] = u32x4{x[0], x[1], y[0], y[1]};
            }
        };
        auto read_b = [&](int buf, int j) {                    // even blocks into b[0], odd ones into b[1]; there is an even number
            b[j & 1].v[0] = win[buf * WIN + b0 + j * 128];
            b[j & 1].v[1] = win[buf * WIN + b1 + j * 128];
            s[j & 1] = reinterpret_cast<const float *>(win + buf * WIN)[s_idx + j * 16];
        };
        auto read_sw = [&](int buf) {
#pragma unroll
            for (int h = 0; h < NS; ++h) sw[h] = reinterpret_cast<const float *>(win + buf * WIN)[ws_idx + h];
        };
        out.zero();
#pragma unroll
        for (int h = 0; h < NS; ++h) scale[h] = 0.f;
#pragma unroll
        for (int i = 0; i < RT; ++i) d[1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < RING; ++w)
#pragma unroll
            for (int l = 0; l < LOADS; ++l)
                if (w < RING - 1 || l < FIRST) fetch(w, w, l);
        wait_vmcnt_le<(RING - 2) * LOADS + FIRST>();             // window 0
        bare_barrier();
        read_sw(0);
#pragma unroll
        for (int i = 0; i < RT; ++i) read_a(0, i);
        read_b(0, 0);
        int cur = 0;
#pragma clang loop unroll(disable)
        for (int w = 0; w < n; ++w) {
            const int nxt = cur == RING - 1 ? 0 : cur + 1, prv = cur == 0 ? RING - 1 : cur - 1;
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                if (j == TT - 1) {
                    __builtin_amdgcn_sched_barrier(0);
                    wait_vmcnt_le<(RING - 2) * LOADS>();         // this wave's loads of window w + 1 have landed
                    wait_lds();                                // and it has all of window w, which is loaded over behind this barrier
                    bare_barrier();
#pragma unroll
                    for (int l = 0; l < FIRST; ++l) fetch(w + RING, cur, l);
                } else {
                    read_b(cur, j + 1);
#pragma unroll
                    for (int l = FIRST + j * EACH; l < FIRST + (j + 1) * EACH && l < LOADS; ++l) fetch(w + RING - 1, prv, l);
                }
                float last_scale[NS];
#pragma unroll
                for (int h = 0; h < NS; ++h) {
                    last_scale[h] = scale[h];
                    scale[h] = s[j & 1] * sw[h];
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if constexpr (EXACT) {
                        if (j == 0) f8_widen(a[i], wide[i]);
                        d[j & 1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                    } else {
                        d[j & 1][i] = f8_mfma(a[i], b[j & 1], f32x4{0.f, 0.f, 0.f, 0.f});
                    }
                }
                if constexpr (EXACT) {
                    F8WideOperand x;
                    f8_widen(b[j & 1], x);
#pragma unroll
                    for (int o = 0; o < 4; ++o)
#pragma unroll
                        for (int i = 0; i < RT; ++i) d[j & 1][i] = BF16::mfma(wide[i].v[o], x.v[o], d[j & 1][i]);
                }
                if (j == TT - 1) {
                    read_sw(nxt);
#pragma unroll
                    for (int i = 0; i < RT; ++i) read_a(nxt, i);
                    read_b(nxt, 0);
                }
                const int before = j == 0 ? TT - 1 : j - 1;
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) out.acc[i][before][v] = fmaf(last_scale[i * NS / RT], d[1 - (j & 1)][i][v], out.acc[i][before][v]);
#pragma unroll
                for (int i = 0; i < (EXACT ? 0 : RT); ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
                    if (j == TT - 1) __builtin_amdgcn_sched_group_barrier(0x100, 5, 0);
                    else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                if (j == TT - 1) __builtin_amdgcn_sched_barrier(0);
            }
            cur = nxt;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) out.acc[i][TT - 1][v] = fmaf(scale[i * NS / RT], d[1][i][v], out.acc[i][TT - 1][v]);
        __builtin_amdgcn_s_waitcnt(0);
        mfma_settle();
    }
};

struct F8PanelArgs {
    Panel8Args p;               // K, windows and partial sums in 16-bit units: p.K = K / 2
    const float *x_scale;       // token t's window kb at t xs_t + kb xs_k
    uint32_t xs_t, xs_k;
};

// One panel, windows w0 .. w0 + n - 1; `slot`: where its sums go if it is not computed whole (gemm_panel8).
template <class T, int PR, int TB, int MAXTB>
__device__ __forceinline__ void f8_panel(const F8PanelArgs &g, int rt, int tt, int w0, int n, f32x4 *slot) {
    extern __shared__ u32x4 win[];
    using Loop = F8PanelLoop<PR, TB>;
    const Panel8Args &p = g.p;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                              // taken afresh for every run, as in gemm_panel8
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave & 3, wt = wave >> 2;
    const int groups = p.N >> 4, windows = p.K >> 6, rgp = rt * 8 * PR, rg0 = rgp + wr * 2 * PR, tok0 = tt * 64 * MAXTB;
    const uint32_t row = (uint32_t)windows * kF8K;
    // rows past N: a copy of the last row group, never stored; tokens past M: the last token
    F8PanelSrc src;
    src.p.a = p.A + (size_t)rgp * row * 16;
    src.w_off = Loop::weight_offset(lane);
#pragma unroll
    for (int i = 0; i < PR; ++i) src.p.a_off[i] = (uint32_t)(min(rgp + Loop::tile(wave, i), groups - 1) - rgp) * row * 16u;
    src.p.b = p.B + (size_t)tok0 * (row / 2);
    p8_token_rows<Loop>(src.p, row, wave, lane, [&](int t) { return min(tok0 + t, p.M - 1) - tok0; });
    if (wave < 4) {
        src.scales = reinterpret_cast<const uint8_t *>(g.x_scale + (size_t)tok0 * g.xs_t);
        src.s_off = (uint32_t)(min(tok0 + wave * 64 + lane, p.M - 1) - tok0) * g.xs_t * 4u;
        src.s_step = g.xs_k * 4u;
    } else {
        src.scales = reinterpret_cast<const uint8_t *>(p.scale + (size_t)(rgp >> 3) * windows);
        src.s_off = (uint32_t)(min((rgp >> 3) + min(lane, PR - 1), (groups - 1) >> 3) - (rgp >> 3)) * windows * 4u;
        src.s_step = 4;
    }
    typename Loop::Acc acc;
    Loop::run(acc, src, w0, n, wave, lane);
    if (slot == nullptr) {
        __syncthreads();
        p8_store_panel<T, PR, TB>(p, acc, rg0, tok0 + wt * 32 * TB, wave, lane, win);
        return;
    }
    const int cols = min(p.cols, 64 * TB);
    acc.each(lane, [](int) {}, [&](int r, int token, f32x4 v) {
        const int block = (wt * TB + (token >> 5)) * 32, width = min(32, cols - block);
        if ((token & 31) < width) slot[p8_slot_quad(cols, wr * PR + (r >> 5), block, width, (r & 31) >> 2, token & 31)] = v;
    });
}

// The panels of a grid as gemm_panel8_kernel takes them.
template <class T, int PR, int MAXTB>
__global__ void __launch_bounds__(512) f8_panel_kernel(F8PanelArgs g) {
    const Panel8Args &p = g.p;
    int line = blockIdx.x & 7, u = blockIdx.x >> 3;
    if (p.band == 0) {
        const int n = p.whole + p.deal, run = (n + 7) >> 3;
        if (u >= run) return;
        u += line * run;
        line = 0;
    }
    const int windows = p.K >> 6;
    int at = u * windows, end = at + windows;
    const int j = u - p.whole;
    if (j >= 0) {
        if (j >= p.deal) return;
        const int total = (p.panels - p.whole) * windows;
        at = p.whole * windows + (int)((long long)j * total / p.deal);
        end = p.whole * windows + (int)((long long)(j + 1) * total / p.deal);
    }
    for (int seg = 0; at < end; seg = 1) {
        const int panel = at / windows, w0 = at - panel * windows, n = min(windows - w0, end - at);
        int rt, tt;
        if (p8_panel(p, line, panel, rt, tt)) {
            f32x4 *slot = n == windows ? nullptr : p.partial + ((size_t)(line * p.deal + j) * p.slots + seg) * (32 * PR * p.cols);
            const int tb = p8_columns(p.M, tt, MAXTB);
            if (MAXTB == 1 || tb == 1) f8_panel<T, PR, 1, MAXTB>(g, rt, tt, w0, n, slot);
            if constexpr (MAXTB >= 2)
                if (tb == 2) f8_panel<T, PR, 2, MAXTB>(g, rt, tt, w0, n, slot);
            if constexpr (MAXTB >= 3)
                if (tb == 3) f8_panel<T, PR, 3, MAXTB>(g, rt, tt, w0, n, slot);
            if constexpr (MAXTB >= 4)
                if (tb == 4) f8_panel<T, PR, 4, MAXTB>(g, rt, tt, w0, n, slot);
        }
        at += n;
        __syncthreads();
    }
}

template <int PR, int TB>
constexpr size_t f8_panel_lds() {
    size_t most = (size_t)8 * 32 * TB * p8_out_pitch(PR);
    if (F8PanelLoop<PR, 1>::lds_bytes > most) most = F8PanelLoop<PR, 1>::lds_bytes;
    if (TB >= 2 && F8PanelLoop<PR, 2>::lds_bytes > most) most = F8PanelLoop<PR, 2>::lds_bytes;
    if (TB >= 3 && F8PanelLoop<PR, 3>::lds_bytes > most) most = F8PanelLoop<PR, 3>::lds_bytes;
    if (TB >= 4 && F8PanelLoop<PR, 4>::lds_bytes > most) most = F8PanelLoop<PR, 4>::lds_bytes;
    return most;
}
template <class T, int PR, int TB>
static int f8_launch_panel_shape(const F8PanelArgs &g, hipStream_t s) {
    constexpr size_t lds = f8_panel_lds<PR, TB>();
    const Panel8Args &p = g.p;
    static bool ready_on[64] = {};
    const int rc = panel_lds_attribute(&f8_panel_kernel<T, PR, TB>, lds, ready_on);
    if (rc != MLK_OK) return rc;
    const int64_t wgs = p.band > 0 ? ((int64_t)p.whole + p.deal) * 8 : (p.whole + p.deal + 7) / 8 * 8;
    MLK_REQUIRE(wgs < 1 << 23, "gemm fp8: more panels than a launch takes");         // of 2^32 threads
    f8_panel_kernel<T, PR, TB><<<(int)wgs, 512, lds, s>>>(g);
    MLK_LAUNCH_CHECK();
    if (p.deal > 0) {
        gemm_panel8_fold_kernel<T><<<dim3(4 * PR * TB, p.panels - p.whole, p.band > 0 ? 8 : 1), 256, 0, s>>>(p, PR, TB);
        MLK_LAUNCH_CHECK();
    }
    return MLK_OK;
}
// Panels of 128 pr rows x 64 tb tokens.
template <class T>
int f8_launch_panel(const F8PanelArgs &g, int pr, int tb, hipStream_t s) {
    switch (pr * 8 + tb) {
        case 8 + 1: return f8_launch_panel_shape<T, 1, 1>(g, s);
        case 8 + 2: return f8_launch_panel_shape<T, 1, 2>(g, s);
        case 8 + 3: return f8_launch_panel_shape<T, 1, 3>(g, s);
        case 8 + 4: return f8_launch_panel_shape<T, 1, 4>(g, s);
        case 16 + 1: return f8_launch_panel_shape<T, 2, 1>(g, s);
        case 16 + 2: return f8_launch_panel_shape<T, 2, 2>(g, s);
        case 16 + 3: return f8_launch_panel_shape<T, 2, 3>(g, s);
        case 16 + 4: return f8_launch_panel_shape<T, 2, 4>(g, s);
    }
    return fail(MLK_ERR_INVALID, "gemm fp8: no such panel shape");
}

}  // namespace mlk
