// Panels of the 4-bit products for many tokens: 256 weight rows x 32 TB tokens a workgroup, eight waves of two row
// groups (32 rows) each, all on the same tokens.
//
// What a panel costs, in cycles of a CU and a window of 128 k (TB = 4; two waves on each SIMD):
//   products        2048   32 x 32 x 16, 32 cycles each: half as many instructions to issue as 16 x 16 x 32
//   vector instr.   1700   one in 5.6 cycles beside matrix instructions, measured: 64 to widen a wave's weights of a window, which all its token blocks
//                          share, and 64 to scale the sums of its four blocks
//   LDS reads       1100   4.3 cycles each, measured: an operand of 32 tokens for every product
// They overlap (widening, scaling and reads are spread between the products).  Measured at 27648 x 5120, 2048 tokens, groups of 128: 512 to 537 us by card, 1.08 to 1.13 PFLOP/s; the matrix
// cores are busy for 63 % of the cycles, and the card runs at 1.85 GHz under this load (2.4 without it).  Nothing may be added to the loop.  So sum x, which the offset of
// 16 + q calls for (mlk_w4.cuh), does not come into this loop: as initial values of the products' sums it took another half of the LDS reads
// (27648 x 5120 at 2048 tokens: 549 us).  It is made by a launch ahead (w4_sums_kernel) and multiplied behind the weights, like 8 more k for every 32, 64 or
// 128:  acc += sum over the groups of o * sum x,  o = -s (16 + z) or s (31 - z), both factors as parts of 8 bits in bf16 whatever the activations' type:
//   sum x = c1 + c2 + c3 (24 bits),   o = b1 + b2 (16 bits at most: exact),   octets {c1 c2 c3 c1 c2 0 0 0} . {b1 b1 b1 b2 b2 0 0 0},
// what is left out is below 2^-24 of the product.
// Until then the running sums hold the offset, and where a token's activations do not average to zero they would grow with k, the result with its root only.  So
// every second window (counted from the panel's first) multiplies its codes' complement, W + s (31 - z) in place of W - s (16 + z) with the scale's sign
// turned: 31 - q = 16 + ~q, and the offsets of two neighbours cancel but for what their scales and activations differ.  Activations of mean 1, fp16, K = 14336, groups of
// 64: the results were off by 1.27 roundings with all windows alike, and by 1.80 with K = 14208 whole in groups of 32; now by less than 1.05 at any mean.  It costs 1 % (2048 tokens
// above: 532 -> 537 us; spread between the products, as the widening is, the 8 instructions of two windows cost 539).
//
// Tokens come into LDS in windows of 128 k by loads that write LDS directly, four windows deep; weights go straight to registers: no wave needs
// another one's.  Order of a window t: tokens t + 3 and weights t + 2 are requested, the products of t run, the weights of t + 1 are widened, the first operands
// of t + 1 read; then the tokens of t + 2 are waited for and the workgroup meets.  Nothing stands between the barrier and the first product.
//
// Operands of v_mfma_f32_32x32x16 (lane = 32 h + i): tokens lane holds token i, eight k; weights lane holds row i, the same k; result lane holds
// row i, tokens 8 a + 4 h + 0..3 in registers 4 a + 0..3.  A dword j of two row groups' tiles (lane 16 o + r: row r, octet 4 j + o) becomes two such
// operands by one exchange of 16 lanes: rows 0..15 the first row group, 16..31 the second, octets 4 j + 2 h and 4 j + 2 h + 1.
// Four tokens of a window are 1 KiB (what a wave's load writes) and 64 bytes of padding; octet c of token i lies at place c ^ (i % 4) of its 256 bytes.
// The sixteen lanes whose 16-byte reads are served together (0..3, 12..15, 20..27 of an operand, and 4..11, 16..19, 28..31) then meet sixteen
// different bank groups, and all but one bit of an operand's octet is an immediate offset: two address registers for all of them.
#pragma once

#include <type_traits>

#include "mlk_panel_lds.cuh"
#include "mlk_w4.cuh"

namespace mlk {

// Octets of sum x of a token: one for each group of a window (128 k), and one of zeros behind the last.
__host__ __device__ constexpr int w4_sum_pitch(int k, int gs) { return k / 128 * (4 / gs) + 1; }

// Sum of eight activations in a lane and those of 32 GS: of 4 GS lanes; and its parts.
template <class T, int GS>
__device__ __forceinline__ float w4_group_sum(const u32x4 &v) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) s += T::to_f32(v[j] & 0xffffu) + T::to_f32(v[j] >> 16);
#pragma unroll
    for (int m = 1; m < 4 * GS; m <<= 1) s += __shfl_xor(s, m);
    return s;
}
__device__ __forceinline__ u32x4 w4_sum_parts(float s) {
    const uint32_t c1 = f32_to_bf16_bits(s);
    const float r1 = s - bf16_bits_to_f32(c1);
    const uint32_t c2 = f32_to_bf16_bits(r1), c3 = f32_to_bf16_bits(r1 - bf16_bits_to_f32(c2));
    return u32x4{c1 | c2 << 16, c3 | c1 << 16, c2, 0u};
}

// c[token][window * G + g] = parts of the sum of the group's 32 GS activations.
template <class T, int GS>
__global__ void __launch_bounds__(256) w4_sums_kernel(const uint16_t *__restrict__ x, u32x4 *__restrict__ c, int tokens, int k) {
    constexpr int LANES = 4 * GS;
    const int per_token = k / 8, pitch = w4_sum_pitch(k, GS);
    const int64_t total = (int64_t)tokens * per_token;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {        // total is a multiple of 16
        const int64_t token = i / per_token;
        const int at = (int)(i - token * per_token);
        const float s = w4_group_sum<T, GS>(ld_global_u32x4(x + i * 8));
        if (at % LANES == 0) c[token * pitch + at / LANES] = w4_sum_parts(s);
        if (at == 0) c[token * pitch + pitch - 1] = u32x4{0u, 0u, 0u, 0u};
    }
}

template <class T, int GS>
static int w4_launch_sums(const uint16_t *x, u32x4 *c, int tokens, int k, hipStream_t s) {
    const int64_t wgs = ((int64_t)tokens * (k / 8) + 255) / 256;
    w4_sums_kernel<T, GS><<<(int)(wgs < 2048 ? wgs : 2048), 256, 0, s>>>(x, c, tokens, k);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

template <class T, int GS, bool ZP, int TB>
struct W4Panel {
    static_assert(TB % 2 == 0, "the products of a block alternate between two sets of registers");
    static constexpr int ROWS = 256, TOK = 32 * TB;
    static constexpr int NLOAD = TB;                       // 16-byte loads of a thread per window
    static constexpr int WIN = TOK * 17;                   // granules of a window
    static constexpr int G = 4 / GS;                       // groups of a window
    static constexpr int NB = TB * G;                      // blocks of a window: 32 tokens, one group
    static constexpr int NM = 2 * GS;                      // products of a block
    static constexpr int RING = 4;                         // token operands in flight from LDS
    static constexpr size_t lds_bytes = (size_t)4 * WIN * 16;

    // Token of the panel that load i of this thread fetches, and the octet of the window.
    __device__ static __forceinline__ int load_token(int i, int tid) { return i * 32 + (tid >> 4); }
    __device__ static __forceinline__ int load_octet(int tid) { return (tid & 15) ^ ((tid >> 4) & 3); }
    // Place of a token's octet in a window.
    __device__ static __forceinline__ int place(int token, int octet) { return token * 16 + (token >> 2) * 4 + (octet ^ (token & 3)); }

    // The two row groups of the wave: codes wave-uniform, scales and zero points of this lane's row.
    struct Rows {
        const uint8_t *codes[2];
        const uint16_t *scales;
        const uint8_t *zeros;
    };
    __device__ static __forceinline__ Rows rows_of(const W4Matrix &m, int rg0, int rg1, int tiles, int blocks, int lane) {
        Rows q;
        q.codes[0] = m.codes + (size_t)rg0 * tiles * kW4TileBytes;
        q.codes[1] = m.codes + (size_t)rg1 * tiles * kW4TileBytes;
        const size_t at = ((size_t)(lane & 16 ? rg1 : rg0) * blocks * 16 + (lane & 15)) * G;
        q.scales = m.scales + at;
        q.zeros = ZP ? m.zeros + at : nullptr;
        return q;
    }
    // The tokens: row of load i is x + row[i] * K, its sums c + row[i] * pitch; both below 4 GiB from their base.
    struct Tokens {
        const uint16_t *x;
        const u32x4 *c;
        uint32_t row[NLOAD];
    };

    // acc[tb] += W . x over the windows t0 .. t0 + n - 1 (n >= 1) for the 32 tokens of block tb.  On return nothing is in flight and LDS is free.
    __device__ static __forceinline__ void run(f32x16 (&acc)[TB], const Rows &rows, const Tokens &tk, int K, int t0, int n, uint32_t inv, u32x4 *win) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int h = lane >> 5, i32 = lane & 31;
        const int last = K / 128 * G, pitch = last + 1, ncorr = (n * G + 15) >> 4;
        const W4Const<T> con;

        // Windows n .. n + ncorr - 1 are the sums, sixteen groups each.  No branch: behind one that may or may not have requested something the
        // compiler waits for everything in flight.
        struct From {
            const void *base;
            uint32_t pitch, lane, at;                      // bytes: of a token's row, of this lane's octet, of the window
        };
        auto from = [&](int t) {
            const bool is_x = t < n;
            const int e = min(t0 * G + (min(t, n + ncorr - 1) - n) * 16 + load_octet(tid), last);              // `last`: the zeros
            From f;
            f.base = is_x ? (const void *)tk.x : (const void *)tk.c;
            f.pitch = is_x ? (uint32_t)K * 2u : (uint32_t)pitch * 16u;
            f.lane = (uint32_t)(is_x ? load_octet(tid) : e) * 16u;
            f.at = is_x ? (uint32_t)(t0 + t) * 256u : 0u;
            return f;
        };
        auto issue = [&](const From &f, int buf, int i) {
            __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)f.base, 0, 0xffffffffu, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, win + buf * WIN + (i * 8 + wave) * 68, 16, __umul24(tk.row[i], f.pitch) + f.lane, f.at, 0, 0);
        };
        const int xat[2] = {place(i32, 2 * h), place(i32, 2 * h + 1)};      // operands (0, s) of block 0: octet 4 j + 2 h + s
        auto operand = [&](int buf, int tb, int q) { return win[buf * WIN + xat[q & 1] + tb * 544 + (q >> 1) * 4]; };

        u32x4 raw[2], nxt[2];
        W4Scale<GS> sc, sn, sp = {};                       // of this window, of the next one, of the one before
        auto load_w = [&](int t, int r) { return ld_global_u32x4(rows.codes[r] + (size_t)(t0 + t) * kW4TileBytes + lane * 16); };
        auto load_s = [&](int t) { return w4_load_scale<GS, false>(rows.scales, nullptr, (size_t)(w4_block(t0 + t, inv) * 16)); };
        auto exchange = [&]() {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                auto p = __builtin_amdgcn_permlane16_swap(raw[0][j], raw[1][j], false, false);
                raw[0][j] = p[0];
                raw[1][j] = p[1];
            }
        };
        // operand register q of a window's 32: step q / 4, register q % 4
        u32x4 w[2][8];
        auto widen = [&](u32x4 (&dst)[8], int q) { dst[q >> 2][q & 3] = w4_widen1<T, false>(raw[(q >> 2) & 1][q >> 3], q & 3, con, con.bits); };
        const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        f32x16 d[2];
        u32x4 x[RING];

#pragma unroll
        for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int i = 0; i < NLOAD; ++i) issue(from(t), t, i);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            raw[r] = load_w(0, r);
            nxt[r] = load_w(min(1, n - 1), r);
        }
        sc = load_s(0);
        __builtin_amdgcn_s_waitcnt(0);                     // nothing is in flight in front of the loop: the waits in it are counted from its own requests
        __syncthreads();
        exchange();
#pragma unroll
        for (int q = 0; q < 32; ++q) widen(w[0], q);
        raw[0] = nxt[0];
        raw[1] = nxt[1];
        d[1] = zero;
#pragma unroll
        for (int q = 0; q < RING; ++q) x[q] = operand(0, 0, q);

        // EVEN: t is even, so t + 1 takes the codes' complement
        auto window = [&](int t, int buf, u32x4 (&wn)[8], u32x4 (&wt)[8], auto even) {
            constexpr bool EVEN = decltype(even)::value;
            const int b1 = (buf + 1) & 3;
            const From f = from(t + 3);
            exchange();
            if constexpr (EVEN) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) raw[r][j] = ~raw[r][j];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int g = b % G, now = b & 1, then = now ^ 1;
                const int pb = (b + NB - 1) % NB, ptb = pb / G;        // the block before, whose products are added now
                const float scale = (b ? EVEN : !EVEN) ? w4_scale<T, GS>(b ? sc : sp, pb % G) : -w4_scale<T, GS>(b ? sc : sp, pb % G);
#pragma unroll
                for (int m = 0; m < NM; ++m) {
                    const int P = b * NM + m, ahead = P + RING;
                    d[now] = T::mfma32(x[P % RING], wn[g * NM + m], m ? d[now] : zero);
                    // the operand of the product RING further on: token block, step (the next window's tokens are there)
                    if (ahead < NB * NM) x[P % RING] = operand(buf, ahead / NM / G, ahead / NM % G * NM + ahead % NM);
                    else x[P % RING] = operand(b1, 0, ahead - NB * NM);
                    // Loads one by one: in one piece in front of the window they held every wave up for 700 cycles of 3500
                    if (P < 2) nxt[P] = load_w(min(t + 2, n - 1), P);
                    if (P == 2) sn = load_s(min(t + 1, n - 1));
#pragma unroll
                    for (int i = 0; i < NLOAD; ++i)
                        if (P == 3 + i * (NB * NM / NLOAD)) issue(f, (buf + 3) & 3, i);
                    // a share of the block before: its last product takes a while, so not behind the first one here
                    constexpr int FIRST = NM > 2 ? NM / 4 : 1;
                    const int i0 = m < FIRST ? 0 : 16 * (m - FIRST) / (NM - FIRST), i1 = m < FIRST ? 0 : 16 * (m + 1 - FIRST) / (NM - FIRST);
#pragma unroll
                    for (int i = i0; i < i1; ++i) acc[ptb][i] = fmaf(scale, d[then][i], acc[ptb][i]);
#pragma unroll
                    for (int k = P * 32 / (NB * NM); k < (P + 1) * 32 / (NB * NM); ++k) {
                        widen(wt, k);
                        asm volatile("" : "+v"(wt[k >> 2][k & 3]));         // here, not in front of the next window's products
                    }
                    if (m == NM - 1) asm volatile("" : "+v"(acc[ptb]));     // the compiler would sink the sums behind the last block
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            sp = sc;
            sc = sn;
            raw[0] = nxt[0];
            raw[1] = nxt[1];
            // The tokens of t + 2 have landed: they were requested before all that this window requests.  The LDS reads in flight are of t + 1: what
            // was read of t has been multiplied.
            asm volatile("" ::: "memory");
            wait_vmcnt_le<NLOAD + 3>();
            bare_barrier();
            return b1;
        };
        int buf = 0, t = 0;
        for (; t + 2 <= n; t += 2) {
            buf = window(t, buf, w[0], w[1], std::true_type());
            buf = window(t + 1, buf, w[1], w[0], std::false_type());
        }
        if (t < n) buf = window(t, buf, w[0], w[1], std::true_type());
        const float scale = n & 1 ? w4_scale<T, GS>(sp, G - 1) : -w4_scale<T, GS>(sp, G - 1);
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[TB - 1][i] = fmaf(scale, d[1][i], acc[TB - 1][i]);
        // what the last window requested may not have landed
        __builtin_amdgcn_s_waitcnt(0);
        bare_barrier();

        for (int c = 0; c < ncorr; ++c) {
#pragma unroll
            for (int i = 0; i < NLOAD; ++i) issue(from(n + c + 3), (buf + 3) & 3, i);
            u32x4 wc[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int e = c * 16 + 4 * (q >> 1) + 2 * h + (q & 1), u = min(e, n * G - 1) + t0 * G;       // group of this lane's octet
                const size_t at = (size_t)w4_block(u / G, inv) * 16 * G + u % G;
                const float z = ZP ? (float)rows.zeros[at] : 8.f;
                const float b = T::to_f32(rows.scales[at]) * (e / G & 1 ? 31.f - z : -16.f - z);
                const uint32_t b1 = e < n * G ? f32_to_bf16_bits(b) : 0u, b2 = e < n * G ? f32_to_bf16_bits(b - bf16_bits_to_f32(b1)) : 0u;
                wc[q] = u32x4{b1 | b1 << 16, b1 | b2 << 16, b2, 0u};
            }
#pragma unroll
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int q = 0; q < 8; ++q) acc[tb] = BF16::mfma32(operand(buf, tb, q), wc[q], acc[tb]);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0);
            bare_barrier();
            buf = (buf + 1) & 3;
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
};

}  // namespace mlk
