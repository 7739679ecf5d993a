// 4-bit weights with group scales: layout, widening and the streaming loop that the linear layers and the expert layers share.
//
//   W[n, k] = s[n, k / G] * (q[n, k] - z[n, k / G]),   q = 0..15, z = 0..15 (8 without zero points), s 16 bit, G = 32, 64 or a multiple of 128
//
// Codes (layout-A of 4-bit weights): tiles of 16 rows x 128 k = 1 KiB, [N/16][K/128][64 lanes][4 dwords]; lane = 16 o + r holds row r, and its
// dword j the eight codes k = 128 t + 32 j + 8 o .. + 7: one 16-byte load per lane and tile is four MFMA operands.  Inside a dword code 2 p sits
// in nibble p and code 2 p + 1 in nibble p + 4, so that one shift and one and-or make the operand's register p.
// Scales: [N/16][K/max(G,128)][16 rows][max(1, 128/G)], zero points (one byte each) the same: what a lane needs for its row and a tile is
// one load of 2 to 8 (1 to 4) bytes.
//
// No weight is rounded: 16 + q is exact in both 16-bit types (the code is the top four bits of the mantissa of a number in 16..31), so the
// matrix cores sum (16 + q) x over a group in fp32, and
//   sum over the group of W x = s * (sum (16 + q) x - (16 + z) * sum x)
// goes to the running sums with two fp32 operations per output, group and lane.  sum x comes from the matrix cores too (an operand of ones), in the
// lanes and registers where the products end.  Widening to q - z instead would need a subtraction per pair of weights, which bf16 has no packed
// instruction for; the 16 costs some two bits of the 24 that the fp32 sums hold.
//
// The products run with the tokens as rows and the weights as columns: a lane then holds one weight row (its column) and four tokens, so it needs
// one scale per tile, not four.
#pragma once

#include "mlk_common.cuh"

namespace mlk {

constexpr int kW4TileBytes = 1024;
constexpr int kW4TileK = 128;

// Group of a tile without a division: `inv` = ceil(2^32 / tiles per group), or 0 where a group is no more than a tile.  Exact for up to 2^16 tiles
// (the rounding of inv adds less than t * tpg / 2^32 < 1 / tpg).
__host__ __device__ __forceinline__ uint32_t w4_inverse(int tpg) { return tpg == 1 ? 0u : (uint32_t)((0x100000000ull + tpg - 1) / tpg); }
__device__ __forceinline__ int w4_block(int t, uint32_t inv) {
    const uint32_t keep = inv ? 0u : ~0u;                  // no branch in the loops
    return (int)(__umulhi((uint32_t)t, inv) + ((uint32_t)t & keep));
}

// Weights of one matrix (or of one expert).
struct W4Matrix {
    const uint8_t *codes;
    const uint16_t *scales;
    const uint8_t *zeros;      // null: 8 everywhere
};

// Mask and bits of 16 for the widening, held in a scalar and a vector register: v_and_or_b32 takes one constant at most, and with both as
// literals the compiler makes two instructions of it.
template <class T>
struct W4Const {
    uint32_t mask, sixteen;
    __device__ __forceinline__ W4Const() {
        mask = T::kind == MLK_BF16 ? 0x00780078u : 0x03c003c0u;
        sixteen = T::kind == MLK_BF16 ? 0x41804180u : 0x4c004c00u;
        asm volatile("" : "+s"(mask));
        asm volatile("" : "+v"(sixteen));
    }
};

// Codes 2 p and 2 p + 1 of a dword, widened to 16 + q in the type T; and all eight: an MFMA operand.
template <class T>
__device__ __forceinline__ uint32_t w4_widen1(uint32_t d, int p, const W4Const<T> &c) {
    constexpr int AT = T::kind == MLK_BF16 ? 3 : 6;        // where the four bits belong
    return ((4 * p <= AT ? d << (AT - 4 * p) : d >> (4 * p - AT)) & c.mask) | c.sixteen;
}
template <class T>
__device__ __forceinline__ u32x4 w4_widen(uint32_t d, const W4Const<T> &c) {
    return u32x4{w4_widen1<T>(d, 0, c), w4_widen1<T>(d, 1, c), w4_widen1<T>(d, 2, c), w4_widen1<T>(d, 3, c)};
}

template <class T>
__device__ __forceinline__ u32x4 w4_ones() {
    constexpr uint32_t one = T::kind == MLK_BF16 ? 0x3f803f80u : 0x3c003c00u;
    return u32x4{one, one, one, one};
}

// Scales of the 4 / GS groups of a tile (GS = k steps of 32 in a group, at most 4), and their zero points.
template <int GS>
struct W4Scale;
template <>
struct W4Scale<4> { uint32_t s, z; };
template <>
struct W4Scale<2> { uint32_t s, z; };
template <>
struct W4Scale<1> { u32x2 s; uint32_t z; };

// `at` = index of the (row group, tile or group of tiles, row) entry; ZP: there are zero points.
template <int GS, bool ZP>
__device__ __forceinline__ W4Scale<GS> w4_load_scale(const uint16_t *scales, const uint8_t *zeros, size_t at) {
    W4Scale<GS> o;
    o.z = 0x08080808u;
    if constexpr (GS == 4) {
        o.s = scales[at];
        if constexpr (ZP) o.z = zeros[at];
    } else if constexpr (GS == 2) {
        o.s = reinterpret_cast<const uint32_t *>(scales)[at];
        if constexpr (ZP) o.z = reinterpret_cast<const uint16_t *>(zeros)[at];
    } else {
        o.s = reinterpret_cast<const u32x2 *>(scales)[at];
        if constexpr (ZP) o.z = reinterpret_cast<const uint32_t *>(zeros)[at];
    }
    return o;
}
template <class T, int GS>
__device__ __forceinline__ float w4_scale(const W4Scale<GS> &c, int g) {
    if constexpr (GS == 4) return T::to_f32(c.s);
    else if constexpr (GS == 2) return T::to_f32((c.s >> (16 * g)) & 0xffffu);
    else return T::to_f32((c.s[g >> 1] >> (16 * (g & 1))) & 0xffffu);
}
template <int GS>
__device__ __forceinline__ float w4_offset(const W4Scale<GS> &c, int g) {      // 16 + z
    return 16.f + (float)((c.z >> (8 * g)) & 0xffu);
}

// One tile (128 k) of R row groups times TT blocks of 16 tokens.
template <class T, int GS, int TT, int R>
__device__ __forceinline__ void w4_tile(f32x4 (&acc)[R][TT], const u32x4 (&w)[R], const W4Scale<GS> (&sc)[R], const u32x4 (&x)[TT][4],
                                        const W4Const<T> &con) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 4 / GS; ++g) {
        f32x4 xs[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            xs[tt] = zero;
#pragma unroll
            for (int j = g * GS; j < (g + 1) * GS; ++j) xs[tt] = T::mfma(x[tt][j], w4_ones<T>(), xs[tt]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f32x4 d[TT];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) d[tt] = zero;
#pragma unroll
            for (int j = g * GS; j < (g + 1) * GS; ++j) {
                const u32x4 b = w4_widen<T>(w[r][j], con);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) d[tt] = T::mfma(x[tt][j], b, d[tt]);
            }
            const float s = w4_scale<T, GS>(sc[r], g), o = w4_offset<GS>(sc[r], g);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[r][tt][v] = fmaf(s, fmaf(-o, xs[tt][v], d[tt][v]), acc[r][tt][v]);
        }
        // The sums are taken here: left alone the compiler sinks them behind the last group and holds the products of every group until then
        // (R = 4, TT = 1, groups of 32: 204 registers, and 134 with this).
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) asm volatile("" : "+v"(acc[r][tt]));
    }
}

// Where a wave's operands come from.  Row group r of the wave is row group rg[r] of its matrix.
template <int R>
struct W4Rows {
    const uint8_t *codes[R];       // first tile of the row group
    const uint16_t *scales[R];     // first entry of the row group
    const uint8_t *zeros[R];
};
// Entries of scales per row group: `blocks` blocks of 16 rows, one for every tile or, with groups of more than 128, for every group.
template <int GS, int R>
__device__ __forceinline__ void w4_row(W4Rows<R> &rows, int r, const W4Matrix &m, size_t rg, int tiles, int blocks) {
    constexpr int per = 4 / GS;
    const size_t entries = rg * blocks * 16;
    rows.codes[r] = m.codes + rg * tiles * kW4TileBytes;
    rows.scales[r] = m.scales + entries * per;
    rows.zeros[r] = m.zeros + entries * per;
}

// acc += W . x over the tiles first, first + step, ... < end.  `xrow[tt]` is the row of this lane's token in block tt (in memory, or with XL in
// LDS: `xl`, one token, broadcast to all sixteen).  Slot u of the ring holds tile first + (i + u) step; the loads of U tiles are in flight.
template <class T, int GS, bool ZP, int TT, int R, int U, bool XL>
__device__ __forceinline__ void w4_stream(f32x4 (&acc)[R][TT], const W4Rows<R> &rows, const uint16_t *const (&xrow)[TT], const u32x4 *xl, int first,
                                          int end, int step, uint32_t inv, int lane, bool wait_x) {
    u32x4 w[U][R], x[U][XL ? 1 : TT][4];
    W4Scale<GS> sc[U][R];
    const int o = lane >> 4, r16 = lane & 15;
    const W4Const<T> con;
    auto load = [&](int u, int t) {
        const int at = w4_block(t, inv) * 16 + r16;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            w[u][r] = ld_stream_u32x4(rows.codes[r] + (size_t)t * kW4TileBytes + lane * 16);
            sc[u][r] = w4_load_scale<GS, ZP>(rows.scales[r], rows.zeros[r], at);
        }
        if constexpr (!XL) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[u][tt][j] = ld_global_u32x4(xrow[tt] + (size_t)t * kW4TileK + j * 32 + o * 8);
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    if constexpr (XL) {
        if (wait_x) __syncthreads();
    }
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
                const int t = first + (i + u) * step;
                if constexpr (XL) {
                    u32x4 xv[TT][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) xv[0][j] = xl[t * 16 + j * 4 + o];
                    w4_tile<T, GS, TT, R>(acc, w[u], sc[u], xv, con);
                } else {
                    w4_tile<T, GS, TT, R>(acc, w[u], sc[u], x[u], con);
                }
                if (i + u + U < n) load(u, t + U * step);
            }
        }
    }
}

}  // namespace mlk
