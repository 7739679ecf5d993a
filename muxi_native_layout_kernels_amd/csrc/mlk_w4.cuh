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
// goes to the running sums with one or two fp32 operations per output, group and lane.  sum x comes from the matrix cores too (an operand of ones), in the
// lanes and registers where the products end.  Widening to q - z instead would need a subtraction per pair of weights, which bf16 has no packed
// instruction for; the 16 costs some two bits of the 24 that the fp32 sums hold, more where a group's activations do not average to zero (the offset of
// one group is then larger than its sum).  The streaming loop takes the offset out of every group; the panels (mlk_w4_panel.cuh) let neighbours cancel.
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

// Widening of the codes: to 16 + q, or (ADD) to 32 + 15 - z + q, where the bits to add hold 32 + 15 - z of the row's group.  AT: where the four bits belong.
// Mask and bits of 16 live in a scalar and a vector register: v_and_or_b32 takes one constant at most, and with both as literals the compiler makes
// two instructions of it.
template <class T, bool ADD = false>
struct W4Const {
    static constexpr int AT = (T::kind == MLK_BF16 ? 3 : 6) - (ADD ? 1 : 0);
    uint32_t mask, bits;
    __device__ __forceinline__ W4Const() {
        mask = 0x000f000fu << AT;
        bits = T::kind == MLK_BF16 ? (ADD ? 0x42004200u : 0x41804180u) : (ADD ? 0x50005000u : 0x4c004c00u);
        asm volatile("" : "+s"(mask));
        asm volatile("" : "+v"(bits));
    }
    // of a group with zero point z, in both halves
    __device__ __forceinline__ uint32_t added(uint32_t z) const { return bits + (15u - z) * (0x00010001u << AT); }
};

// Codes 2 p and 2 p + 1 of a dword; and all eight: an MFMA operand.
template <class T, bool ADD>
__device__ __forceinline__ uint32_t w4_widen1(uint32_t d, int p, const W4Const<T, ADD> &c, uint32_t bits) {
    constexpr int AT = W4Const<T, ADD>::AT;
    const uint32_t q = (4 * p <= AT ? d << (AT - 4 * p) : d >> (4 * p - AT)) & c.mask;
    return ADD ? q + bits : q | bits;
}
template <class T, bool ADD>
__device__ __forceinline__ u32x4 w4_widen(uint32_t d, const W4Const<T, ADD> &c, uint32_t bits) {
    return u32x4{w4_widen1<T, ADD>(d, 0, c, bits), w4_widen1<T, ADD>(d, 1, c, bits), w4_widen1<T, ADD>(d, 2, c, bits), w4_widen1<T, ADD>(d, 3, c, bits)};
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

// How a tile takes the offset of the widened codes out again, sum (q - z) x = sum (offset + q) x - (offset + z) sum x with sum x by an operand of ones:
// where the offset is the same for all rows, as the initial value of the products' sums, whose operand of ones then holds minus the offset.  Without zero points it
// is 24; with them 47, if 15 - z is added to every pair of codes (16 instructions a row group and tile instead of four for every block of tokens and
// group: ADD from five of these on).
template <int GS, bool ZP, int TT>
__host__ __device__ constexpr bool w4_add() { return ZP && TT * (4 / GS) > 4; }
template <class T>
__device__ __forceinline__ u32x4 w4_minus24() {
    constexpr uint32_t v = T::kind == MLK_BF16 ? 0xc1c0c1c0u : 0xce00ce00u;
    return u32x4{v, v, v, v};
}
template <class T>
__device__ __forceinline__ u32x4 w4_minus47() {
    constexpr uint32_t v = T::kind == MLK_BF16 ? 0xc23cc23cu : 0xd1e0d1e0u;
    return u32x4{v, v, v, v};
}

// One tile (128 k) of R row groups times TT blocks of 16 tokens.
template <class T, int GS, bool ZP, int TT, int R>
__device__ __forceinline__ void w4_tile(f32x4 (&acc)[R][TT], const u32x4 (&w)[R], const W4Scale<GS> (&sc)[R], const u32x4 (&x)[TT][4],
                                        const W4Const<T, w4_add<GS, ZP, TT>()> &con) {
    constexpr bool ADD = w4_add<GS, ZP, TT>(), START = !ZP || ADD;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = !ZP ? w4_minus24<T>() : (ADD ? w4_minus47<T>() : w4_ones<T>());
#pragma unroll
    for (int g = 0; g < 4 / GS; ++g) {
        f32x4 xs[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            xs[tt] = zero;
#pragma unroll
            for (int j = g * GS; j < (g + 1) * GS; ++j) xs[tt] = T::mfma(x[tt][j], ones, xs[tt]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t bits = ADD ? con.added((sc[r].z >> (8 * g)) & 0xffu) : con.bits;
            f32x4 d[TT];
#pragma unroll
            for (int j = g * GS; j < (g + 1) * GS; ++j) {
                const u32x4 b = w4_widen<T, ADD>(w[r][j], con, bits);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) d[tt] = T::mfma(x[tt][j], b, j > g * GS ? d[tt] : (START ? xs[tt] : zero));
            }
            const float s = w4_scale<T, GS>(sc[r], g), o = w4_offset<GS>(sc[r], g);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[r][tt][v] = fmaf(s, START ? d[tt][v] : fmaf(-o, xs[tt][v], d[tt][v]), acc[r][tt][v]);
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
    const W4Const<T, w4_add<GS, ZP, TT>()> con;
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
                    w4_tile<T, GS, ZP, TT, R>(acc, w[u], sc[u], xv, con);
                } else {
                    w4_tile<T, GS, ZP, TT, R>(acc, w[u], sc[u], x[u], con);
                }
                if (i + u + U < n) load(u, t + U * step);
            }
        }
    }
}

}  // namespace mlk
