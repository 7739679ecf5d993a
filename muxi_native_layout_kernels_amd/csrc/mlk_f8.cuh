// Products in e4m3 with a scale for every block of 128: what the linear and the expert layers share.
//
//   y[t, n] = sum over the windows kb of 128 k of  a[t, kb] s[n / 128, kb] sum over the window of p[t, k] q[n, k]
// with codes p, q of e4m3, fp32 scales a of the activations and s of the weights.  v_mfma_f32_16x16x128_f8f6f4 multiplies a window of 16 rows x 16 tokens,
// and its sums, which start from 0, are scaled and added in fp32: one fused multiply-add an element and window, a s is one product a lane.
//
// Weights stay in layout A with one byte an element, [N/16, K/8, 16, 8], as the soft-FP8 products take them: 16 rows x 128 k are 2 KiB in a row.  The matrix
// instruction takes the k of a window in any order that both operands share.  Lane 16 q + r holds 16 q .. + 15 and 64 + 16 q .. + 15: of a row of activations two
// pieces of 16 bytes, of the weights four of 8 bytes (whole lines of 128 bytes a load and quarter).
#pragma once

#include <type_traits>

#include "mlk_common.cuh"

namespace mlk {

typedef __attribute__((ext_vector_type(8))) int i32x8;

constexpr int kF8K = 128;                    // k of a window
constexpr int kF8TileBytes = 16 * kF8K;      // 16 rows of weights

struct F8Operand {
    u32x4 v[2];
};
__device__ __forceinline__ f32x4 f8_mfma(const F8Operand &w, const F8Operand &x, f32x4 c) {
    const i32x8 a = {(int)w.v[0][0], (int)w.v[0][1], (int)w.v[0][2], (int)w.v[0][3], (int)w.v[1][0], (int)w.v[1][1], (int)w.v[1][2], (int)w.v[1][3]};
    const i32x8 b = {(int)x.v[0][0], (int)x.v[0][1], (int)x.v[0][2], (int)x.v[0][3], (int)x.v[1][0], (int)x.v[1][1], (int)x.v[1][2], (int)x.v[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);      // e4m3 both, no scales
}

// ---------------------------------------------------------------------------------------------------------------- quantising
// The scale of a block is the smallest power of two, 2^-100 at least, with max |x| <= 448 scale: a power of two loses nothing on the way, so codes do not depend on
// how they are computed, and a floating format keeps its relative precision under it.  The exponent from the bits of the maximum (0 for none): m 2^e with 1 <= m < 2 fits
// 448 = 1.75 2^8 from scale 2^(e - 8) on if m <= 1.75.
__device__ __forceinline__ int f8_exponent(float most) {
    const uint32_t b = __float_as_uint(most);
    return max((int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), -100);
}
__device__ __forceinline__ float f8_two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// |x| if it counts in the maximum: infinities and NaN do not
__device__ __forceinline__ float f8_magnitude(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}
// Four values times 2^-e as codes, round to nearest even; infinities and NaN become the NaN code.
__device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d, float inverse) {
    auto scaled = [&](float x) { return fabsf(x) < INFINITY ? x * inverse : __uint_as_float(0x7fc00000u); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(a), scaled(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(c), scaled(d), w, true);
}

// Largest value of the 16 lanes that a lane belongs to.
__device__ __forceinline__ float f8_max16(float v) {
    auto other = [](float x, auto ctrl) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
    v = fmaxf(v, other(v, std::integral_constant<int, 0xb1>()));         // lane ^ 1
    v = fmaxf(v, other(v, std::integral_constant<int, 0x4e>()));         // lane ^ 2
    v = fmaxf(v, other(v, std::integral_constant<int, 0x141>()));        // the other quad of 8
    return fmaxf(v, other(v, std::integral_constant<int, 0x140>()));     // the other 8
}

// Eight values of a lane as they lie in memory.
template <class T>
struct F8In {
    u32x4 raw;
    __device__ __forceinline__ void load(const void *x, size_t i) { raw = ld_stream_u32x4(reinterpret_cast<const uint16_t *>(x) + i); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = T::to_f32(raw[j] & 0xffffu);
            v[2 * j + 1] = T::to_f32(raw[j] >> 16);
        }
    }
};
template <>
struct F8In<float> {
    f32x4 lo, hi;
    __device__ __forceinline__ void load(const void *x, size_t i) {
        lo = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(x) + i));
        hi = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(x) + i) + 1);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = lo[j];
            v[4 + j] = hi[j];
        }
    }
};

// Eight codes as bf16, exactly.
__device__ __forceinline__ u32x4 f8_widen(u32x2 q) {
    uint32_t a, b, c, d;
    fp8x4_to_bf16x4_pow2(q[0], 1.f, a, b);
    fp8x4_to_bf16x4_pow2(q[1], 1.f, c, d);
    return u32x4{a, b, c, d};
}

// One block of 128 by 16 lanes of eight values: codes of this lane, scale of the block.
__device__ __forceinline__ u32x2 f8_block(const float (&v)[8], float &scale) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fmaxf(most, f8_magnitude(v[j]));
    const int e = f8_exponent(f8_max16(most));
    scale = f8_two_to(e);
    const float inverse = f8_two_to(-e);
    return u32x2{f8_codes(v[0], v[1], v[2], v[3], inverse), f8_codes(v[4], v[5], v[6], v[7], inverse)};
}

// x [T][K] of kind x_kind (fp32 too) -> codes [T][K], scales [K / 128][T] (token t's block kb at kb scale_k + t scale_t).
int launch_quantize_fp8(const void *x, int x_kind, uint8_t *codes, float *scales, int64_t scale_t, int64_t scale_k, int64_t T, int K, hipStream_t s);

// ---------------------------------------------------------------------------------------------------------------- streaming
// Row group r of a wave: its tiles of 128 k, and the scales of the 128 rows that it lies in, one a window.
template <int R>
struct F8Rows {
    const uint8_t *w[R];
    const float *s[R];
};
template <int R>
__device__ __forceinline__ void f8_row(F8Rows<R> &rows, int r, const uint8_t *w, const float *s, size_t rg, int windows) {
    rows.w[r] = w + rg * windows * kF8TileBytes;
    rows.s[r] = s + (rg >> 3) * windows;
}

// This lane's token of each block of 16: its codes, and where its scales are.
template <int TT>
struct F8Tokens {
    const uint8_t *x[TT];
    const float *a[TT];
    size_t step;                 // floats from one window's scale to the next
};
// The same of one block of tokens that lies in LDS: windows first .. of this lane's token.
struct F8Staged {
    const u32x4 *x;              // eight pieces of 16 bytes a window
    const float *a;
    int first;
};

__device__ __forceinline__ void f8_load_weights(F8Operand &o, const uint8_t *tile, int lane) {
    const uint8_t *at = tile + (lane >> 4) * 256 + (lane & 15) * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const u32x2 a = ld_stream_u32x2(at + h * 1024), b = ld_stream_u32x2(at + h * 1024 + 128);
        o.v[h] = u32x4{a[0], a[1], b[0], b[1]};
    }
}
__device__ __forceinline__ void f8_load_tokens(F8Operand &o, const uint8_t *row, int lane) {
    const uint8_t *at = row + (lane >> 4) * 16;
    o.v[0] = ld_global_u32x4(at);
    o.v[1] = ld_global_u32x4(at + 64);
}

// One window: acc += s a (w . x).
template <int TT, int R>
__device__ __forceinline__ void f8_window(f32x4 (&acc)[R][TT], const F8Operand (&w)[R], const float (&s)[R], const F8Operand (&x)[TT], const float (&a)[TT]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const f32x4 d = f8_mfma(w[r], x[tt], f32x4{0.f, 0.f, 0.f, 0.f});
            const float c = s[r] * a[tt];
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[r][tt][v] = fmaf(c, d[v], acc[r][tt][v]);
        }
}

// acc += the windows first, first + step, ... < end.  The loads of U windows are in flight.
template <int TT, int R, int U>
__device__ __forceinline__ void f8_stream(f32x4 (&acc)[R][TT], const F8Rows<R> &rows, const F8Tokens<TT> &tokens, int first, int end, int step, int lane) {
    F8Operand w[U][R], x[U][TT];
    float s[U][R], a[U][TT];
    auto load = [&](int u, int t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f8_load_weights(w[u][r], rows.w[r] + (size_t)t * kF8TileBytes, lane);
            s[u][r] = rows.s[r][t];
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            f8_load_tokens(x[u][tt], tokens.x[tt] + (size_t)t * kF8K, lane);
            a[u][tt] = tokens.a[tt][(size_t)t * tokens.step];
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
                f8_window<TT, R>(acc, w[u], s[u], x[u], a[u]);
                if (i + u + U < n) load(u, first + (i + u + U) * step);
            }
        }
    }
}

// The same with the tokens in LDS: `ready` is called behind the first loads and ahead of the first read of a token.
template <int R, int U, class Ready>
__device__ __forceinline__ void f8_stream_staged(f32x4 (&acc)[R][1], const F8Rows<R> &rows, const F8Staged &tokens, int first, int end, int step, int lane, Ready ready) {
    F8Operand w[U][R];
    float s[U][R];
    auto load = [&](int u, int t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f8_load_weights(w[u][r], rows.w[r] + (size_t)t * kF8TileBytes, lane);
            s[u][r] = rows.s[r][t];
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    ready();
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
                const int t = first + (i + u) * step - tokens.first;
                F8Operand x[1];
                x[0].v[0] = tokens.x[t * 8 + (lane >> 4)];
                x[0].v[1] = tokens.x[t * 8 + 4 + (lane >> 4)];
                const float a[1] = {tokens.a[t]};
                f8_window<1, R>(acc, w[u], s[u], x, a);
                if (i + u + U < n) load(u, first + (i + u + U) * step);
            }
        }
    }
}

// The same with tokens of 16 bits that the wave quantises on the way: a window of a token lies in four lanes, 32 values in each, so its maximum is two exchanges.  Each window of the
// tokens is quantised once a workgroup, by the wave that multiplies it.
struct F8Raw {
    u32x4 v[4];                  // values 16 q .. + 7, + 8 .. + 15, 64 + 16 q .. and + 8 of the window
};
template <int TT>
struct F8RawTokens {
    const uint16_t *x[TT];
};
template <class T>
__device__ __forceinline__ void f8_quantize_operand(const F8Raw &in, F8Operand &o, float &scale) {
    float v[32], most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        v[2 * i] = T::to_f32(in.v[i >> 2][i & 3] & 0xffffu);
        v[2 * i + 1] = T::to_f32(in.v[i >> 2][i & 3] >> 16);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) most = fmaxf(most, f8_magnitude(v[i]));
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const int e = f8_exponent(most);
    scale = f8_two_to(e);
    const float inverse = f8_two_to(-e);
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i >> 2][i & 3] = f8_codes(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inverse);
}
template <class T, int TT, int R, int U>
__device__ __forceinline__ void f8_stream_raw(f32x4 (&acc)[R][TT], const F8Rows<R> &rows, const F8RawTokens<TT> &tokens, int first, int end, int step, int lane) {
    F8Operand w[U][R];
    F8Raw x[U][TT];
    float s[U][R];
    auto load = [&](int u, int t) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const uint16_t *at = tokens.x[tt] + (size_t)t * kF8K + (lane >> 4) * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][tt].v[j] = ld_global_u32x4(at + (j >> 1) * 64 + (j & 1) * 8);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f8_load_weights(w[u][r], rows.w[r] + (size_t)t * kF8TileBytes, lane);
            s[u][r] = rows.s[r][t];
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
                F8Operand o[TT];
                float a[TT];
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) f8_quantize_operand<T>(x[u][tt], o[tt], a[tt]);
                f8_window<TT, R>(acc, w[u], s[u], o, a);
                if (i + u + U < n) load(u, first + (i + u + U) * step);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- products that feed codes
// The matrix cores add eight products of e4m3 with 13 bits below the largest of them (measured: any shape of the instruction, cut off towards zero), 1.4e-5 of a sum over many in the
// root mean square, and up to 9e-5 where a few columns of the activations are 30 to 1000 times larger than the rest.  Against the rounding of a result that is little (fp16 of such columns 2.07e-4 ->
// 2.26e-4, bf16 not to be seen), but what becomes a code next moves to a neighbour wherever a border lies that near, and with the largest of a block its scale: expert layers of 2048 x 512 with gate
// and up from such sums are 1.8e-3 to 3.6e-3 off the definition, single tokens up to 1.9e-2, where bf16 rounds by 1.66e-3 (fp16 by 2.1e-4, quantising itself costs 2.6e-2).  So gate and up go through
// v_mfma_f32_16x16x32_bf16: codes are exact in bf16 and so are their products, a window is four instructions, whose sums round to fp32 as those of the windows do.  Then only the results' own rounding is seen.
// Where the weights' bytes set the pace widening the weights hides behind their loads; the panels pay for it (mlk_f8_moe_panel.cuh).  Lane 16 q + r holds octet 4 j + q of row r: 512 bytes a load in a row.
struct F8WideOperand {
    u32x4 v[4];
};
struct F8RawTile {
    u32x2 v[4];
};
__device__ __forceinline__ void f8_load_tile(F8RawTile &o, const uint8_t *tile, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = ld_stream_u32x2(tile + j * 512 + lane * 8);
}
__device__ __forceinline__ void f8_widen(const F8Operand &in, F8WideOperand &o) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = f8_widen(u32x2{in.v[j >> 1][(j & 1) * 2], in.v[j >> 1][(j & 1) * 2 + 1]});
}
__device__ __forceinline__ f32x4 f8_wide_mfma(const F8RawTile &w, const F8WideOperand &x) {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) d = BF16::mfma(f8_widen(w.v[j]), x.v[j], d);
    return d;
}

// f8_stream with the tokens' codes as bf16, 256 bytes a window: tokens.x are rows of those.
template <int TT, int R, int U>
__device__ __forceinline__ void f8_wide_stream(f32x4 (&acc)[R][TT], const F8Rows<R> &rows, const F8Tokens<TT> &tokens, int first, int end, int step, int lane) {
    F8RawTile w[U][R];
    F8WideOperand x[U][TT];
    float s[U][R], a[U][TT];
    auto load = [&](int u, int t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f8_load_tile(w[u][r], rows.w[r] + (size_t)t * kF8TileBytes, lane);
            s[u][r] = rows.s[r][t];
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][tt].v[j] = ld_global_u32x4(tokens.x[tt] + (size_t)t * 256 + j * 64 + (lane >> 4) * 16);
            a[u][tt] = tokens.a[tt][(size_t)t * tokens.step];
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) {
                        const f32x4 d = f8_wide_mfma(w[u][r], x[u][tt]);
                        const float c = s[u][r] * a[u][tt];
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[r][tt][v] = fmaf(c, d[v], acc[r][tt][v]);
                    }
                if (i + u + U < n) load(u, first + (i + u + U) * step);
            }
        }
    }
}
// The same of one token in LDS, whose windows begin at `x` (16 pieces of 16 bytes each) with scales at `a`: all sixteen columns are that token.
template <int R, int U, class Ready>
__device__ __forceinline__ void f8_wide_stream_staged(f32x4 (&acc)[R][1], const F8Rows<R> &rows, const u32x4 *x, const float *a, int first, int end, int step, int lane,
                                                      Ready ready) {
    F8RawTile w[U][R];
    float s[U][R];
    auto load = [&](int u, int t) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            f8_load_tile(w[u][r], rows.w[r] + (size_t)t * kF8TileBytes, lane);
            s[u][r] = rows.s[r][t];
        }
    };
    const int n = end > first ? (end - first + step - 1) / step : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) load(u, first + u * step);
    ready();
    for (int i = 0; i < n; i += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u < n) {
                const int t = first + (i + u) * step;
                F8WideOperand o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o.v[j] = x[t * 16 + j * 4 + (lane >> 4)];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const f32x4 d = f8_wide_mfma(w[u][r], o);
                    const float c = s[u][r] * a[t];
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[r][0][v] = fmaf(c, d[v], acc[r][0][v]);
                }
                if (i + u + U < n) load(u, first + (i + u + U) * step);
            }
        }
    }
}

}  // namespace mlk
