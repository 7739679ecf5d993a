// Router logits of the three kinds in registers, and folds over the lanes that hold a token: for the balance loss and the routing.
#pragma once

#include <type_traits>

#include "mlk_common.cuh"

namespace mlk {

struct BalF32 {
    typedef f32x4 V4;
    typedef float V1;
    __device__ static __forceinline__ void unpack(const f32x4 &v, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
    }
    __device__ static __forceinline__ f32x4 pack(const float (&x)[4]) { return f32x4{x[0], x[1], x[2], x[3]}; }
    __device__ static __forceinline__ float to_f32(float v) { return v; }
    __device__ static __forceinline__ float from_f32(float v) { return v; }
};
template <class T>
struct Bal16 {
    typedef u32x2 V4;
    typedef uint16_t V1;
    __device__ static __forceinline__ void unpack(const u32x2 &v, float (&x)[4]) {
        x[0] = T::to_f32(v[0] & 0xffffu);
        x[1] = T::to_f32(v[0] >> 16);
        x[2] = T::to_f32(v[1] & 0xffffu);
        x[3] = T::to_f32(v[1] >> 16);
    }
    __device__ static __forceinline__ u32x2 pack(const float (&x)[4]) { return u32x2{T::from_f32x2(x[0], x[1]), T::from_f32x2(x[2], x[3])}; }
    __device__ static __forceinline__ float to_f32(uint16_t v) { return T::to_f32(v); }
    __device__ static __forceinline__ uint16_t from_f32(float v) { return (uint16_t)T::from_f32(v); }
};

// A value of another lane of the same 16, without LDS: lane ^ 1, lane ^ 2 (quad_perm), the other quad of 8 and the other 8 (mirrors).
template <int STEP>
__device__ __forceinline__ float bal_other(float v) {
    constexpr int ctrl = STEP == 1 ? 0xb1 : (STEP == 2 ? 0x4e : (STEP == 4 ? 0x141 : 0x140));
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xf, 0xf, true));
}
template <int LPT, class F>
__device__ __forceinline__ float bal_fold(float v, F f) {
    v = f(v, bal_other<1>(v));
    v = f(v, bal_other<2>(v));
    if constexpr (LPT >= 8) v = f(v, bal_other<4>(v));
    if constexpr (LPT >= 16) v = f(v, bal_other<8>(v));
    return v;
}

}  // namespace mlk
