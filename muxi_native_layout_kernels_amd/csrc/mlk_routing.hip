// Routing to experts that trains: the picks of each token with their weights, and the gradient of the logits.
//
//   rank      the logits themselves, or with a bias the scores + bias in 64 bits (neighbours keep their order there); scores are softmax(x) or sigmoid(x)
//   groups    score of a group: its largest rank, with a bias the sum of its two largest; the best `kept` groups stay, ties to the lower group
//   picks     the K largest ranks, ties to the lower expert.  Experts with logits or biases of -inf or NaN are never picked: id -1, weight 0.  A logit of
//             +inf counts as the largest finite number
//   weights   w = c s / S (renormalised) or c s, s the score without bias and S its sum over the picks
// Renormalised weights do not need the score's denominator: softmax gives exp(x - m) over their sum, sigmoids e^(x - min(m, 0)) / (1 + e^x), which neither loses the bits of
// small ones nor underflows (m the largest picked logit).  With w' = s / S and g the gradient of w:
//   dx_k = (c g_k - sum c g w') w'_k r_k  (renormalised),  c g_k s_k r_k  (sigmoid),  c g_k s_k - s_k sum c g s over the picks, - s_e sum c g s elsewhere  (softmax)
// with r = 1 - sigmoid, 1 for softmax.
//
// 16 lanes take a token (64 where tokens are few and experts many), so that a wave takes four at a time and a maximum over the experts is four exchanges within 16 lanes.
// After the picks lane k holds pick k.
//
// What bounds it: a chain of dependent steps (the load, of biased ranks the exponentials and divisions in 64 bits, then K times a maximum over registers and lanes), not the bytes.
// 256 experts in 8 groups, 8 picks, bias, fp32: 16 tokens 7.1 us, 8191 tokens 17.2 us (9 MB; 27.3 with 64-bit exchanges through LDS, all ranks of a group read by its lane and
// the picks' logits read again from memory); 64 experts, 6 picks, bf16, 16384 tokens 5.7 us.  Gradient of the same: 3.6, 4.6 and 4.4 us, of which a launch is 3.
#include <algorithm>

#include "mlk_logits.cuh"

namespace mlk {

constexpr int kRouteExperts = 512;
constexpr int kRoutePicks = 32;

struct RouteArgs {
    const void *logits;          // [T][E]
    const float *bias;           // [E] or null
    const uint8_t *mask;         // [T] or null
    int T, E, K, G, kept, score_fun, renorm;
    float scaling;
    int32_t *ids;                // [T][K]
    void *weights;               // [T][K]
    const void *dweights;        // [T][K]
    void *dlogits;               // [T][E]
};

// A value of another lane of the same 16 (bal_other), of 32 or 64 bits; of lane `from` of the wave.
template <int STEP, class V>
__device__ __forceinline__ V route_other(V v) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, bal_other<STEP>(__builtin_bit_cast(float, v)));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __float_as_uint(bal_other<STEP>(__uint_as_float((uint32_t)b))), hi = __float_as_uint(bal_other<STEP>(__uint_as_float((uint32_t)(b >> 32))));
        return __builtin_bit_cast(V, (uint64_t)hi << 32 | lo);
    }
}
template <class V>
__device__ __forceinline__ V route_from(V v, int from) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), from));
    } else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(V, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, from));
    }
}
template <int LPT, class V, class F>
__device__ __forceinline__ V route_fold(V v, F f) {
    v = f(v, route_other<1>(v));
    v = f(v, route_other<2>(v));
    v = f(v, route_other<4>(v));
    v = f(v, route_other<8>(v));
    if constexpr (LPT == 64) v = f(f(route_from(v, 0), route_from(v, 16)), f(route_from(v, 32), route_from(v, 48)));
    return v;
}
template <int LPT>
__device__ __forceinline__ float route_sum(float v) { return route_fold<LPT>(v, [](float a, float b) { return a + b; }); }
template <int LPT>
__device__ __forceinline__ float route_max(float v) { return route_fold<LPT>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int LPT>
__device__ __forceinline__ int route_min(int v) { return route_fold<LPT>(v, [](int a, int b) { return min(a, b); }); }

// A logit as it counts: -inf for NaN, the largest finite number for +inf.
__device__ __forceinline__ float route_logit(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }

// Experts of a lane: slot 4 v + i holds 4 (v LPT + lane) + i.
template <int LPT>
__device__ __forceinline__ int route_expert(int slot, int l) { return ((slot >> 2) * LPT + l) * 4 + (slot & 3); }
template <class L, int LPT, int NE>
__device__ __forceinline__ void route_load(const RouteArgs &p, int t, int l, bool vec, float (&x)[NE]) {
    const typename L::V1 *row = reinterpret_cast<const typename L::V1 *>(p.logits) + (size_t)t * p.E;
    if (vec) {
        typename L::V4 raw[NE / 4];
#pragma unroll
        for (int v = 0; v < NE / 4; ++v) raw[v] = *reinterpret_cast<const typename L::V4 *>(row + min(route_expert<LPT>(4 * v, l), p.E - 4));
#pragma unroll
        for (int v = 0; v < NE / 4; ++v) {
            float y[4];
            L::unpack(raw[v], y);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * v + i] = route_expert<LPT>(4 * v, l) + i < p.E ? route_logit(y[i]) : -INFINITY;
        }
    } else {
#pragma unroll
        for (int s = 0; s < NE; ++s) {
            const int e = route_expert<LPT>(s, l);
            const float y = L::to_f32(row[min(e, p.E - 1)]);
            x[s] = e < p.E ? route_logit(y) : -INFINITY;
        }
    }
}

// Score of the picks of a lane, 0 for none (x = -inf), and 1 - sigmoid.  m: the largest of the picks; renormalised: of sigmoids e^-min(m, 0) times, of softmax e^-m and
// without the denominator.
__device__ __forceinline__ float route_score(const RouteArgs &p, float x, float m, float &rest) {
    rest = 1.f;
    if (x == -INFINITY) return 0.f;
    if (p.score_fun == 0) return expf(x - m);
    const float low = p.renorm ? fminf(m, 0.f) : 0.f, e = expf(-fabsf(x)), r = 1.f / (1.f + e);
    rest = x >= 0.f ? e * r : r;
    return x >= 0.f ? r : expf(x - low) * r;
}

// The two largest of a group's ranks, as they come.
template <class V>
struct RouteBest {
    V a, b;
    __device__ __forceinline__ void add(V v) {
        b = v > a ? a : (v > b ? v : b);
        a = v > a ? v : a;
    }
};

// Places of the ranks and of the groups of a token in LDS; an even number, so that the next token's lie on whole words.
__host__ __device__ __forceinline__ int route_lds(int E, int G) { return G > 1 ? (E + G + 1) & ~1 : 0; }

// V: what picks are ranked by, float or double.
// LDS of a token, in V: two largest of each four consecutive experts that share a group (QUADS) or all ranks, a score and then a flag a group; then, of doubles, the logits.
template <class L, int LPT, int NE, class V>
__global__ void __launch_bounds__(64) route_kernel(RouteArgs p, bool vec) {
    constexpr int TOK = 64 / LPT;
    constexpr bool BIASED = sizeof(V) == 8;
    extern __shared__ char lds[];
    const int l = threadIdx.x & (LPT - 1), mine = threadIdx.x / LPT, t = min((int)blockIdx.x * TOK + mine, p.T - 1);
    const bool here = (int)blockIdx.x * TOK + mine < p.T;
    const V lowest = -INFINITY;
    V *ranks = reinterpret_cast<V *>(lds) + (size_t)mine * route_lds(p.E, p.G), *best = ranks + p.E;
    float *logits = reinterpret_cast<float *>(reinterpret_cast<V *>(lds) + (size_t)TOK * route_lds(p.E, p.G)) + (size_t)mine * p.E;
    float x[NE], bias[NE];
    if constexpr (BIASED)
#pragma unroll
        for (int s = 0; s < NE; ++s) bias[s] = p.bias[min(route_expert<LPT>(s, l), p.E - 1)];
    route_load<L, LPT, NE>(p, t, l, vec, x);
    const bool valid = !p.mask || p.mask[t];
    V rank[NE];
    float top = -INFINITY, sum = 1.f;
#pragma unroll
    for (int s = 0; s < NE; ++s) {
        top = fmaxf(top, x[s]);
        rank[s] = x[s];
    }
    if constexpr (BIASED) {
        double total = 1.;
        if (p.score_fun == 0) {
            top = route_max<LPT>(top);
            total = 0.;
#pragma unroll
            for (int s = 0; s < NE; ++s) {
                rank[s] = x[s] == -INFINITY ? 0. : exp((double)x[s] - (double)top);
                total += rank[s];
            }
            total = route_fold<LPT>(total, [](double a, double b) { return a + b; });
            sum = (float)total;
#pragma unroll
            for (int s = 0; s < NE; ++s) rank[s] /= total;
        } else {
#pragma unroll
            for (int s = 0; s < NE; ++s) rank[s] = 1. / (1. + exp(-(double)x[s]));
        }
#pragma unroll
        for (int s = 0; s < NE; ++s) {
            const int e = route_expert<LPT>(s, l);
            if (e < p.E) logits[e] = x[s];
            rank[s] = e >= p.E || x[s] == -INFINITY || bias[s] != bias[s] ? lowest : rank[s] + (double)bias[s];
        }
    } else if (p.score_fun == 0 && !p.renorm) {
        top = route_max<LPT>(top);
        sum = 0.f;
#pragma unroll
        for (int s = 0; s < NE; ++s) sum += x[s] == -INFINITY ? 0.f : expf(x[s] - top);
        sum = route_sum<LPT>(sum);
    }
    if (p.G > 1) {
        const int each = p.E / p.G;
        const bool quads = (each & 3) == 0;
        if (quads) {
#pragma unroll
            for (int v = 0; v < NE / 4; ++v) {
                RouteBest<V> q = {rank[4 * v], lowest};
                for (int i = 1; i < 4; ++i) q.add(rank[4 * v + i]);
                const int e = route_expert<LPT>(4 * v, l);
                if (e < p.E) {
                    ranks[e >> 1] = q.a;
                    ranks[(e >> 1) + 1] = q.b;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < NE; ++s) {
                const int e = route_expert<LPT>(s, l);
                if (e < p.E) ranks[e] = rank[s];
            }
        }
        wave_lds_sync();
        const int n = quads ? each >> 1 : each;
        for (int g = l; g < p.G; g += LPT) {
            RouteBest<V> q = {lowest, lowest};
#pragma unroll 8
            for (int i = 0; i < n; ++i) q.add(ranks[g * n + i]);
            best[g] = BIASED && q.b != lowest ? q.a + q.b : q.a;
        }
        wave_lds_sync();
        // a group stays if fewer than `kept` are better, or as good and lower; the flags take the place of the ranks
        for (int g = l; g < p.G; g += LPT) {
            const V own = best[g];
            int ahead = 0;
#pragma unroll 8
            for (int q = 0; q < p.G; ++q) ahead += best[q] > own || (best[q] == own && q < g) ? 1 : 0;
            ranks[g] = ahead < p.kept ? (V)0 : lowest;
        }
        wave_lds_sync();
        if (quads) {
#pragma unroll
            for (int v = 0; v < NE / 4; ++v) {
                const V keep = ranks[min(route_expert<LPT>(4 * v, l) / each, p.G - 1)];
#pragma unroll
                for (int i = 0; i < 4; ++i) rank[4 * v + i] = keep == lowest ? lowest : rank[4 * v + i];
            }
        } else {
#pragma unroll
            for (int s = 0; s < NE; ++s) rank[s] = ranks[min(route_expert<LPT>(s, l) / each, p.G - 1)] == lowest ? lowest : rank[s];
        }
    }
    // K times the largest, then the lowest expert that has it
    int id[2] = {-1, -1};
    float xk[2] = {-INFINITY, -INFINITY};
    for (int k = 0; k < p.K; ++k) {
        V high = rank[0];
#pragma unroll
        for (int s = 1; s < NE; ++s) high = rank[s] > high ? rank[s] : high;
        high = route_fold<LPT>(high, [](V a, V b) { return a > b ? a : b; });
        int at = 0x7fffffff;
#pragma unroll
        for (int s = NE - 1; s >= 0; --s) at = rank[s] == high ? route_expert<LPT>(s, l) : at;
        at = route_min<LPT>(at);
#pragma unroll
        for (int s = 0; s < NE; ++s) rank[s] = route_expert<LPT>(s, l) == at ? lowest : rank[s];
        if ((k & (LPT - 1)) == l && high != lowest) {
            id[k / LPT] = at;
            if constexpr (!BIASED) xk[k / LPT] = high;
        }
    }
    if constexpr (BIASED) {
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (id[j] >= 0) xk[j] = logits[id[j]];
    }
    const float m = p.renorm ? route_max<LPT>(fmaxf(xk[0], xk[1])) : top;
    float s[2], rest;
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = route_score(p, xk[j], m, rest);
    if (p.renorm) sum = route_sum<LPT>(s[0] + s[1]);
    else if (p.score_fun != 0) sum = 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int k = j * LPT + l;
        if (!here || k >= p.K) continue;
        p.ids[(size_t)t * p.K + k] = valid ? id[j] : -1;
        reinterpret_cast<typename L::V1 *>(p.weights)[(size_t)t * p.K + k] = L::from_f32(valid && id[j] >= 0 ? p.scaling * (s[j] / sum) : 0.f);
    }
}

// The gradient of a token's row goes through LDS: zeros, or the share of the softmax's denominator, and the picks' on top.
template <class L, int LPT, int NE>
__global__ void __launch_bounds__(64) route_grad_kernel(RouteArgs p, bool vec) {
    constexpr int TOK = 64 / LPT;
    __shared__ float row[TOK][LPT * NE];
    const int l = threadIdx.x & (LPT - 1), mine = threadIdx.x / LPT, t = min((int)blockIdx.x * TOK + mine, p.T - 1);
    const bool here = (int)blockIdx.x * TOK + mine < p.T;
    typedef typename L::V1 E1;
    int id[2];
    float g[2], xk[2], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int k = j * LPT + l;
        id[j] = k < p.K ? p.ids[(size_t)t * p.K + k] : -1;
        g[j] = id[j] >= 0 ? p.scaling * L::to_f32(reinterpret_cast<const E1 *>(p.dweights)[(size_t)t * p.K + k]) : 0.f;
        xk[j] = id[j] >= 0 ? route_logit(L::to_f32(reinterpret_cast<const E1 *>(p.logits)[(size_t)t * p.E + id[j]])) : -INFINITY;
        m = fmaxf(m, xk[j]);
    }
    float d[NE];
#pragma unroll
    for (int s = 0; s < NE; ++s) d[s] = 0.f;
    const bool all = p.score_fun == 0 && !p.renorm;       // every logit is in the denominator
    float sum = 1.f;
    if (all) {
        float top = -INFINITY;
        route_load<L, LPT, NE>(p, t, l, vec, d);
#pragma unroll
        for (int s = 0; s < NE; ++s) top = fmaxf(top, d[s]);
        m = route_max<LPT>(top);
        sum = 0.f;
#pragma unroll
        for (int s = 0; s < NE; ++s) {
            d[s] = d[s] == -INFINITY ? 0.f : expf(d[s] - m);
            sum += d[s];
        }
        sum = route_sum<LPT>(sum);
    } else {
        m = route_max<LPT>(m);
    }
    float s[2], rest[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = route_score(p, xk[j], m, rest[j]);
    if (p.renorm) sum = route_sum<LPT>(s[0] + s[1]);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        s[j] *= inv;
        dot = fmaf(g[j], s[j], dot);
    }
    dot = p.renorm || all ? route_sum<LPT>(dot) : 0.f;
    if (all) {
        const float c = -dot * inv;
#pragma unroll
        for (int q = 0; q < NE; ++q) d[q] *= c;
    }
#pragma unroll
    for (int v = 0; v < NE / 4; ++v)
        *reinterpret_cast<f32x4 *>(&row[mine][route_expert<LPT>(4 * v, l)]) = f32x4{d[4 * v], d[4 * v + 1], d[4 * v + 2], d[4 * v + 3]};
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (id[j] >= 0) row[mine][id[j]] = (g[j] - dot) * s[j] * rest[j];
    wave_lds_sync();
    if (!here) return;
    E1 *out = reinterpret_cast<E1 *>(p.dlogits) + (size_t)t * p.E;
#pragma unroll
    for (int v = 0; v < NE / 4; ++v) {
        const int e = route_expert<LPT>(4 * v, l);
        const f32x4 q = *reinterpret_cast<const f32x4 *>(&row[mine][e]);
        const float y[4] = {q[0], q[1], q[2], q[3]};
        if (vec) {
            if (e < p.E) *reinterpret_cast<typename L::V4 *>(out + e) = L::pack(y);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + i < p.E) out[e + i] = L::from_f32(y[i]);
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------- host
template <class L, int LPT, int NE>
static void route_launch(const RouteArgs &a, bool vec, bool grad, hipStream_t s) {
    const int wgs = (a.T + 64 / LPT - 1) / (64 / LPT);
    const size_t lds = (size_t)(64 / LPT) * (route_lds(a.E, a.G) * (a.bias ? 8 : 4) + (a.bias ? a.E * 4 : 0));
    if (grad) route_grad_kernel<L, LPT, NE><<<wgs, 64, 0, s>>>(a, vec);
    else if (a.bias) route_kernel<L, LPT, NE, double><<<wgs, 64, lds, s>>>(a, vec);
    else route_kernel<L, LPT, NE, float><<<wgs, 64, lds, s>>>(a, vec);
}
template <class L>
static void route_launch_size(const RouteArgs &a, bool vec, bool grad, hipStream_t s) {
    // 16 -> 64 lanes a token: 256 experts with bias at 16 tokens 11.1 -> 7.1 us, 2048 12.2 -> 10.4, 4096 12.9 -> 12.8, 8191 17.2 -> 21.1; 512 at 4096 19.2 -> 16.6, 8191
    // 26.6 -> 28.2; 160 experts without bias at 1024 6.8 -> 5.4; 64 experts at 16 tokens 3.4 -> 4.8
    if (a.T <= 4096 && a.E > 64) {
        if (a.E <= 256) route_launch<L, 64, 4>(a, vec, grad, s);
        else route_launch<L, 64, 8>(a, vec, grad, s);
    } else if (a.E <= 64) {
        route_launch<L, 16, 4>(a, vec, grad, s);
    } else if (a.E <= 128) {
        route_launch<L, 16, 8>(a, vec, grad, s);
    } else if (a.E <= 256) {
        route_launch<L, 16, 16>(a, vec, grad, s);
    } else {
        route_launch<L, 16, 32>(a, vec, grad, s);
    }
}
static void route_launch_kind(const RouteArgs &a, int kind, bool vec, bool grad, hipStream_t s) {
    if (kind == MLK_F32) route_launch_size<BalF32>(a, vec, grad, s);
    else if (kind == MLK_F16) route_launch_size<Bal16<F16>>(a, vec, grad, s);
    else route_launch_size<Bal16<BF16>>(a, vec, grad, s);
}
// A launch has fewer than 2^32 threads: at 16 a token up to 2^27 tokens each, 128 tokens of whatever type on 16 bytes (route_vec holds for all parts).
constexpr int kRouteTokens = 1 << 27;
static int route_launch_all(const RouteArgs &all, int kind, bool vec, bool grad, hipStream_t s) {
    const size_t size = kind == MLK_F32 ? 4 : 2;
    auto at = [&](const void *p, size_t bytes) { return p ? (void *)((uintptr_t)p + bytes) : nullptr; };
    for (int t0 = 0; t0 < all.T; t0 += std::min(kRouteTokens, all.T - t0)) {
        RouteArgs a = all;
        a.T = std::min(kRouteTokens, all.T - t0);
        a.logits = at(all.logits, (size_t)t0 * a.E * size);
        a.mask = all.mask ? all.mask + t0 : nullptr;
        a.ids = all.ids + (size_t)t0 * a.K;
        a.weights = at(all.weights, (size_t)t0 * a.K * size);
        a.dweights = at(all.dweights, (size_t)t0 * a.K * size);
        a.dlogits = at(all.dlogits, (size_t)t0 * a.E * size);
        route_launch_kind(a, kind, vec, grad, s);
        MLK_LAUNCH_CHECK();
    }
    return MLK_OK;
}
static bool route_vec(const void *p, int kind, int E) { return E % 4 == 0 && ((uintptr_t)p & (kind == MLK_F32 ? 15 : 7)) == 0; }

static int route_check(const void *logits, int kind, int score_fun, int T, int E, int K) {
    MLK_REQUIRE(kind == MLK_F16 || kind == MLK_BF16 || kind == MLK_F32, "routing: logits must be fp16, bf16 or fp32");
    MLK_REQUIRE(score_fun == 0 || score_fun == 1, "routing: score function must be 0 (softmax) or 1 (sigmoid)");
    MLK_REQUIRE(T >= 0 && T <= (1 << 30), "routing: 0..2^30 tokens");
    MLK_REQUIRE(E >= 1 && E <= kRouteExperts, "routing: 1..512 experts");
    MLK_REQUIRE(K >= 1 && K <= kRoutePicks && K <= E, "routing: picks must be in 1..min(32, experts)");
    MLK_REQUIRE(T == 0 || logits, "routing: null pointer");
    return MLK_OK;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

int mlk_moe_routing(const void *logits, int x_kind, int score_fun, int n_tokens, int n_experts, int n_groups, int topk_groups, int topk, const float *bias,
                    int renormalize, float scaling, const uint8_t *token_mask, int32_t *ids, void *weights, void *stream) {
    const int rc = route_check(logits, x_kind, score_fun, n_tokens, n_experts, topk);
    if (rc != MLK_OK) return rc;
    MLK_REQUIRE(n_groups >= 1 && n_experts % n_groups == 0, "routing: n_groups must divide the expert count");
    MLK_REQUIRE(topk_groups >= 1 && topk_groups <= n_groups && topk <= n_experts / n_groups * topk_groups,
                "routing: topk_groups must be in 1..n_groups, and the kept groups hold as many experts as are picked");
    if (n_tokens == 0) return MLK_OK;
    MLK_REQUIRE(ids && weights, "routing: null pointer");
    RouteArgs a = {};
    a.logits = logits;
    a.bias = bias;
    a.mask = token_mask;
    a.T = n_tokens;
    a.E = n_experts;
    a.K = topk;
    a.G = n_groups;
    a.kept = topk_groups;
    a.score_fun = score_fun;
    a.renorm = renormalize != 0;
    a.scaling = scaling;
    a.ids = ids;
    a.weights = weights;
    return route_launch_all(a, x_kind, route_vec(logits, x_kind, n_experts), false, (hipStream_t)stream);
}

int mlk_moe_routing_grad(const void *logits, int x_kind, int score_fun, int n_tokens, int n_experts, int topk, int renormalize, float scaling, const int32_t *ids,
                         const void *dweights, void *dlogits, void *stream) {
    const int rc = route_check(logits, x_kind, score_fun, n_tokens, n_experts, topk);
    if (rc != MLK_OK) return rc;
    if (n_tokens == 0) return MLK_OK;
    MLK_REQUIRE(ids && dweights && dlogits, "routing: null pointer");
    RouteArgs a = {};
    a.logits = logits;
    a.T = n_tokens;
    a.E = n_experts;
    a.K = topk;
    a.score_fun = score_fun;
    a.renorm = renormalize != 0;
    a.scaling = scaling;
    a.ids = const_cast<int32_t *>(ids);
    a.dweights = dweights;
    a.dlogits = dlogits;
    return route_launch_all(a, x_kind, route_vec(logits, x_kind, n_experts) && route_vec(dlogits, x_kind, n_experts), true, (hipStream_t)stream);
}

}  // extern "C"
