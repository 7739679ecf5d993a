// Per-expert counts of a routing decision, and the balance loss of a router with its gradient.
//
// For sequences s with valid tokens V_s (not masked), n_s = |V_s| > 0, S' such sequences, K picks a token and E experts:
//   c[s,e] = pairs of V_s routed to e,   P[s,e] = sum over V_s of p[t,e],   g[s,e] = coef / S' * E / (K n_s^2) * c[s,e],   loss = sum g P
// with p = softmax(x) or sigmoid(x) / sum sigmoid(x); the counts are constants of the differentiation, so dloss/dp[t,e] = g[s(t),e] and
//   softmax  dx = p (g - sum p g),      sigmoid  dx = p (1 - sigmoid) (g - sum p g).
// A row of logits that are all -inf has p = 0.
//
// Forward: a workgroup takes a chunk of consecutive tokens and walks the sequences that it meets; 4 to 16 lanes hold a token, 4 to 16 experts each, so that
// a wave takes at least four tokens at a time and a sum over the experts is at most four exchanges within 16 lanes.  Its sums for (chunk c, sequence s)
// go to slot c + s: going through the tokens either the chunk or the sequence moves on, so no two share a slot.  A second launch adds the slots of a
// sequence in order, for 64 experts a workgroup; the last workgroup adds their shares of the loss.  No floating-point atomics: the results do not depend on
// the order in which workgroups run.
// Backward: the same walk, the logits are read again and their gradient written; a lane keeps the shares of its experts until the sequence changes.
// 32749 tokens x 256 experts in fp32, 9 sequences (33.5 MB: 4.9 us forward, 9.7 backward), sigmoid: 20.4 + 6.0 us forward, 20.0 backward (in a graph 22.3 and 17.5 in all, softmax
// 18.9 and 15.1); with 64 lanes of four experts a token and exchanges through LDS 22 and 33, without the next token's logits in flight 23 and 25, where this form took 19.4 and 18.4.
// Below about 16384 x 64 bf16 (4.6 + 7.4 and 4.7 us) it is the launches and the dependent loads at a chunk's start.
#include <algorithm>

#include "mlk_logits.cuh"

namespace mlk {

constexpr int kBalThreads = 256;
constexpr int kBalExperts = 256;
constexpr int kBalCounterBytes = 2048;      // in front: the loss's ticket, at 256 that of the counts, at 512 their totals
constexpr int kBalMost = 1 << 30;    // tokens and routed pairs: a step past the last one still is an int
constexpr int kBalManySeq = 64;      // sequences from which on a launch of its own counts their tokens

struct BalanceArgs {
    const void *logits;
    const int32_t *ids;
    const uint8_t *mask;         // null: every token counts
    const int32_t *cu;           // [S + 1] or null: one sequence
    int T, E, K, S, score_fun;
    int chunk, chunks;
    float coef;
    float *P;                    // [chunks + S][E]
    int32_t *cnt;                // [chunks + S][E]
    int32_t *valid;              // [chunks + S]
    int32_t *seq_valid;          // [S + 1]: valid tokens of each, and how many sequences have any (kBalManySeq and more only)
    float *part;                 // [S * expert blocks]
    int32_t *ticket;             // zero between calls
    float *loss, *share;         // [1], [S][E]
    int32_t *counts;             // [E]
    const float *grad;           // [1]
    void *dlogits;
};

// Experts of a lane: vector v holds 4 (v LPT + lane) .. + 3.
template <int LPT>
__device__ __forceinline__ int bal_expert(int v, int l) { return (v * LPT + l) * 4; }

// The logits of a token as they lie in memory; experts past the last one read the last again.  No branch: the next token's are in flight while one
// is computed.
template <class L, int NV, bool VEC>
struct BalRaw {
    typename L::V4 v[VEC ? NV : 1];
    typename L::V1 e[VEC ? 1 : NV][4];
};
template <class L, int LPT, int NV, bool VEC>
__device__ __forceinline__ void bal_load(const BalanceArgs &p, int t, int l, BalRaw<L, NV, VEC> &raw) {
    const typename L::V1 *row = reinterpret_cast<const typename L::V1 *>(p.logits) + (size_t)t * p.E;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int e0 = bal_expert<LPT>(v, l);
        if constexpr (VEC) {
            raw.v[v] = *reinterpret_cast<const typename L::V4 *>(row + min(e0, p.E - 4));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw.e[v][i] = row[min(e0 + i, p.E - 1)];
        }
    }
}
template <class L, int NV, bool VEC>
__device__ __forceinline__ void bal_unpack(const BalRaw<L, NV, VEC> &raw, float (&x)[NV][4]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if constexpr (VEC) {
            L::unpack(raw.v[v], x[v]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[v][i] = L::to_f32(raw.e[v][i]);
        }
    }
}

template <int LPT>
__device__ __forceinline__ float bal_sum(float v) { return bal_fold<LPT>(v, [](float a, float b) { return a + b; }); }
template <int LPT>
__device__ __forceinline__ float bal_max(float v) { return bal_fold<LPT>(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float bal_wave_sum(float v) {
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// Probabilities of one token (0 beyond the last expert); `rest`: 1 - sigmoid, 1 for softmax.  Sigmoids from e^-|x|, so that neither loses the bits of what is near 0.  Where all
// logits are below 0 only what the sigmoids are to each other matters, and e^(x - max) / (1 + e^x) says it also where they would underflow.
template <int LPT, int NV>
__device__ __forceinline__ void bal_probs(const BalanceArgs &p, int l, const float (&x)[NV][4], float (&pr)[NV][4], float (&rest)[NV][4]) {
    float sum = 0.f, m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (bal_expert<LPT>(v, l) + i < p.E) m = fmaxf(m, x[v][i]);
    m = bal_max<LPT>(m);
    if (m == -INFINITY) m = 0.f;
    if (p.score_fun != 0) m = fminf(m, 0.f);
    const float em = expf(m);                             // of sigmoids
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool is = bal_expert<LPT>(v, l) + i < p.E;
            rest[v][i] = 1.f;
            if (p.score_fun == 0) {
                pr[v][i] = is ? expf(x[v][i] - m) : 0.f;
            } else {
                const bool up = x[v][i] >= 0.f;           // then m = 0
                const float e = expf(-fabsf(x[v][i]) - m), r = 1.f / fmaf(e, em, 1.f), er = e * r;
                rest[v][i] = up ? er : r;
                pr[v][i] = is ? (up ? r : er) : 0.f;
            }
            sum += pr[v][i];
        }
    sum = bal_sum<LPT>(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[v][i] *= inv;
}

// First sequence that ends behind token t (S if there is none), for the whole wave: 64 ends at a time, one load for up to 64 sequences.
__device__ __forceinline__ int bal_first(const BalanceArgs &p, int t) {
    if (!p.cu) return 0;
    int lo = 0, n = p.S;                                  // lo ends are known to be no later than t, the next n may be
    while (n > 0) {
        const int step = (n + 63) / 64, at = lo + ((int)(threadIdx.x & 63) + 1) * step;
        const int ahead = __popcll(__ballot(at <= lo + n && p.cu[min(at, p.S)] <= t));
        lo += ahead * step;
        n = min(step - 1, p.S - lo);
    }
    return lo;
}
__device__ __forceinline__ void bal_range(const BalanceArgs &p, int s, int &a, int &b) {
    a = p.cu ? max(p.cu[s], 0) : 0;
    b = p.cu ? min(p.cu[s + 1], p.T) : p.T;
}

__device__ __forceinline__ bool bal_counts(const BalanceArgs &p, int t) { return !p.mask || p.mask[t]; }

template <class L, int LPT, int NV, bool VEC>
__global__ void __launch_bounds__(kBalThreads) balance_partial_kernel(BalanceArgs p) {
    constexpr int ROWS = kBalThreads / LPT, COLS = LPT * NV * 4;         // tokens at a time, experts with room for
    __shared__ float sums[ROWS * COLS];
    __shared__ int32_t cnt[kBalExperts];
    __shared__ int32_t valid;
    const int tid = threadIdx.x, row = tid / LPT, l = tid % LPT;
    const int c0 = blockIdx.x * p.chunk, c1 = min(c0 + p.chunk, p.T);
    if (blockIdx.x == 0)
        for (int e = tid; e <= p.E; e += kBalThreads) (e < p.E ? p.counts[e] : p.seq_valid[p.S]) = 0;        // later launches add to them
    for (int s = bal_first(p, c0); s < p.S; ++s) {
        int a, b;
        bal_range(p, s, a, b);
        if (a >= c1) break;
        a = max(a, c0);
        b = min(b, c1);
        if (a >= b) continue;
        BalRaw<L, NV, VEC> next;
        bal_load<L, LPT, NV, VEC>(p, min(a + row, b - 1), l, next);
        bool next_is = bal_counts(p, min(a + row, b - 1));
        for (int e = tid; e < p.E; e += kBalThreads) cnt[e] = 0;
        if (tid == 0) valid = 0;
        __syncthreads();
        for (int i = a * p.K + tid; i < b * p.K; i += kBalThreads) {
            const int e = p.ids[i];
            if (e >= 0 && e < p.E && (!p.mask || p.mask[i / p.K])) atomicAdd(&cnt[e], 1);
        }
        float sum[NV][4] = {};
        int n = 0;
        for (int t = a + row; t < b; t += ROWS) {
            float x[NV][4], pr[NV][4], rest[NV][4];
            bal_unpack<L, NV, VEC>(next, x);
            const bool is = next_is;
            bal_load<L, LPT, NV, VEC>(p, min(t + ROWS, b - 1), l, next);
            next_is = bal_counts(p, min(t + ROWS, b - 1));
            if (!is) continue;                              // the lanes of a token agree
            bal_probs<LPT, NV>(p, l, x, pr, rest);
            ++n;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[v][i] += pr[v][i];
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
            *reinterpret_cast<f32x4 *>(&sums[row * COLS + bal_expert<LPT>(v, l)]) = f32x4{sum[v][0], sum[v][1], sum[v][2], sum[v][3]};
        if (l == 0 && n) atomicAdd(&valid, n);
        __syncthreads();
        const size_t slot = (size_t)blockIdx.x + s;
        for (int e = tid; e < p.E; e += kBalThreads) {
            float v = 0.f;
            for (int r = 0; r < ROWS; ++r) v += sums[r * COLS + e];
            p.P[slot * p.E + e] = v;
            p.cnt[slot * p.E + e] = cnt[e];
        }
        if (tid == 0) p.valid[slot] = valid;
        __syncthreads();
    }
}

// Slots of sequence s: those of the chunks from c_first to c_last, none where it is empty.
__device__ __forceinline__ void bal_slots(const BalanceArgs &p, int s, int &first, int &n) {
    int a, b;
    bal_range(p, s, a, b);
    first = s + (a < b ? a / p.chunk : 0);
    n = a < b ? s + (b - 1) / p.chunk - first + 1 : 0;
}

// With many sequences their valid tokens are counted once, a thread per sequence: 20000 sequences of two tokens, 64 experts: 458 us forward, with every workgroup of the second launch counting all of them 815.
__global__ void __launch_bounds__(256) balance_valid_kernel(BalanceArgs p) {
    const int q = blockIdx.x * 256 + threadIdx.x;
    int first = 0, n = 0, v = 0;
    if (q < p.S) bal_slots(p, q, first, n);
    for (int i = 0; i < n; ++i) v += p.valid[first + i];
    if (q < p.S) p.seq_valid[q] = v;
    const int any = __popcll(__ballot(v > 0));
    if ((threadIdx.x & 63) == 0 && any) atomicAdd(&p.seq_valid[p.S], any);
}

// grid (blocks of 64 experts, sequences), 16 waves: wave w adds slots w, w + 16, ... of its 64 experts.
__global__ void __launch_bounds__(1024) balance_reduce_kernel(BalanceArgs p) {
    __shared__ float psum[16][64];
    __shared__ int32_t csum[16][64];
    __shared__ int32_t nonempty, mine;
    __shared__ int last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = blockIdx.y, e = blockIdx.x * 64 + lane;
    if (tid == 0) nonempty = mine = 0;
    __syncthreads();
    // how many sequences have a valid token: a wave per sequence
    if (p.S < kBalManySeq) {
        for (int q = wave; q < p.S; q += 16) {
            int first, n, v = 0;
            bal_slots(p, q, first, n);
            for (int i = lane; i < n; i += 64) v += p.valid[first + i];
            for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
            if (lane == 0 && v) atomicAdd(&nonempty, 1);
            if (lane == 0 && q == s) mine = v;
        }
    } else if (tid == 0) {
        nonempty = p.seq_valid[p.S];
        mine = p.seq_valid[s];
    }
    int first, n;
    bal_slots(p, s, first, n);
    float ps = 0.f;
    int32_t cs = 0;
    if (e < p.E) {
#pragma unroll 4
        for (int i = wave; i < n; i += 16) {
            ps += p.P[(size_t)(first + i) * p.E + e];
            cs += p.cnt[(size_t)(first + i) * p.E + e];
        }
    }
    psum[wave][lane] = ps;
    csum[wave][lane] = cs;
    __syncthreads();
    float share_of_loss = 0.f;
    if (wave == 0) {
        for (int w = 1; w < 16; ++w) {
            ps += psum[w][lane];
            cs += csum[w][lane];
        }
        const float nv = (float)mine;
        const float g = mine > 0 ? p.coef * ((float)p.E / ((float)p.K * (float)nonempty)) * ((float)cs / nv) / nv : 0.f;
        if (e < p.E) {
            p.share[(size_t)s * p.E + e] = g;
            if (cs) atomicAdd(&p.counts[e], cs);
            share_of_loss = g * ps;
        }
        share_of_loss = bal_wave_sum(share_of_loss);
        // agent-scope stores: the caches of the XCDs are not coherent for ordinary ones
        if (lane == 0) {
            __hip_atomic_store(&p.part[(size_t)s * gridDim.x + blockIdx.x], share_of_loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_s_waitcnt(0);
            const int total = gridDim.x * gridDim.y;
            const int before = __hip_atomic_fetch_add(p.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = before == total - 1;
            if (last) __hip_atomic_store(p.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    __syncthreads();
    if (!last) return;
    const int total = gridDim.x * gridDim.y;
    float v = 0.f;
    for (int i = tid; i < total; i += 1024) v += __hip_atomic_load(&p.part[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    v = bal_wave_sum(v);
    if (lane == 0) psum[wave][0] = v;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < 16; ++w) v += psum[w][0];
        *p.loss = v;
    }
}

template <class L, int LPT, int NV, bool VEC>
__global__ void __launch_bounds__(kBalThreads) balance_grad_kernel(BalanceArgs p) {
    constexpr int ROWS = kBalThreads / LPT;
    const int tid = threadIdx.x, row = tid / LPT, l = tid % LPT;
    const int c0 = blockIdx.x * p.chunk, c1 = min(c0 + p.chunk, p.T);
    BalRaw<L, NV, VEC> next;
    bal_load<L, LPT, NV, VEC>(p, min(c0 + row, c1 - 1), l, next);
    bool next_is = bal_counts(p, min(c0 + row, c1 - 1));
    const float up = *p.grad;
    // the sequence that this token lies in or ahead of, tokens a .. b - 1, and its shares
    int s = bal_first(p, c0), a = 0, b = 0;
    float g[NV][4] = {};
    auto enter = [&]() {
        if (s >= p.S) {
            a = b = p.T;
            return;
        }
        bal_range(p, s, a, b);
        const float *share = p.share + (size_t)s * p.E;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int e0 = bal_expert<LPT>(v, l);
            if constexpr (VEC) {
                BalF32::unpack(*reinterpret_cast<const f32x4 *>(share + min(e0, p.E - 4)), g[v]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) g[v][i] = share[min(e0 + i, p.E - 1)];
            }
        }
    };
    enter();
    for (int t = c0 + row; t < c1; t += ROWS) {
        float x[NV][4], d[NV][4] = {};
        bal_unpack<L, NV, VEC>(next, x);
        bool is = next_is;
        bal_load<L, LPT, NV, VEC>(p, min(t + ROWS, c1 - 1), l, next);
        next_is = bal_counts(p, min(t + ROWS, c1 - 1));
        if (t >= b && s < p.S) {
            do ++s;
            while (s < p.S && p.cu[s + 1] <= t);
            enter();
        }
        if (is && a <= t && t < b) {
            float pr[NV][4], rest[NV][4];
            bal_probs<LPT, NV>(p, l, x, pr, rest);
            float dot = 0.f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) dot = fmaf(pr[v][i], g[v][i], dot);
            dot = bal_sum<LPT>(dot);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) d[v][i] = pr[v][i] * rest[v][i] * (g[v][i] - dot) * up;
        }
        typename L::V1 *out = reinterpret_cast<typename L::V1 *>(p.dlogits) + (size_t)t * p.E;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int e0 = bal_expert<LPT>(v, l);
            if constexpr (VEC) {
                if (e0 < p.E) *reinterpret_cast<typename L::V4 *>(out + e0) = L::pack(d[v]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (e0 + i < p.E) out[e0 + i] = L::from_f32(d[v][i]);
            }
        }
    }
}

// How the sums of the workgroups get to counts: added to it (integer atomics: any order gives the same), stored by the only workgroup, or added to `total`, which is
// zero between calls, until the last workgroup stores that and clears it (30000 tokens, 6 picks: with a launch that clears counts ahead 10.9 us a call, so 7.0).
enum class CountsTo { kAdd, kStore, kTotal };
template <CountsTo TO>
__global__ void __launch_bounds__(256) expert_counts_kernel(const int32_t *__restrict__ ids, const uint8_t *__restrict__ mask, int64_t pairs, int K, int E,
                                                            int32_t *__restrict__ counts, int32_t *__restrict__ total, int32_t *__restrict__ ticket) {
    __shared__ int32_t cnt[kBalExperts];
    __shared__ int last;
    const int tid = threadIdx.x;
    for (int e = tid; e < E; e += 256) cnt[e] = 0;
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < pairs; i += (int64_t)gridDim.x * 256) {
        const int e = ids[i];
        if (e >= 0 && e < E && (!mask || mask[i / K])) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    int32_t *to = TO == CountsTo::kTotal ? total : counts;
    for (int e = tid; e < E; e += 256) {
        if constexpr (TO == CountsTo::kStore) to[e] = cnt[e];
        else if (cnt[e]) atomicAdd(&to[e], cnt[e]);
    }
    if constexpr (TO == CountsTo::kTotal) {
        // every wave waits for its own additions before the barrier and the arrival is counted behind it
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0) {
            last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
            if (last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last) return;
        for (int e = tid; e < E; e += 256) {
            counts[e] = __hip_atomic_load(&total[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(&total[e], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------- host
// Tokens of a chunk: enough for a workgroup of every CU, no fewer than a few passes of a workgroup.
static int balance_chunk(int T) {
    const int c = (T + 511) / 512;
    return c < 32 ? 32 : (c + 31) / 32 * 32;
}

struct BalanceScratch {
    int32_t *ticket, *cnt, *valid, *seq_valid;
    float *P, *part;
};
static size_t balance_carve(uint8_t *base, int T, int E, int S, BalanceScratch *out) {
    const int chunk = balance_chunk(T);
    const size_t slots = (size_t)(T + chunk - 1) / chunk + S;
    size_t off = kBalCounterBytes;
    auto take = [&](size_t bytes) {
        uint8_t *ptr = base ? base + off : nullptr;
        off = (off + bytes + 255) / 256 * 256;
        return ptr;
    };
    BalanceScratch b;
    b.ticket = (int32_t *)base;
    b.P = (float *)take(slots * E * 4);
    b.cnt = (int32_t *)take(slots * E * 4);
    b.valid = (int32_t *)take(slots * 4);
    b.seq_valid = (int32_t *)take(((size_t)S + 1) * 4);
    b.part = (float *)take((size_t)S * ((E + 63) / 64) * 4);
    if (out) *out = b;
    return off;
}

static int balance_check(const void *logits, int x_kind, int score_fun, int T, int E, const int32_t *cu, int n_seq) {
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16 || x_kind == MLK_F32, "balance: logits must be fp16, bf16 or fp32");
    MLK_REQUIRE(score_fun == 0 || score_fun == 1, "balance: score function must be 0 (softmax) or 1 (sigmoid)");
    MLK_REQUIRE(T >= 0 && T <= kBalMost, "balance: 0..2^30 tokens");
    MLK_REQUIRE(E >= 1 && E <= kBalExperts, "balance: 1..256 experts");
    MLK_REQUIRE(cu ? n_seq >= 0 && n_seq <= 65535 : n_seq == 1, "balance: 0..65535 sequences, one without cu_seqlens");
    MLK_REQUIRE(T == 0 || logits, "balance: null pointer");
    return MLK_OK;
}

// Rows of four experts can be moved whole.
static bool balance_vec(const void *p, int x_kind, int E) { return E % 4 == 0 && ((uintptr_t)p & (x_kind == MLK_F32 ? 15 : 7)) == 0; }

template <class L, bool VEC>
static void balance_launch(const BalanceArgs &a, bool grad, hipStream_t s) {
#define MLK_BAL(LPT, NV)                                                                       \
    do {                                                                                       \
        if (grad) balance_grad_kernel<L, LPT, NV, VEC><<<a.chunks, kBalThreads, 0, s>>>(a);    \
        else balance_partial_kernel<L, LPT, NV, VEC><<<a.chunks, kBalThreads, 0, s>>>(a);      \
    } while (0)
    if (a.E <= 16) MLK_BAL(4, 1);
    else if (a.E <= 32) MLK_BAL(8, 1);
    else if (a.E <= 64) MLK_BAL(16, 1);
    else if (a.E <= 128) MLK_BAL(16, 2);
    else MLK_BAL(16, 4);
#undef MLK_BAL
}
template <class L>
static void balance_launch_vec(const BalanceArgs &a, bool vec, bool grad, hipStream_t s) {
    if (vec) balance_launch<L, true>(a, grad, s);
    else balance_launch<L, false>(a, grad, s);
}
static void balance_launch_kind(const BalanceArgs &a, int x_kind, bool vec, bool grad, hipStream_t s) {
    if (x_kind == MLK_F32) balance_launch_vec<BalF32>(a, vec, grad, s);
    else if (x_kind == MLK_F16) balance_launch_vec<Bal16<F16>>(a, vec, grad, s);
    else balance_launch_vec<Bal16<BF16>>(a, vec, grad, s);
}

__global__ void balance_nothing_kernel(float *loss, int32_t *counts, int E) {
    if (threadIdx.x == 0) *loss = 0.f;
    for (int e = threadIdx.x; e < E; e += 256) counts[e] = 0;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

int mlk_expert_counts(const int32_t *topk_ids, const uint8_t *token_mask, int n_tokens, int topk, int n_experts, int accumulate, int32_t *counts,
                      void *workspace, void *stream) {
    MLK_REQUIRE(n_tokens >= 0 && topk >= 1, "expert_counts: negative token count, or no picks");
    MLK_REQUIRE(n_experts >= 1 && n_experts <= kBalExperts, "expert_counts: 1..256 experts");
    MLK_REQUIRE(counts && (n_tokens == 0 || topk_ids), "expert_counts: null pointer");
    hipStream_t s = (hipStream_t)stream;
    // one workgroup up to 4096 pairs: it has no others to wait for, and takes 3 us for them
    const int64_t pairs = (int64_t)n_tokens * topk;
    const int wgs = pairs <= 4096 ? 1 : (int)std::min<int64_t>((pairs + 1023) / 1024, 256);
    if (pairs == 0 && accumulate) return MLK_OK;
    if (accumulate) {
        expert_counts_kernel<CountsTo::kAdd><<<wgs, 256, 0, s>>>(topk_ids, token_mask, pairs, topk, n_experts, counts, nullptr, nullptr);
    } else if (wgs == 1) {
        expert_counts_kernel<CountsTo::kStore><<<1, 256, 0, s>>>(topk_ids, token_mask, pairs, topk, n_experts, counts, nullptr, nullptr);
    } else {
        MLK_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, "expert_counts: more than 4096 pairs need a workspace, on 16 bytes");
        int32_t *w = (int32_t *)workspace;
        expert_counts_kernel<CountsTo::kTotal><<<wgs, 256, 0, s>>>(topk_ids, token_mask, pairs, topk, n_experts, counts, w + 128, w + 64);
    }
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

size_t mlk_balance_workspace_bytes(int n_tokens, int n_experts, int n_seq) {
    if (n_tokens < 0 || n_tokens > kBalMost || n_experts < 1 || n_experts > kBalExperts || n_seq < 0 || n_seq > 65535) return 0;
    return balance_carve(nullptr, n_tokens, n_experts, n_seq, nullptr);
}
size_t mlk_balance_counter_bytes(void) { return kBalCounterBytes; }

int mlk_balance_loss(const void *logits, int x_kind, int score_fun, int n_tokens, int n_experts, int topk, const int32_t *topk_ids,
                     const uint8_t *token_mask, const int32_t *cu_seqlens, int n_seq, float coef, float *loss, int32_t *counts, float *share,
                     void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = balance_check(logits, x_kind, score_fun, n_tokens, n_experts, cu_seqlens, n_seq);
    if (rc != MLK_OK) return rc;
    MLK_REQUIRE(topk >= 1 && (int64_t)n_tokens * topk <= kBalMost, "balance: at least one pick, at most 2^30 routed pairs");
    MLK_REQUIRE(loss && counts && (n_seq == 0 || share), "balance: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (n_tokens == 0 || n_seq == 0) {
        balance_nothing_kernel<<<1, 256, 0, s>>>(loss, counts, n_experts);
        MLK_LAUNCH_CHECK();
        return MLK_OK;
    }
    MLK_REQUIRE(topk_ids && workspace && ((uintptr_t)workspace & 15) == 0, "balance: null pointer, or workspace off 16 bytes");
    if (workspace_bytes < mlk_balance_workspace_bytes(n_tokens, n_experts, n_seq)) return fail(MLK_ERR_WORKSPACE, "balance: workspace too small");
    BalanceArgs a = {};
    BalanceScratch w;
    balance_carve((uint8_t *)workspace, n_tokens, n_experts, n_seq, &w);
    a.logits = logits;
    a.ids = topk_ids;
    a.mask = token_mask;
    a.cu = cu_seqlens;
    a.T = n_tokens;
    a.E = n_experts;
    a.K = topk;
    a.S = n_seq;
    a.score_fun = score_fun;
    a.chunk = balance_chunk(n_tokens);
    a.chunks = (n_tokens + a.chunk - 1) / a.chunk;
    a.coef = coef;
    a.P = w.P;
    a.cnt = w.cnt;
    a.valid = w.valid;
    a.seq_valid = w.seq_valid;
    a.part = w.part;
    a.ticket = w.ticket;
    a.loss = loss;
    a.share = share;
    a.counts = counts;
    balance_launch_kind(a, x_kind, balance_vec(logits, x_kind, n_experts), false, s);
    MLK_LAUNCH_CHECK();
    if (n_seq >= kBalManySeq) {
        balance_valid_kernel<<<(n_seq + 255) / 256, 256, 0, s>>>(a);
        MLK_LAUNCH_CHECK();
    }
    balance_reduce_kernel<<<dim3((n_experts + 63) / 64, n_seq), 1024, 0, s>>>(a);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

int mlk_balance_loss_grad(const void *logits, int x_kind, int score_fun, int n_tokens, int n_experts, const uint8_t *token_mask,
                          const int32_t *cu_seqlens, int n_seq, const float *share, const float *grad, void *dlogits, void *stream) {
    const int rc = balance_check(logits, x_kind, score_fun, n_tokens, n_experts, cu_seqlens, n_seq);
    if (rc != MLK_OK) return rc;
    if (n_tokens == 0) return MLK_OK;
    MLK_REQUIRE((n_seq == 0 || share) && grad && dlogits, "balance: null pointer");
    BalanceArgs a = {};
    a.logits = logits;
    a.mask = token_mask;
    a.cu = cu_seqlens;
    a.T = n_tokens;
    a.E = n_experts;
    a.S = n_seq;
    a.score_fun = score_fun;
    const bool vec = balance_vec(logits, x_kind, n_experts) && balance_vec(dlogits, x_kind, n_experts) && ((uintptr_t)share & 15) == 0;
    a.chunk = balance_chunk(n_tokens);
    a.chunks = (n_tokens + a.chunk - 1) / a.chunk;
    a.share = const_cast<float *>(share);
    a.grad = grad;
    a.dlogits = dlogits;
    balance_launch_kind(a, x_kind, vec, true, (hipStream_t)stream);
    MLK_LAUNCH_CHECK();
    return MLK_OK;
}

}  // extern "C"
