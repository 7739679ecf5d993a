// Expert layers over 4-bit weights: arguments, workspace, passes.
#include <algorithm>
#include <initializer_list>

#include "mlk_w4_moe_panel.cuh"

namespace mlk {

#define MLK_W4_EXTERN(T, GS)                                                                              \
    extern template int w4_launch_moe<T, GS, false>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);   \
    extern template int w4_launch_moe<T, GS, true>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);    \
    extern template int w4_launch_moe_panel<T, GS, false>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);   \
    extern template int w4_launch_moe_panel<T, GS, true>(const W4MoeArgs &, const W4MoePlan &, hipStream_t);
MLK_W4_EXTERN(F16, 4)
MLK_W4_EXTERN(F16, 2)
MLK_W4_EXTERN(F16, 1)
MLK_W4_EXTERN(BF16, 4)
MLK_W4_EXTERN(BF16, 2)
MLK_W4_EXTERN(BF16, 1)
#undef MLK_W4_EXTERN

int launch_moe_align(const int32_t *topk_ids, int n_pairs, int E, const int32_t *experts_map, int id_limit, int32_t *sorted, int32_t *cumsum,
                     int32_t *padded, int32_t *experts_ids, MoeTask *tasks, int32_t *n_tasks, int cb_max, hipStream_t s);

constexpr int kW4MoePairs = 16384;      // routed pairs of a pass: bounds the scratch of long prompts

static int w4_moe_pass_tokens(int n_tokens, int topk) { return n_tokens < kW4MoePairs / topk ? n_tokens : kW4MoePairs / topk; }

static W4MoePlan w4_moe_plan(int tokens, int E, int n_router, int topk, int hidden, int inter) {
    W4MoePlan pl = {};
    pl.slices = 1;
    const int cus = device_cus(), pairs = tokens * topk;
    if (tokens == 1 && hidden <= 64 * 1024) {                // the token is staged in LDS
        pl.tt = 0;
        pl.max_tasks = topk;
        return pl;
    }
    // Routed pairs of an expert that is reached.  Up to 8 on average a block of 16 tokens is a task, above up to two blocks, and with many panels (us with one, two, panels):
    //   8 experts of 4096 x 14336, top-2      at 32 tokens (8) 141, 143, 234; at 36 (9) 178, 154, 240; at 100 (25) 309, 220, 245; at 160 (40) 442, 265, 252; at 300 (75) two 440, 328
    //   256 of 7168 x 2048, top-8             at 400 (12) 1453, 1164, 1753; at 1000 (31) 2689, 1880, 2098; at 2000 (62) two 3177, 2817
    //   128 of 2048 x 768, top-8              at 130 (8) 97, 100, 164; at 160 (10) 109, 107, 181; at 800 (50) 257, 224, 268; at 1300 (81) two 325, 330; at 2000 (125) 468, 437
    //   64 of 2048 x 1408, top-6              at 100 (9) 84, 82, 126; at 500 (46) 205, 157, 176; at 1000 (93) two 263, 257
    // With E of the router's experts here that share of the pairs is expected here.
    const int here = (int)std::max<int64_t>(1, std::min<int64_t>(pairs, (int64_t)pairs * E / n_router));
    const int reached = std::min(here, E), load = (here + reached - 1) / reached;
    pl.panels = load > ((int64_t)hidden * inter <= (1 << 23) ? 80 : 40) && (int64_t)tokens * hidden < (1ll << 31);
    pl.tt = pl.panels ? 8 : (load > 8 ? 2 : 1);
    // an expert's last task may be short: at most one more than its blocks fill
    const int64_t most = (int64_t)E + pairs / (16 * pl.tt);
    pl.max_tasks = (int)(most < pairs ? most : pairs);
    if (!pl.panels) {
        pl.few = pl.tt == 1 && pairs <= 64;
        return pl;
    }
    // Two K slices of a long down projection that would leave CUs without a panel in its last round: 8 experts of 4096 x 14336 at 100 tokens 276 -> 240 us, at
    // 320 389 -> 343, at 1000 853 -> 811; with 16 windows (2048) or panels for two rounds the second sum costs more (64 experts at 300 tokens 144 -> 161).
    const int wgs = (hidden + 255) / 256 * reached * ((load + 16 * pl.tt - 1) / (16 * pl.tt));
    if (wgs < 2 * cus && inter / 128 >= 64) pl.slices = 2;
    return pl;
}

struct W4MoeWorkspace {
    MoeTask *tasks;
    int32_t *n_tasks, *sorted, *cumsum, *padded, *experts_ids;
    uint16_t *hbuf;
    float *obuf;
    u32x4 *sums1, *sums2;
};

static size_t w4_moe_carve(uint8_t *base, const W4MoePlan &pl, int tokens, int E, int topk, int hidden, int inter, int group, W4MoeWorkspace *ws) {
    const int64_t pairs = (int64_t)tokens * topk, padded = pairs + E * 15, blocks = (padded + 15) / 16;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        uint8_t *ptr = base ? base + off : nullptr;
        off = (off + bytes + 255) / 256 * 256;
        return ptr;
    };
    W4MoeWorkspace w;
    w.tasks = (MoeTask *)take(sizeof(MoeTask) * (size_t)(blocks + 1));
    w.n_tasks = (int32_t *)take(sizeof(int32_t));
    w.sorted = (int32_t *)take(sizeof(int32_t) * (size_t)(blocks * 16));
    w.cumsum = (int32_t *)take(sizeof(int32_t) * (size_t)(E + 1));
    w.padded = (int32_t *)take(sizeof(int32_t));
    w.experts_ids = (int32_t *)take(sizeof(int32_t) * (size_t)blocks);
    w.hbuf = (uint16_t *)take((size_t)blocks * 16 * inter * 2);
    w.obuf = (float *)take((size_t)pairs * pl.slices * hidden * 4);
    const int gs = group < 128 ? group / 32 : 4;
    w.sums1 = (u32x4 *)take(pl.panels ? (size_t)tokens * w4_sum_pitch(hidden, gs) * 16 : 0);
    w.sums2 = (u32x4 *)take(pl.panels ? (size_t)blocks * 16 * w4_sum_pitch(inter, gs) * 16 : 0);
    if (ws) *ws = w;
    return off;
}

}  // namespace mlk

using namespace mlk;

extern "C" {

// What a call needs: a long one goes in passes of one size and a shorter last one, whose plan may differ.
size_t mlk_experts_w4_workspace_bytes(int n_tokens, int n_experts, int n_router_experts, int topk, int hidden, int inter, int group) {
    if (n_tokens <= 0 || n_experts <= 0 || n_experts > 256 || n_router_experts <= 0 || topk <= 0 || topk > 32 || hidden <= 0 || inter <= 0 || group < 32) return 0;
    const int step = w4_moe_pass_tokens(n_tokens, topk), rest = n_tokens % step;
    size_t most = 0;
    for (int t : {step, rest}) {
        if (t == 0) continue;
        const size_t need = w4_moe_carve(nullptr, w4_moe_plan(t, n_experts, n_router_experts, topk, hidden, inter), t, n_experts, topk, hidden, inter, group, nullptr);
        if (need > most) most = need;
    }
    return most;
}

int mlk_fused_experts_w4(const void *w1, const void *w1_scale, const void *w1_zero, const void *w2, const void *w2_scale, const void *w2_zero,
                         const void *x, int n_tokens, int n_experts, int n_router_experts, int topk, int hidden, int inter, int group, int x_kind,
                         const int32_t *topk_ids, const void *topk_weights, const int32_t *experts_map, void *y, void *workspace,
                         size_t workspace_bytes, void *stream) {
    MLK_REQUIRE(x_kind == MLK_F16 || x_kind == MLK_BF16, "experts w4: activations must be fp16 or bf16");
    MLK_REQUIRE(n_tokens >= 0, "experts w4: negative token count");
    MLK_REQUIRE(n_experts >= 1 && n_experts <= 256, "experts w4: 1..256 experts");
    MLK_REQUIRE(n_router_experts >= 1 && (experts_map || n_router_experts == n_experts), "experts w4: fewer experts than the router's need an experts_map");
    MLK_REQUIRE(topk >= 1 && topk <= 32, "experts w4: topk must be in 1..32");
    MLK_REQUIRE(hidden > 0 && inter > 0 && hidden % 128 == 0 && inter % 128 == 0, "experts w4: hidden and intermediate sizes must be multiples of 128");
    MLK_REQUIRE(hidden < (1 << 23) && inter < (1 << 23), "experts w4: hidden and intermediate sizes must be below 2^23");
    MLK_REQUIRE(group == 32 || group == 64 || (group >= 128 && group % 128 == 0 && hidden % group == 0 && inter % group == 0),
                "experts w4: the group must be 32, 64 or a multiple of 128 that divides both sizes");
    MLK_REQUIRE((w1_zero == nullptr) == (w2_zero == nullptr), "experts w4: zero points for both matrices or for none");
    if (n_tokens == 0) return MLK_OK;
    MLK_REQUIRE(w1 && w1_scale && w2 && w2_scale && x && topk_ids && topk_weights && y && workspace, "experts w4: null pointer");
    MLK_REQUIRE(aligned16(w1) && aligned16(w2) && aligned16(x) && aligned16(y) && aligned16(workspace),
                "experts w4: weights, activations, outputs and workspace must lie on 16 bytes");
    MLK_REQUIRE((((uintptr_t)w1_scale | (uintptr_t)w2_scale) & 7) == 0 && (((uintptr_t)w1_zero | (uintptr_t)w2_zero) & 3) == 0,
                "experts w4: scales must lie on 8 bytes, zero points on 4");
    if (workspace_bytes < mlk_experts_w4_workspace_bytes(n_tokens, n_experts, n_router_experts, topk, hidden, inter, group))
        return fail(MLK_ERR_WORKSPACE, "experts w4: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    W4MoeArgs a;
    a.w1 = W4Matrix{(const uint8_t *)w1, (const uint16_t *)w1_scale, (const uint8_t *)w1_zero};
    a.w2 = W4Matrix{(const uint8_t *)w2, (const uint16_t *)w2_scale, (const uint8_t *)w2_zero};
    a.map = experts_map;
    a.id_limit = n_router_experts;
    a.K = topk;
    a.H = hidden;
    a.I = inter;
    a.E = n_experts;
    const int wide = group > 128 ? group : 128;
    a.blocks1 = hidden / wide;
    a.blocks2 = inter / wide;
    a.inv = w4_inverse(wide / 128);
    const int step = w4_moe_pass_tokens(n_tokens, topk);
    for (int t0 = 0; t0 < n_tokens; t0 += step) {
        a.T = n_tokens - t0 < step ? n_tokens - t0 : step;
        a.n_pairs = a.T * topk;
        a.X = (const uint16_t *)x + (size_t)t0 * hidden;
        a.Y = (uint16_t *)y + (size_t)t0 * hidden;
        a.ids = topk_ids + (size_t)t0 * topk;
        a.wts = (const uint16_t *)topk_weights + (size_t)t0 * topk;
        const W4MoePlan pl = w4_moe_plan(a.T, n_experts, n_router_experts, topk, hidden, inter);
        W4MoeWorkspace ws;
        w4_moe_carve((uint8_t *)workspace, pl, a.T, n_experts, topk, hidden, inter, group, &ws);
        a.sorted = ws.sorted;
        a.tasks = ws.tasks;
        a.n_tasks = ws.n_tasks;
        a.hbuf = ws.hbuf;
        a.obuf = ws.obuf;
        a.slices = pl.slices;
        a.sums1 = ws.sums1;
        a.sums2 = ws.sums2;
        int rc = MLK_OK;
        if (pl.tt && !pl.few) {
            rc = launch_moe_align(a.ids, a.n_pairs, n_experts, experts_map, a.id_limit, ws.sorted, ws.cumsum, ws.padded, ws.experts_ids, ws.tasks,
                                  ws.n_tasks, pl.tt, s);
            if (rc != MLK_OK) return rc;
        }
        const bool zp = w1_zero != nullptr, f16 = x_kind == MLK_F16;
#define MLK_W4_GO(T, GS)                                                                                                                     \
    do {                                                                                                                                         \
        if (pl.panels)                                                                                                                           \
            rc = zp ? w4_launch_moe_panel<T, GS, true>(a, pl, s) : w4_launch_moe_panel<T, GS, false>(a, pl, s);                                  \
        else                                                                                                                                     \
            rc = zp ? w4_launch_moe<T, GS, true>(a, pl, s) : w4_launch_moe<T, GS, false>(a, pl, s);                                              \
    } while (0)
        if (group == 32) {
            if (f16) MLK_W4_GO(F16, 1);
            else MLK_W4_GO(BF16, 1);
        } else if (group == 64) {
            if (f16) MLK_W4_GO(F16, 2);
            else MLK_W4_GO(BF16, 2);
        } else {
            if (f16) MLK_W4_GO(F16, 4);
            else MLK_W4_GO(BF16, 4);
        }
#undef MLK_W4_GO
        if (rc != MLK_OK) return rc;
    }
    return MLK_OK;
}

}  // extern "C"
