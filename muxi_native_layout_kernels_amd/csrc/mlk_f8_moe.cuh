// Arguments of the expert layers in e4m3.
#pragma once

#include "mlk_f8.cuh"
#include "mlk_moe_args.cuh"

namespace mlk {

struct F8MoeArgs {
    const uint8_t *w1, *w2;      // of expert 0
    const float *s1, *s2;
    const uint8_t *X;            // [T][H] codes; as bf16 for f8_moe_gate_up_kernel
    const void *raw;             // [T][H] activations (one token)
    const float *xs;             // [H / 128][T]
    uint16_t *Y;                 // [T][H]
    const int32_t *ids;          // [T * K]
    const uint16_t *wts;         // [T * K]
    const int32_t *map;          // [id_limit] or null
    int id_limit, T, K, H, I, E, n_pairs, slots;
    const int32_t *sorted;
    const MoeTask *tasks;
    const int32_t *n_tasks;
    uint8_t *hbuf;               // [slot][I]
    float *hs;                   // [I / 128][slot]
    float *hraw;                 // [pick][I] (one token)
    f32x4 *hpart;                // [task][I / 128][row group][block of pairs][64]
    int32_t *counters;           // [task][I / 128]; of the panels the queues
    float *obuf;                 // [pair][slice][H]
    int slices;                  // of the down projection's k
};

// Local expert of a pair, -1: dropped.
__device__ __forceinline__ int f8_expert(const F8MoeArgs &p, int pair) {
    int e = p.ids[pair];
    if (e < 0 || e >= p.id_limit) return -1;
    if (p.map) e = p.map[e];
    return e >= 0 && e < p.E ? e : -1;
}

// The panels (mlk_f8_moe_panel.cuh): gate/up and down projection of tasks of up to kF8PanelBlocks blocks of 16 pairs.
constexpr int kF8PanelBlocks = 16;
template <class T>
int f8_launch_moe_panels(const F8MoeArgs &a, int max_tasks, hipStream_t s);

}  // namespace mlk
