// Internal interface of the E4M3 block-scaled operators: quantisers (k3_fp8_quantize.cu), products
// (k3_fp8_product.cu chooses between k3_fp8_few.cu and k3_fp8_wide.cu), and what is composed of
// them (k3_fp8_experts.cu).
#pragma once

#include "k3_common.cuh"
#include "k3_moe_fp8.h"

namespace k3::fp8 {

constexpr uint32_t kBlock = 128;

constexpr uint32_t pitch_of(uint32_t columns) { return (columns + 15u) & ~15u; }
constexpr uint32_t blocks_of(uint32_t n) { return (n + kBlock - 1u) / kBlock; }
constexpr uint32_t scale_pitch_of(uint32_t columns) { return (blocks_of(columns) + 3u) & ~3u; }

// every extent of an entry point: coordinates and row numbers stay well inside 32 bits
inline bool extent_ok(uint32_t n) { return n != 0u && n <= (1u << 30); }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

// Rows of x quantised and put where a dispatch wants them: row t goes to rows place[t * top_k + r] of
// codes and scales.  A route whose id is no expert (ids[...] >= experts) goes nowhere, and its place is
// set to `spare`; zero_row (zero_bytes, whole 16-byte units) is cleared on the way.
struct Placement {
    uint32_t *place;
    const uint32_t *ids;
    uint32_t top_k, experts, spare;
};
bool quantize_placed(void *codes, void *scales, const void *x_bf16, uint32_t rows, uint32_t columns,
                     const Placement &placement, void *zero_row, uint32_t zero_bytes, cudaStream_t stream);

enum Epilogue : int { kOutBf16 = 0, kOutF32 = 1, kOutActivated = 2 };

// out [rows, n] = a [rows, k] b^T.  With offsets (u32 [groups + 1] on the device) a's rows are grouped:
// rows [offsets[g], offsets[g + 1]) are multiplied by matrix g of b [groups, n, k].  kOutActivated: b is
// the gate, b2 the up matrix, and what is written is the activation, quantised by rows (out,
// out_scales).  Other grouped products write f32.
struct Product {
    void *out, *out_scales;
    const void *a, *a_scales;
    const void *b, *b_scales, *b2, *b2_scales;
    const uint32_t *offsets;
    const uint32_t *ids;             // token_gateup, token_down: the routes' matrices, u32 [top_k]
    const float *weights;            // token_down: f32 [top_k]
    const void *shared;              // token_down: bf16 [n] or null
    uint32_t top_k;
    uint32_t groups, rows, n, k;
    int b_scale_layout, epilogue, accumulate;
    int activation;
    float beta, linear_beta;
    // The launch in front writes neither b nor the offsets, and lets this one start only behind its own wait
    // for what is in front of it (a quantiser of rows, a product): b may be read before this one's wait.
    bool b_ready;
};
bool product(const Product &p, cudaStream_t stream);

// ---- the kernels behind it
// tiles of 128 rows of a
bool wide_product(const Product &p, cudaStream_t stream);
// tiles of 16 rows of one matrix or 64 of a group; b in 128 x 128 blocks
constexpr uint32_t grouped_few_rows = 40;    // per group on average
constexpr bool grouped_few(uint32_t rows, uint32_t groups) { return rows <= grouped_few_rows * groups; }
bool few_product(const Product &p, cudaStream_t stream);
// the same of up to 16 rows of a as bf16 (p.a and p.a_scales unused), quantised by rows on the way; out bf16
constexpr uint32_t few_linear_rows = 16;
bool few_linear(const Product &p, const void *x_bf16, cudaStream_t stream);
// one token's experts: a [1, k] times the gate and up matrices of each route -> activated rows [top_k, n]; and
// out bf16 [n] = sum over routes of weight * (a [top_k, k] row) times its down matrix, plus shared
bool token_gateup(const Product &p, cudaStream_t stream);
bool token_down(const Product &p, cudaStream_t stream);

// Parts that the depth of an item is cut into, a cluster of one block per part: the number with the shortest
// time for `items` items of `blocks` steps each, where a wave of as many clusters as fit takes the steps of
// a part (a multiple of `multiple`) and `fixed` steps more.
inline uint32_t best_parts(uint64_t items, uint32_t blocks, uint32_t multiple, uint32_t fixed, const ActiveClusters &active) {
    uint32_t best = 1u;
    uint64_t shortest = ~0ull;
    for (uint32_t s = 1u; s <= 8u; s++) {
        const uint32_t steps = ((blocks + s - 1u) / s + multiple - 1u) / multiple * multiple;
        if ((blocks + steps - 1u) / steps != s || active.of_size[s] == 0u) continue;      // rounding gives fewer parts, or none fit
        const uint64_t time = (items + active.of_size[s] - 1u) / active.of_size[s] * (steps + fixed);
        if (time < shortest) {
            shortest = time;
            best = s;
        }
    }
    return best;
}

}  // namespace k3::fp8
