// What is composed of the E4M3 quantisers and products: a linear layer, its weight's gradient, and the
// routed experts (dispatch, rows quantised into place, gate/up with the activation, down, combine).
#include "k3_common.cuh"
#include "k3_fp8.h"
#include "k3_moe_layer.h"
#include "k3_moe_ops.h"

using namespace k3;
using namespace k3::fp8;

namespace {

// out[t] = bf16(sum_r weights[t, r] * rows[index[t, r]]), and bf16(that + shared[t]) with shared, of f32 rows: what
// k3_moe_combine does of bf16 ones.  Rows rounded to bf16 would add an error as large as that of the output's own
// rounding (2.4e-3 of the norm instead of 1.7e-3), so they are f32 for any number of tokens, and a token's precision
// does not depend on how many share its call.  4096 tokens, 16 of 64 experts of 7168 x 2048: 4.18 ms, with bf16 rows,
// 0.94 GB less each way, 3.85.
__global__ void __launch_bounds__(128)
combine_f32_kernel(uint16_t *out, const float *rows, const uint32_t *index, const float *weights, const uint16_t *shared,
                   uint32_t top_k, uint32_t hidden) {
    __shared__ float weights_s[32];
    __shared__ uint32_t index_s[32];
    pdl_wait();
    const uint32_t token = blockIdx.x, c = (blockIdx.y * 128u + threadIdx.x) * 4u;
    if (threadIdx.x < top_k) {
        weights_s[threadIdx.x] = weights[(uint64_t)token * top_k + threadIdx.x];
        index_s[threadIdx.x] = index[(uint64_t)token * top_k + threadIdx.x];
    }
    __syncthreads();
    if (c >= hidden) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (uint32_t r = 0; r < top_k; r++) {
        const float4 v = *reinterpret_cast<const float4 *>(rows + (uint64_t)index_s[r] * hidden + c);
        const float w = weights_s[r];
        sum[0] = fmaf(w, v.x, sum[0]);
        sum[1] = fmaf(w, v.y, sum[1]);
        sum[2] = fmaf(w, v.z, sum[2]);
        sum[3] = fmaf(w, v.w, sum[3]);
    }
    const uint64_t at = (uint64_t)token * hidden + c;
    uint32_t h[4];
#pragma unroll
    for (uint32_t j = 0; j < 4u; j++) {
        h[j] = float_to_bf16_bits(sum[j]);
        if (shared) h[j] = float_to_bf16_bits(bf16_bits_to_float(h[j]) + bf16_bits_to_float(shared[at + j]));
    }
    *reinterpret_cast<uint2 *>(out + at) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Pieces of a caller's workspace, each on 256 bytes; with base null only the total is counted.
struct Carve {
    char *base;
    size_t total = 0;
    void *take(uint64_t bytes) {
        void *p = base ? base + total : nullptr;
        total += (size_t)((bytes + 255u) / 256u * 256u);
        return p;
    }
};

struct Rows {                        // codes with scales per row
    void *codes, *scales;
    Rows(Carve &c, uint64_t rows, uint32_t columns)
        : codes(c.take(rows * pitch_of(columns))), scales(c.take(rows * scale_pitch_of(columns) * sizeof(float))) {}
};

struct ExpertsWorkspace {
    Carve carve;
    uint32_t *offsets, *sorted_route, *sorted_token, *inv_perm;
    size_t dispatch_bytes;
    void *dispatch;
    Rows x, act;
    float *rows_out;                 // one row more than there are routes: the spare one
    ExpertsWorkspace(const k3_moe_fp8_experts_desc *d, uint32_t tokens, void *base)
        : carve{(char *)base},
          offsets((uint32_t *)carve.take((d->experts + 1u) * sizeof(uint32_t))),
          sorted_route((uint32_t *)carve.take((uint64_t)tokens * d->top_k * sizeof(uint32_t))),
          sorted_token((uint32_t *)carve.take((uint64_t)tokens * d->top_k * sizeof(uint32_t))),
          inv_perm((uint32_t *)carve.take((uint64_t)tokens * d->top_k * sizeof(uint32_t))),
          dispatch_bytes(k3_moe_dispatch_workspace_bytes(tokens, d->top_k, d->experts)),
          dispatch(carve.take(dispatch_bytes)),
          x(carve, (uint64_t)tokens * d->top_k, d->hidden),
          act(carve, (uint64_t)tokens * d->top_k, d->expert_hidden),
          rows_out((float *)carve.take(((uint64_t)tokens * d->top_k + 1u) * d->hidden * sizeof(float))) {}
};

bool experts_ok(const k3_moe_fp8_experts_desc *d, uint32_t tokens) {
    return d && extent_ok(d->hidden) && d->hidden % 16u == 0 && extent_ok(d->expert_hidden) && d->expert_hidden % 16u == 0 &&
           d->experts != 0u && d->experts <= 1024u && d->top_k != 0u && d->top_k <= 32u && d->top_k <= d->experts &&
           (d->activation == K3_MOE_ACT_SITU || d->activation == K3_MOE_ACT_SWIGLU) &&
           (d->activation != K3_MOE_ACT_SITU || (d->beta > 0.0f && d->linear_beta > 0.0f)) &&
           (uint64_t)d->experts * d->hidden <= (1u << 30) && (uint64_t)d->experts * d->expert_hidden <= (1u << 30) &&
           tokens != 0u && (uint64_t)tokens * d->top_k <= (1u << 30);
}

bool table_ok(const void *codes, const void *scales) { return codes && scales && aligned16(codes) && ((uintptr_t)scales & 3u) == 0u; }

}  // namespace

extern "C" size_t k3_moe_fp8_linear_workspace_bytes(uint32_t tokens, uint32_t columns) {
    if (!extent_ok(tokens) || !extent_ok(columns)) return 0;
    Carve c{nullptr};
    Rows x(c, tokens, columns);
    return c.total;
}

extern "C" bool k3_moe_fp8_linear(void *out, const void *x, const void *w, const void *w_scales, uint32_t tokens, uint32_t rows,
                                  uint32_t columns, void *workspace, size_t workspace_bytes, void *stream) {
    if (!out || !x || !table_ok(w, w_scales) || !extent_ok(tokens) || !extent_ok(rows) || !extent_ok(columns) || !workspace ||
        !aligned16(workspace) || (((uintptr_t)out | (uintptr_t)x) & 1u) != 0u) {
        return false;
    }
    Carve c{(char *)workspace};
    const Rows q(c, tokens, columns);
    if (workspace_bytes < c.total) return false;
    Product p{};
    p.out = out;
    p.a = q.codes;
    p.a_scales = q.scales;
    p.b = w;
    p.b_scales = w_scales;
    p.groups = 1u;
    p.rows = tokens;
    p.n = rows;
    p.k = columns;
    p.b_scale_layout = K3_MOE_FP8_BLOCKS;
    p.epilogue = kOutBf16;
    p.b_ready = true;
    if (tokens <= few_linear_rows) return few_linear(p, x, (cudaStream_t)stream);
    return k3_moe_fp8_quantize_rows(q.codes, q.scales, x, tokens, columns, K3_MOE_FP8_BF16, stream) &&
           product(p, (cudaStream_t)stream);
}

extern "C" size_t k3_moe_fp8_weight_gradient_workspace_bytes(uint32_t tokens, uint32_t rows, uint32_t columns) {
    if (!extent_ok(tokens) || !extent_ok(rows) || !extent_ok(columns)) return 0;
    Carve c{nullptr};
    Rows dy(c, rows, tokens), x(c, columns, tokens);
    return c.total;
}

extern "C" bool k3_moe_fp8_weight_gradient(void *dw, const void *dy, const void *x, uint32_t tokens, uint32_t rows,
                                           uint32_t columns, int accumulate, void *workspace, size_t workspace_bytes,
                                           void *stream) {
    if (!dw || !dy || !x || !extent_ok(tokens) || !extent_ok(rows) || !extent_ok(columns) || !workspace ||
        !aligned16(workspace) || ((uintptr_t)dw & 3u) != 0u || (((uintptr_t)dy | (uintptr_t)x) & 1u) != 0u) {
        return false;
    }
    Carve c{(char *)workspace};
    const Rows dyq(c, rows, tokens), xq(c, columns, tokens);
    if (workspace_bytes < c.total) return false;
    return k3_moe_fp8_quantize_columns(dyq.codes, dyq.scales, dy, tokens, rows, K3_MOE_FP8_BF16, stream) &&
           k3_moe_fp8_quantize_columns(xq.codes, xq.scales, x, tokens, columns, K3_MOE_FP8_BF16, stream) &&
           k3_moe_fp8_product(dw, dyq.codes, dyq.scales, xq.codes, xq.scales, rows, columns, tokens, K3_MOE_FP8_ROWS,
                              K3_MOE_FP8_F32, accumulate, stream);
}

extern "C" size_t k3_moe_fp8_experts_workspace_bytes(const k3_moe_fp8_experts_desc *d, uint32_t tokens) {
    if (!experts_ok(d, tokens)) return 0;
    return ExpertsWorkspace(d, tokens, nullptr).carve.total;
}

extern "C" bool k3_moe_fp8_experts_forward(const k3_moe_fp8_experts_desc *d, void *out, const void *x, const void *ids,
                                           const void *weights, const void *shared, uint32_t tokens, void *workspace,
                                           size_t workspace_bytes, void *stream_pointer) {
    if (!experts_ok(d, tokens) || !out || !x || !ids || !weights || !workspace || !aligned16(workspace) ||
        !table_ok(d->w1, d->w1_scales) || !table_ok(d->w3, d->w3_scales) || !table_ok(d->w2, d->w2_scales) ||
        (((uintptr_t)out | (uintptr_t)shared) & 15u) != 0u || ((uintptr_t)x & 1u) != 0u ||
        (((uintptr_t)ids | (uintptr_t)weights) & 3u) != 0u) {
        return false;
    }
    const ExpertsWorkspace w(d, tokens, workspace);
    if (workspace_bytes < w.carve.total) return false;
    cudaStream_t stream = (cudaStream_t)stream_pointer;
    const uint32_t routes = tokens * d->top_k;
    // One token: its routes are the groups as they come, and the down product forms their weighted sum.  Three
    // launches; with dispatch, placed rows and combine 16 of 64 experts of 7168 x 2048 took 141 us.
    const bool token = tokens == 1u;
    if (token) {
        if (!k3_moe_fp8_quantize_rows(w.x.codes, w.x.scales, x, 1u, d->hidden, K3_MOE_FP8_BF16, stream)) return false;
    } else {
        if (!k3_moe_dispatch_build(w.offsets, w.sorted_route, w.sorted_token, w.inv_perm, ids, tokens, d->top_k, d->experts,
                                   w.dispatch, w.dispatch_bytes, stream)) {
            return false;
        }
        const Placement at{w.inv_perm, (const uint32_t *)ids, d->top_k, d->experts, routes};
        if (!quantize_placed(w.x.codes, w.x.scales, x, tokens, d->hidden, at, w.rows_out + (uint64_t)routes * d->hidden,
                             d->hidden * (uint32_t)sizeof(float), stream)) {
            return false;
        }
    }
    Product p{};
    p.out = w.act.codes;
    p.out_scales = w.act.scales;
    p.a = w.x.codes;
    p.a_scales = w.x.scales;
    p.b = d->w1;
    p.b_scales = d->w1_scales;
    p.b2 = d->w3;
    p.b2_scales = d->w3_scales;
    p.offsets = token ? nullptr : w.offsets;
    p.ids = (const uint32_t *)ids;
    p.top_k = d->top_k;
    p.groups = d->experts;
    p.rows = token ? 1u : routes;
    p.n = d->expert_hidden;
    p.k = d->hidden;
    p.b_scale_layout = K3_MOE_FP8_BLOCKS;
    p.epilogue = kOutActivated;
    p.b_ready = true;                // the launch in front is the quantiser, then the gate/up product
    p.activation = d->activation;
    p.beta = d->beta;
    p.linear_beta = d->linear_beta;
    if (token ? !token_gateup(p, stream) : !product(p, stream)) return false;
    p.out = w.rows_out;
    p.out_scales = nullptr;
    p.a = w.act.codes;
    p.a_scales = w.act.scales;
    p.b = d->w2;
    p.b_scales = d->w2_scales;
    p.b2 = p.b2_scales = nullptr;
    p.n = d->hidden;
    p.k = d->expert_hidden;
    p.epilogue = token ? kOutBf16 : kOutF32;
    if (token) {
        p.out = out;
        p.rows = 1u;
        p.weights = (const float *)weights;
        p.shared = shared;
        return token_down(p, stream);
    }
    if (!product(p, stream)) return false;
    return launch_chained(combine_f32_kernel, dim3(tokens, (d->hidden / 4u + 127u) / 128u), 128, 0, stream, (uint16_t *)out,
                          (const float *)w.rows_out, (const uint32_t *)w.inv_perm, (const float *)weights,
                          (const uint16_t *)shared, d->top_k, d->hidden);
}
