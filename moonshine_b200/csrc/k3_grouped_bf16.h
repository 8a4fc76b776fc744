// Internal interface of the bf16 products grouped by expert: entry points and choice (k3_grouped_bf16.cu), the
// tensor-core kernels (k3_grouped_bf16_tc.cu), the kernel for any sizes (k3_grouped_bf16_any.cu).
#pragma once

#include "k3_common.cuh"
#include "k3_moe_grouped.h"

namespace k3::gb {

constexpr uint32_t kMaxGroups = 1024;

enum Form : int { kForward = 0, kByInput = 1, kByWeight = 2 };

// forward: a = x [rows, k], b = w; by input: a = dy [rows, n], b = w; by weight: a = dy, b = x [rows, k].
struct Product {
    void *out;
    const void *a, *b;
    const uint32_t *offsets;
    uint32_t rows, groups, n, k;
    int form;
    bool f32, accumulate;
    void *workspace;
};

// The rows of group g, whatever the offsets hold: inside [0, rows).
K3_DEVINL void group_rows(const uint32_t *offsets, uint32_t g, uint32_t rows, uint32_t &begin, uint32_t &end) {
    begin = min(offsets[g], rows);
    end = max(begin, min(offsets[g + 1u], rows));
}

bool product_any(const Product &p, cudaStream_t stream);
// n and k multiples of 8, all pointers but the offsets on 16 bytes
bool product_tc(const Product &p, cudaStream_t stream);
uint64_t tc_workspace_bytes(uint32_t rows, uint32_t groups);
// by weight, as product_tc, for the groups of up to kOuterRows rows
constexpr uint32_t kOuterRows = 16;
bool product_outer(const Product &p, cudaStream_t stream);

}  // namespace k3::gb
