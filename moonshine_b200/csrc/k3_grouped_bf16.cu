// Entry points of the bf16 products grouped by expert (include/k3_moe_grouped.h).
#include "k3_grouped_bf16.h"

using namespace k3;
using namespace k3::gb;

namespace {

bool extent_ok(uint32_t n) { return n != 0u && n <= (1u << 30); }
bool aligned(const void *p, uint32_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }

bool run(const Product &p, int out_type, size_t workspace_bytes, void *stream) {
    if (!p.out || !p.a || !p.b || !p.offsets || !p.workspace) return false;
    if (!extent_ok(p.rows) || !extent_ok(p.n) || !extent_ok(p.k) || p.groups == 0u || p.groups > kMaxGroups) return false;
    if (out_type != K3_MOE_GROUPED_BF16 && out_type != K3_MOE_GROUPED_F32) return false;
    if (p.accumulate && !p.f32) return false;
    if (!aligned(p.out, p.f32 ? 4u : 2u) || !aligned(p.a, 2u) || !aligned(p.b, 2u) || !aligned(p.offsets, 4u) ||
        !aligned(p.workspace, 16u) || workspace_bytes < k3_moe_grouped_workspace_bytes(p.rows, p.groups)) {
        return false;
    }
    // what the TMA unit reads: rows of whole 16-byte units
    const bool tc = p.n % 8u == 0u && p.k % 8u == 0u && aligned(p.out, 16u) && aligned(p.a, 16u) && aligned(p.b, 16u);
    return tc ? product_tc(p, (cudaStream_t)stream) : product_any(p, (cudaStream_t)stream);
}

}  // namespace

extern "C" size_t k3_moe_grouped_workspace_bytes(uint32_t rows, uint32_t groups) {
    if (!extent_ok(rows) || groups == 0u || groups > kMaxGroups) return 0;
    return tc_workspace_bytes(rows, groups);
}

extern "C" bool k3_moe_grouped_product(void *out, const void *x, const void *w, const void *offsets, uint32_t rows,
                                       uint32_t groups, uint32_t n, uint32_t k, int out_type, int accumulate,
                                       void *workspace, size_t workspace_bytes, void *stream) {
    return run({out, x, w, (const uint32_t *)offsets, rows, groups, n, k, kForward, out_type == K3_MOE_GROUPED_F32,
                accumulate != 0, workspace}, out_type, workspace_bytes, stream);
}

extern "C" bool k3_moe_grouped_by_input(void *dx, const void *dy, const void *w, const void *offsets, uint32_t rows,
                                        uint32_t groups, uint32_t n, uint32_t k, int out_type, int accumulate,
                                        void *workspace, size_t workspace_bytes, void *stream) {
    return run({dx, dy, w, (const uint32_t *)offsets, rows, groups, n, k, kByInput, out_type == K3_MOE_GROUPED_F32,
                accumulate != 0, workspace}, out_type, workspace_bytes, stream);
}

extern "C" bool k3_moe_grouped_by_weight(void *dw, const void *dy, const void *x, const void *offsets, uint32_t rows,
                                         uint32_t groups, uint32_t n, uint32_t k, int out_type, int accumulate,
                                         void *workspace, size_t workspace_bytes, void *stream) {
    return run({dw, dy, x, (const uint32_t *)offsets, rows, groups, n, k, kByWeight, out_type == K3_MOE_GROUPED_F32,
                accumulate != 0, workspace}, out_type, workspace_bytes, stream);
}
