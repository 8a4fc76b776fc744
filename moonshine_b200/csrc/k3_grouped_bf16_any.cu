// bf16 products grouped by expert for matrices whose rows are not whole units of 16 bytes, which the TMA unit
// cannot read: f32 FMAs from tiles in shared memory.
//
//   D[m, c] = sum_r A(m, r) B(c, r)
//     forward    m a row of the group, c < n, r < k:   A = x[m, r],  B = w_g[c, r]
//     by input   m a row of the group, c < k, r < n:   A = dy[m, r], B = w_g[r, c]
//     by weight  m < n, c < k, r a row of the group:   A = dy[r, m], B = x[r, c]
//
// One block of 256 threads makes a tile of 64 x 64, 4 x 4 per thread, over steps of 16 of the depth.  A sum of d products
// that are added one by one is off by up to 2^-23 / sqrt(12) sqrt(d / 2) of itself (8.7e-7 measured at 7169, 2.3e-6 at 32770), so
// every 512 it is closed and added to those before: 1.8e-7 at 7169.  8 groups of 256 rows, 2047 x 1023: 457 us forward (453
// without), 516 by input (514), 276 by weight (268); 2 of 100, 130 x 7169, 658 (569).  Bound by the FMA pipes and the
// two-byte loads around them; nothing here is meant to be fast, and shapes that models have take the other kernels.
#include "k3_grouped_bf16.h"

using namespace k3;
using namespace k3::gb;

namespace {

constexpr uint32_t kTile = 64, kDepth = 16, kThreads = 256, kSegment = 512;

struct AnyArgs {
    void *out;
    const uint16_t *a, *b;
    const uint32_t *offsets;
    uint32_t rows, groups, n, k, column_tiles;
    int accumulate;
};

// The group that row tile `tile` of all groups' tiles belongs to and its first row; false past the last tile.
// All threads of the block call it.
K3_DEVINL bool find_tile(const AnyArgs &a, uint32_t tile, uint32_t &group, uint32_t &row, uint32_t &end) {
    __shared__ uint64_t sums[kThreads / kWarp];                    // 64 bits: overlapping groups can have more than 2^32 tiles
    __shared__ uint32_t found[3];
    constexpr uint32_t kEach = kMaxGroups / kThreads;
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    uint32_t tiles[kEach];
    uint64_t mine = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t g = threadIdx.x * kEach + i;
        uint32_t begin = 0u, past = 0u;
        if (g < a.groups) group_rows(a.offsets, g, a.rows, begin, past);
        tiles[i] = (past - begin + kTile - 1u) / kTile;
        mine += tiles[i];
    }
    uint64_t scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= (uint32_t)o) scan += up;
    }
    if (lane == 31u) sums[warp] = scan;
    if (threadIdx.x == 0u) found[0] = 0xffffffffu;
    __syncthreads();
    uint64_t first = scan - mine;
    for (uint32_t w = 0; w < warp; w++) first += sums[w];
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        if (tile >= first && tile < first + tiles[i]) {
            uint32_t begin, past;
            group_rows(a.offsets, threadIdx.x * kEach + i, a.rows, begin, past);
            found[0] = threadIdx.x * kEach + i;
            found[1] = begin + (tile - (uint32_t)first) * kTile;
            found[2] = past;
        }
        first += tiles[i];
    }
    __syncthreads();
    group = found[0];
    row = found[1];
    end = found[2];
    return group != 0xffffffffu;
}

template <int kForm, bool kF32>
__global__ void __launch_bounds__(kThreads) grouped_any_kernel(AnyArgs a) {
    pdl_wait();
    __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4];
    uint32_t group, m0, m_end, c0, c_end, depth;           // the tile's extents, ends not included
    uint32_t r0 = 0u;                                      // by weight: the group's first row
    if (kForm == kByWeight) {
        const uint32_t tiles_n = (a.n + kTile - 1u) / kTile;
        group = blockIdx.x / (tiles_n * a.column_tiles);
        const uint32_t at = blockIdx.x - group * tiles_n * a.column_tiles;
        m0 = at / a.column_tiles * kTile;
        c0 = at % a.column_tiles * kTile;
        m_end = a.n;
        c_end = a.k;
        uint32_t past;
        group_rows(a.offsets, group, a.rows, r0, past);
        depth = past - r0;
        if (depth == 0u && a.accumulate) return;
    } else {
        if (!find_tile(a, blockIdx.x / a.column_tiles, group, m0, m_end)) return;
        c0 = blockIdx.x % a.column_tiles * kTile;
        c_end = kForm == kForward ? a.n : a.k;
        depth = kForm == kForward ? a.k : a.n;
    }
    const uint16_t *w = a.b + (kForm == kByWeight ? 0u : (uint64_t)group * a.n * a.k);
    const uint32_t tm = threadIdx.x / 16u * 4u, tc = threadIdx.x % 16u * 4u;
    float sum[4][4] = {}, closed[4][4] = {};
    for (uint32_t d0 = 0; d0 < depth; d0 += kDepth) {
#pragma unroll
        for (uint32_t i = 0; i < kTile * kDepth / kThreads; i++) {
            const uint32_t e = threadIdx.x + i * kThreads;
            // neighbouring threads along what lies side by side in memory
            const uint32_t am = kForm == kByWeight ? e % kTile : e / kDepth, ad = kForm == kByWeight ? e / kTile : e % kDepth;
            const uint32_t bc = kForm == kForward ? e / kDepth : e % kTile, bd = kForm == kForward ? e % kDepth : e / kTile;
            float va = 0.f, vb = 0.f;
            if (m0 + am < m_end && d0 + ad < depth) {
                const uint64_t at = kForm == kForward ? (uint64_t)(m0 + am) * a.k + d0 + ad
                                    : kForm == kByInput ? (uint64_t)(m0 + am) * a.n + d0 + ad
                                                        : (uint64_t)(r0 + d0 + ad) * a.n + m0 + am;
                va = bf16_bits_to_float(a.a[at]);
            }
            if (c0 + bc < c_end && d0 + bd < depth) {
                const uint64_t at = kForm == kForward ? (uint64_t)(c0 + bc) * a.k + d0 + bd
                                    : kForm == kByInput ? (uint64_t)(d0 + bd) * a.k + c0 + bc
                                                        : (uint64_t)(r0 + d0 + bd) * a.k + c0 + bc;
                vb = bf16_bits_to_float(w[at]);
            }
            as[ad][am] = va;
            bs[bd][bc] = vb;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t d = 0; d < kDepth; d++) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) sum[i][j] = fmaf(as[d][tm + i], bs[d][tc + j], sum[i][j]);
            }
        }
        __syncthreads();
        if (d0 % kSegment == kSegment - kDepth || d0 + kDepth >= depth) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) {
                    closed[i][j] += sum[i][j];
                    sum[i][j] = 0.0f;
                }
            }
        }
    }
    const uint32_t pitch = c_end;
    const uint64_t base = kForm == kByWeight ? (uint64_t)group * a.n * a.k : 0u;
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) {
            if (m0 + tm + i >= m_end || c0 + tc + j >= c_end) continue;
            const uint64_t at = base + (uint64_t)(m0 + tm + i) * pitch + c0 + tc + j;
            if (kF32) ((float *)a.out)[at] = a.accumulate ? ((float *)a.out)[at] + closed[i][j] : closed[i][j];
            else ((uint16_t *)a.out)[at] = float_to_bf16_bits(closed[i][j]);
        }
    }
}

template <int kForm>
bool launch(const Product &p, cudaStream_t stream) {
    AnyArgs a{p.out, (const uint16_t *)p.a, (const uint16_t *)p.b, p.offsets, p.rows, p.groups, p.n, p.k, 0u, p.accumulate};
    const uint32_t columns = kForm == kForward ? p.n : p.k;
    a.column_tiles = (columns + kTile - 1u) / kTile;
    const uint64_t tiles = kForm == kByWeight ? (uint64_t)p.groups * ((p.n + kTile - 1u) / kTile)
                                              : (uint64_t)p.rows / kTile + min(p.rows, p.groups);
    const uint64_t blocks = tiles * a.column_tiles;
    if (blocks > 0x7fffffffull) return false;
    return p.f32 ? launch_chained(grouped_any_kernel<kForm, true>, (uint32_t)blocks, kThreads, 0, stream, a)
                 : launch_chained(grouped_any_kernel<kForm, false>, (uint32_t)blocks, kThreads, 0, stream, a);
}

}  // namespace

bool k3::gb::product_any(const Product &p, cudaStream_t stream) {
    if (p.form == kForward) return launch<kForward>(p, stream);
    return p.form == kByInput ? launch<kByInput>(p, stream) : launch<kByWeight>(p, stream);
}
