// Weight gradients of groups of up to 16 rows: dw_g[n, k] = sum over the group's rows of dy[r, n] x[r, k].
//
// A group is one step of the depth of mma.sync (m16n8k16).  A warp makes 64 rows of a matrix by 32 columns at a time, of several
// tiles along n (x stays in registers, the next tile's dy is on its way), with operands as they lie in memory: no shared
// memory and no barrier stands before the stores, whose bytes bound it.  Which rows and columns of the tile an MMA stands for is
// free, so that a lane's registers of all MMAs come from whole units: MMA i of four along n has in its rows l and l + 8 the
// rows 8 l + 2 i and 8 l + 2 i + 1; MMA j of four along k has in its column c, for bf16, column c / 2 * 8 + 2 j + c % 2, so
// that a lane's results of all j are 8 neighbouring columns (f32: 4 of j = 0, 1 and 4 of j = 2, 3).
// 32 groups of 1 row, 2048 x 7168: bf16 147 us, 6.4 TB/s, f32 272, 6.9; of 8 rows 164 and 287.  f32 FMAs in its place take 200 us
// for 1 row and 14 more (896 groups of 264 x 520) for each further one.
#include "k3_fp8_ptx.cuh"
#include "k3_grouped_bf16.h"

#include <algorithm>

using namespace k3;
using namespace k3::gb;
using k3::fp8::bf16x2;

namespace {

constexpr uint32_t kThreads = 256, kTileN = 64, kTileK = 32;

struct OuterArgs {
    void *out;
    const uint16_t *dy, *x;
    const uint32_t *offsets;
    uint32_t rows, groups, n, k;
    uint32_t each;                                                       // tiles along n of a warp
    uint32_t parts_n, tiles_k;
    int accumulate;
};

K3_DEVINL void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
K3_DEVINL uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
K3_DEVINL uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// A lane's part of 16 rows of the group from `row` on: units of dy from column m, of x from column c on.
K3_DEVINL void load_dy(const OuterArgs &a, uint32_t row, uint32_t end, uint32_t q, uint32_t m, uint4 (&dy)[4]) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
        const uint32_t r = row + 2u * q + (i & 1u) + (i / 2u) * 8u;
        dy[i] = r < end && m < a.n ? *reinterpret_cast<const uint4 *>(a.dy + (uint64_t)r * a.n + m) : make_uint4(0u, 0u, 0u, 0u);
    }
}
template <bool kF32>
K3_DEVINL void load_x(const OuterArgs &a, uint32_t row, uint32_t end, uint32_t l, uint32_t q, uint32_t k0, uint32_t (&b)[4][2]) {
    const uint32_t c = kF32 ? k0 + l / 2u * 4u : k0 + l / 2u * 8u, second = kF32 ? 16u : 4u;
    uint2 x[4][2];
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
        const uint32_t r = row + 2u * q + (i & 1u) + (i / 2u) * 8u;
        const uint16_t *from = a.x + (uint64_t)r * a.k + c;
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            x[i][h] = r < end && c + h * second < a.k ? *reinterpret_cast<const uint2 *>(from + h * second) : make_uint2(0u, 0u);
        }
    }
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) {
#pragma unroll
        for (uint32_t j = 0; j < 2u; j++) {
            const uint2 lo = x[2u * h][j], hi = x[2u * h + 1u][j];
            b[2u * j][h] = l & 1u ? high_halves(lo.x, hi.x) : low_halves(lo.x, hi.x);
            b[2u * j + 1u][h] = l & 1u ? high_halves(lo.y, hi.y) : low_halves(lo.y, hi.y);
        }
    }
}
K3_DEVINL void multiply(float (&sum)[4][4], uint32_t d0, uint32_t d1, uint32_t d2, uint32_t d3, const uint32_t (&b)[4][2]) {
    const uint32_t a0 = low_halves(d0, d1), a1 = high_halves(d0, d1), a2 = low_halves(d2, d3), a3 = high_halves(d2, d3);
#pragma unroll
    for (uint32_t j = 0; j < 4u; j++) mma16(sum[j], a0, a1, a2, a3, b[j][0], b[j][1]);
}
K3_DEVINL uint32_t word(const uint4 &v, uint32_t i) { return i == 0u ? v.x : i == 1u ? v.y : i == 2u ? v.z : v.w; }

// Two rows of dw from element `at` on, a lane's columns of them.
template <bool kF32>
K3_DEVINL void store(const OuterArgs &a, uint64_t at, uint32_t k0, uint32_t q, const float (&sum)[4][4]) {
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) {
        const uint64_t row = at + (uint64_t)h * a.k;
        if constexpr (kF32) {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j += 2u) {
                const uint32_t c = k0 + j / 2u * 16u + q * 4u;
                if (c >= a.k) continue;
                float4 *to = reinterpret_cast<float4 *>((float *)a.out + row + c);
                float4 v = make_float4(sum[j][2u * h], sum[j][2u * h + 1u], sum[j + 1u][2u * h], sum[j + 1u][2u * h + 1u]);
                if (a.accumulate) {
                    const float4 was = *to;
                    v = make_float4(was.x + v.x, was.y + v.y, was.z + v.z, was.w + v.w);
                }
                *to = v;
            }
        } else if (k0 + q * 8u < a.k) {
            uint32_t v[4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) v[j] = bf16x2(sum[j][2u * h], sum[j][2u * h + 1u]);
            *reinterpret_cast<uint4 *>((uint16_t *)a.out + row + k0 + q * 8u) = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads) grouped_outer_kernel(OuterArgs a) {
    pdl_trigger();                                                       // the kernel behind: once all blocks have begun
    pdl_wait();
    const uint32_t lane = threadIdx.x % kWarp, l = lane / 4u, q = lane % 4u;
    const uint64_t task = (uint64_t)blockIdx.x * (kThreads / kWarp) + threadIdx.x / kWarp;
    const uint32_t tasks = a.parts_n * a.tiles_k;
    if (task >= (uint64_t)a.groups * tasks) return;
    const uint32_t group = (uint32_t)(task / tasks), at = (uint32_t)(task - (uint64_t)group * tasks);
    uint32_t row, end;
    group_rows(a.offsets, group, a.rows, row, end);
    if (end - row > kOuterRows || (row == end && a.accumulate)) return;
    if (row == end) {
        // zeros: the matrix from end to end, a part per warp (896 groups of 264 x 520, 75 of them with rows: 47 us, by tiles 63)
        const uint64_t units = (uint64_t)a.n * a.k / (kF32 ? 4u : 8u), part = (units + tasks - 1u) / tasks;
        uint4 *to = reinterpret_cast<uint4 *>(a.out) + group * units;
        const uint64_t past = min(units, (at + 1u) * part);
        for (uint64_t i = at * part + lane; i < past; i += kWarp) to[i] = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const uint32_t k0 = at % a.tiles_k * kTileK;
    uint32_t m0 = at / a.tiles_k * a.each * kTileN;
    const uint32_t m_end = min(m0 + a.each * kTileN, a.n);
    const uint64_t matrix = (uint64_t)group * a.n * a.k;
    uint32_t b[4][2];
    uint4 dy[4];
    load_x<kF32>(a, row, end, l, q, k0, b);
    uint4 next[4];
    load_dy(a, row, end, q, m0 + l * 8u, next);
    for (; m0 < m_end; m0 += kTileN) {
        const uint32_t m = m0 + l * 8u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) dy[i] = next[i];
        if (m0 + kTileN < m_end) load_dy(a, row, end, q, m + kTileN, next);
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            float sum[4][4] = {};
            multiply(sum, word(dy[0], i), word(dy[1], i), word(dy[2], i), word(dy[3], i), b);
            if (m < a.n) store<kF32>(a, matrix + (uint64_t)(m + 2u * i) * a.k, k0, q, sum);
        }
    }
}

}  // namespace

bool k3::gb::product_outer(const Product &p, cudaStream_t stream) {
    const uint32_t tiles_n = (p.n + kTileN - 1u) / kTileN, tiles_k = (p.k + kTileK - 1u) / kTileK;
    // up to eight tiles per warp while every SM has 32 warps (32 groups, 2048 x 7168, bf16: one 229 us, two 182, four 160, eight 152)
    const uint64_t tiles = (uint64_t)tiles_n * tiles_k * p.groups;
    const uint32_t most = (uint32_t)std::min<uint64_t>(8u, std::max<uint64_t>(1u, tiles / ((uint64_t)sm_count() * 32u)));
    const uint32_t parts_n = (tiles_n + most - 1u) / most, each = (tiles_n + parts_n - 1u) / parts_n;
    const OuterArgs a{p.out, (const uint16_t *)p.a, (const uint16_t *)p.b, p.offsets, p.rows, p.groups, p.n, p.k, each, parts_n, tiles_k, p.accumulate};
    const uint64_t tasks = (uint64_t)parts_n * tiles_k, blocks = (tasks * p.groups + kThreads / kWarp - 1u) / (kThreads / kWarp);
    if (tasks > 0xffffffffull || blocks > 0x7fffffffull) return false;
    return p.f32 ? launch_chained(grouped_outer_kernel<true>, (uint32_t)blocks, kThreads, 0, stream, a)
                 : launch_chained(grouped_outer_kernel<false>, (uint32_t)blocks, kThreads, 0, stream, a);
}
