// Products of E4M3 matrices with few rows on tcgen05 (kind::f8f6f4): what has to be read is b, a weight
// table, and HBM bounds it.
//
//   out[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in kb} a[m, k] b[n, k]
//
// Here b's rows are the lanes (the MMA's 128) and a's rows its N extent, 16 to 64 columns, so a few rows
// of a cost no more than their own loads.  128 lanes share a block scale; a row's scale goes with the
// column, so the factors sa sb of a block lie in shared memory and every lane reads the same one.
//
// kSplit (one matrix, up to 16 rows): a work item is 128 rows of b and a part of the depth; the parts of an
// item are a cluster, which adds its sums through distributed shared memory in ascending order of the
// depth.  Two blocks fit an SM.
// Otherwise (groups of a few dozen rows): one block per SM goes over items of 256 rows of b (kOutActivated:
// 128 of gate and the same 128 of up) and up to 64 of a over the whole depth.
//
// kQuantize (a linear layer's call with up to 16 rows, split): a is bf16, and four more warps quantise the
// part of its rows that a block needs, a block of 128 columns each, straight into the operand's place. Every
// tile of b does so again, which is little beside the launch it saves: one token of 3584 x 7168 takes 7.6 us,
// with a launch of its own 10.0.
// kToken (the routed experts of one token): the groups are the token's routes, one row each, without a
// dispatch.  Gate/up (grouped): item (route, 128 columns), all routes read the same row of a.  Down (split):
// the depth runs over the routes one after the other and a route's weight is part of its factors, so the
// sum over the experts is formed like any other and nothing is written in between.  A route whose id is no
// expert reads zeros.
// b_ready: the kernel in front writes neither b nor the offsets, and has waited for everything in front of it
// before it let this one start, so b's first stages are fetched while it runs.
//
// Warps: 0 loads by TMA, 1 MMA issuer and owner of the tensor memory, 2 factors, then four per 32 rows
// of a with the running sums, then the quantising ones.  Every wait is bounded; on give-up the block
// raises the status word, waits for its copies and frees its tensor memory.
//
// Measured: one row of 7168 x 7168 11.6 us (4.4 TB/s of the table; a launch, the first loads and the way
// through the cluster are half of it), 16 of 64 experts of 7168 x 2048 for one token 120 us (5.9 TB/s,
// 0.89 of the copy rate), 61 tokens through 8 of 64 experts 375 us (the tables they select at 6.5 TB/s).
#include "k3_fp8_ptx.cuh"
#include "k3_grouped.h"
#include "k3_moe_layer.h"

#include <algorithm>

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kMaxGroups = 1024;
constexpr uint32_t kMaxSplits = 8;                                   // of the depth: the portable cluster
constexpr uint32_t kGroupRows = 64;                                  // of a group per item
constexpr uint32_t kBoxRows = 16;                                    // a's rows per box: what an MMA column step is

__device__ uint32_t g_fp8_few_status = 0;

template <uint32_t kTiles, uint32_t kRows, bool kSplit, bool kQuantize>
struct Layout {
    static_assert(!kSplit || kRows == 16u, "more rows of one matrix: k3_fp8_wide.cu");
    static_assert(kSplit || !kQuantize, "only a linear layer quantises here");
    static constexpr uint32_t kHalves = (kRows + 31u) / 32u;
    static constexpr uint32_t kSumWarps = 4u * kHalves, kQuantizeWarps = kQuantize ? 4u : 0u;
    static constexpr uint32_t kThreads = (4u + kSumWarps + kQuantizeWarps) * kWarp;
    static constexpr uint32_t kPerSm = kSplit ? 2u : 1u;
    static constexpr uint32_t kBTile = kBlock * kBlock;              // 128 rows of b, 128 columns
    static constexpr uint32_t kStageBytes = kTiles * kBTile + kRows * kBlock;
    static constexpr uint32_t kStages = kRows <= 16u ? 6u : 5u;
    // factors travel four blocks at a time, or with the codes
    static constexpr uint32_t kSlots = kQuantize ? 8u : 2u, kSlotBlocks = kQuantize ? 1u : 4u;
    static constexpr uint32_t kFactors = kStages * kStageBytes;      // f32 [kSlots][kSlotBlocks][kTiles][kRows]
    static constexpr uint32_t kSlotFloats = kSlotBlocks * kTiles * kRows;
    static constexpr uint32_t kLargest = kFactors + kSlots * kSlotFloats * 4u;   // f32 bits [4][kRows]
    static constexpr uint32_t kPrefix = kLargest + 4u * kRows * 4u;
    static constexpr uint32_t kRoutes = kPrefix;                     // kToken: ids [32], weights [32] in the prefix's place
    static constexpr uint32_t kBars = (kPrefix + (kSplit ? 256u : (kMaxGroups + 1u) * 4u) + 15u) / 16u * 16u;
    static constexpr uint32_t kBytes = kBars + 512u + 1024u;         // the last: alignment
    static constexpr uint32_t kTmem = kTiles * kRows * 2u < 32u ? 32u : kTiles * kRows * 2u;
    static_assert(kBytes <= (kPerSm == 2u ? 115000u : 232448u), "two blocks of a split product share an SM");
    static_assert(!kSplit || kRows * kBlock * 4u <= kFactors, "partial sums take the ring's place");
};

struct FewArgs {
    void *out;
    float *out_scales;
    const float *a_scales, *b_scales, *b2_scales;
    const uint16_t *x;                             // kQuantize: a as bf16
    bool x_vector;                                 // its rows are whole 16-byte units
    bool b_ready;
    const uint32_t *offsets;
    const uint32_t *ids;                           // kToken
    const float *weights;
    const uint16_t *shared;                        // kToken, split: bf16 [n] or null
    uint32_t top_k;
    uint32_t groups, rows, n, k;
    uint32_t column_items;                         // grouped: items along b's rows
    uint32_t split_blocks;                         // kSplit: blocks of 128 per part of the depth
    int accumulate;
    int activation;
    float beta, by_beta, linear_beta, by_linear_beta;                // by_: the reciprocals
};

struct Item {
    uint32_t group, row, rows, column, kb_begin, kb_end;
};

K3_DEVINL void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
K3_DEVINL void tmem_ld_wait_for(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

template <int kEpilogue, uint32_t kTiles, uint32_t kRows, bool kSplit, bool kQuantize, bool kToken>
__global__ void __launch_bounds__(Layout<kTiles, kRows, kSplit, kQuantize>::kThreads, Layout<kTiles, kRows, kSplit, kQuantize>::kPerSm)
fp8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_b2, FewArgs a) {
    using L = Layout<kTiles, kRows, kSplit, kQuantize>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(base + L::kBars);  // [kStages]
    uint64_t *empty = full + L::kStages;                             // [kStages]
    uint64_t *sum_full = empty + L::kStages;                         // [2] a block's products are in tensor memory
    uint64_t *sum_empty = sum_full + 2;                              // [2] and have been read
    uint64_t *factor_full = sum_empty + 2;                           // [kSlots]
    uint64_t *factor_empty = factor_full + L::kSlots;                // [kSlots]
    uint64_t *largest_full = factor_empty + L::kSlots;               // [2] one per half
    uint64_t *done = largest_full + 2;                               // [1] every MMA issued has run
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    uint32_t *total_s = tmem_slot + 2;
    uint32_t *prefix = reinterpret_cast<uint32_t *>(base + L::kPrefix);
    uint32_t *ids_s = reinterpret_cast<uint32_t *>(base + L::kRoutes);
    float *weights_s = reinterpret_cast<float *>(ids_s + 32);
    const uint32_t warp = warp_index(), lane = threadIdx.x % kWarp;
    const uint32_t blocks = blocks_of(a.k);
    constexpr uint32_t kColumns = kEpilogue == kOutActivated ? kBlock : kTiles * kBlock;

    auto item_of = [&](uint32_t w) {
        Item it;
        it.kb_begin = 0u;
        it.kb_end = blocks;
        if (kSplit) {
            it.group = 0u;
            it.row = blockIdx.z * kRows;
            it.rows = min(kRows, a.rows - it.row);
            it.column = blockIdx.y * kBlock;
            it.kb_begin = blockIdx.x * a.split_blocks;
            it.kb_end = min(kToken ? a.top_k * blocks : blocks, it.kb_begin + a.split_blocks);
            return it;
        }
        const uint32_t tile = w / a.column_items;
        it.column = (w - tile * a.column_items) * kColumns;
        if (kToken) {
            it.group = ids_s[tile];
            it.row = tile;
            it.rows = 1u;
            return it;
        }
        uint32_t lo = 0u, hi = a.groups;                             // the last group whose first tile is at most `tile`
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (prefix[mid] <= tile) lo = mid; else hi = mid;
        }
        it.group = lo;
        it.row = a.offsets[lo] + (tile - prefix[lo]) * kRows;
        it.rows = min(kRows, a.offsets[lo + 1u] - it.row);
        return it;
    };

    const uint64_t stream_once = l2_policy_evict_first();
    // kToken, split: step kb of the depth is block kb % blocks of this route
    auto route_of = [&](uint32_t kb) { return kSplit && kToken ? kb / blocks : 0u; };
    auto load_b = [&](const Item &it, uint32_t stage, uint32_t kb, uint32_t group) {
        unsigned char *st = base + stage * L::kStageBytes;
        const int32_t x = (int32_t)((kb - route_of(kb) * blocks) * kBlock);
        // past the table's end: zeros
        const int32_t y = (int32_t)(kToken && group >= a.groups ? a.groups * a.n : group * a.n + it.column);
        const uint32_t boxes = kQuantize ? 0u : (it.rows + kBoxRows - 1u) / kBoxRows;
        mbar_arrive_expect_tx(&full[stage], kTiles * L::kBTile + boxes * kBoxRows * kBlock);
        tma_load_2d_hint(st, &map_b, &full[stage], x, y, stream_once);
        if (kTiles == 2u) {
            if (kEpilogue == kOutActivated) tma_load_2d_hint(st + L::kBTile, &map_b2, &full[stage], x, y, stream_once);
            else tma_load_2d_hint(st + L::kBTile, &map_b, &full[stage], x, y + (int32_t)kBlock, stream_once);
        }
    };

    if (warp == 0u && elect_one()) {
        *abort_flag = 0u;
        for (uint32_t s = 0; s < L::kStages; s++) {
            mbar_init(&full[s], kQuantize ? 2u : 1u);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t s = 0; s < 2u; s++) {
            mbar_init(&sum_full[s], 1);
            mbar_init(&sum_empty[s], L::kSumWarps);
            mbar_init(&largest_full[s], 4);
        }
        for (uint32_t s = 0; s < L::kSlots; s++) {
            mbar_init(&factor_full[s], kQuantize ? 1u : kWarp);
            mbar_init(&factor_empty[s], L::kSumWarps);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_b);
        if (kEpilogue == kOutActivated) prefetch_tensormap(&map_b2);
        if (!kQuantize) prefetch_tensormap(&map_a);
        if (kSplit) {                                                // b's first stages, before anyone waits for anyone
            if (!a.b_ready) pdl_wait();
            const Item it = item_of(0u);
            uint32_t route = 0xffffffffu, group = 0u;
            for (uint32_t i = 0; i < min(L::kStages, it.kb_end - it.kb_begin); i++) {
                const uint32_t kb = it.kb_begin + i;
                if (kToken && route_of(kb) != route) {
                    route = route_of(kb);
                    group = a.ids[route];
                }
                load_b(it, i, kb, group);
            }
            pdl_wait();
        }
    }
    if (warp == 1u) {
        tmem_alloc(tmem_slot, L::kTmem);
        tmem_relinquish();
    }
    if (kSplit ? warp != 0u : !a.b_ready) pdl_wait();
    if (kToken && warp == 3u && lane < a.top_k) {
        ids_s[lane] = a.ids[lane];
        weights_s[lane] = kSplit ? a.weights[lane] : 0.f;
        if (!kSplit && blockIdx.x == 0u && ids_s[lane] >= a.groups) atomicOr(&g_fp8_few_status, 2u);
    }
    if (kToken && !kSplit && threadIdx.x == 0u) *total_s = a.top_k * a.column_items;
    if (!kSplit && !kToken && warp == 2u) {
        // exclusive prefix of the groups' row tiles, 32 groups at a time
        uint32_t before = 0u;
        for (uint32_t g0 = 0; g0 < a.groups; g0 += kWarp) {
            const uint32_t g = g0 + lane;
            const uint32_t n = g < a.groups ? (a.offsets[g + 1u] - a.offsets[g] + kRows - 1u) / kRows : 0u;
            uint32_t scan = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
                if (lane >= (uint32_t)o) scan += up;
            }
            if (g < a.groups) prefix[g] = before + scan - n;
            before += __shfl_sync(0xffffffffu, scan, 31);
        }
        if (lane == 0u) *total_s = before * a.column_items;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t first_item = kSplit ? 0u : blockIdx.x, step = kSplit ? 1u : gridDim.x, total = kSplit ? 1u : *total_s;

    if (warp == 0u) {
        // ----------------------------------------------------------------------------- loads
        if (elect_one()) {
            uint32_t s = 0u, ph = 0u, issued = 0u, early = 0u;
            bool ok = true;
            if (kSplit) {
                const Item it = item_of(0u);
                early = min(L::kStages, it.kb_end - it.kb_begin);
            }
            if (!kSplit && a.b_ready) {
                if (first_item < total) {
                    const Item it = item_of(first_item);
                    early = min(L::kStages, it.kb_end);
                    for (uint32_t i = 0; i < early; i++) load_b(it, i, i, it.group);
                }
                pdl_wait();
            }
            for (uint32_t w = first_item; ok && w < total; w += step) {
                const Item it = item_of(w);
                const uint32_t boxes = (it.rows + kBoxRows - 1u) / kBoxRows;
                for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb++) {
                    if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) { ok = false; break; }
                    const uint32_t route = route_of(kb), group = kSplit && kToken ? ids_s[route] : it.group;
                    if (issued >= early) load_b(it, s, kb, group);
                    unsigned char *rows = base + s * L::kStageBytes + kTiles * L::kBTile;
                    // one token: its only row, or the route's
                    const uint32_t row = !kToken ? it.row : kSplit ? (group < a.groups ? route : a.top_k) : 0u;
                    for (uint32_t i = 0; !kQuantize && i < boxes; i++) {
                        tma_load_2d(rows + i * kBoxRows * kBlock, &map_a, &full[s], (int32_t)((kb - route * blocks) * kBlock),
                                    (int32_t)(row + i * kBoxRows));
                    }
                    issued++;
                    if (++s == L::kStages) { s = 0u; ph ^= 1u; }
                }
            }
            pdl_trigger();                                           // the blocks of the next kernel may take places as these leave
            if (*abort_flag != 0u) {                                 // nothing may land in a block that has left
                issued = max(issued, early);
                for (uint32_t i = issued > L::kStages ? issued - L::kStages : 0u; i < issued; i++) {
                    mbar_drain(&full[i % L::kStages], (i / L::kStages) & 1u);
                }
            }
        }
    } else if (warp == 1u) {
        // ------------------------------------------------------------------------------- MMA
        if (elect_one()) {
            uint32_t s = 0u, ph = 0u, at = 0u, aph = 0u;
            bool ok = true;
            for (uint32_t w = first_item; ok && w < total; w += step) {
                const Item it = item_of(w);
                const uint32_t idesc = make_idesc_e4m3(kBlock, (it.rows + 15u) & ~15u);
                for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb++) {
                    if (!mbar_wait(&sum_empty[at], aph ^ 1u, abort_flag) || !mbar_wait(&full[s], ph, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t addr = smem_u32(base + s * L::kStageBytes), d = tmem + at * (kTiles * kRows);
                    const uint64_t rows = make_desc_sw128(addr + kTiles * L::kBTile);
#pragma unroll
                    for (uint32_t t = 0; t < kTiles; t++) {
                        const uint64_t lanes = make_desc_sw128(addr + t * L::kBTile);
#pragma unroll
                        for (uint32_t j = 0; j < 4u; j++) {
                            mma_e4m3_ss(d + t * kRows, lanes + 2u * j, rows + 2u * j, idesc, j != 0u);
                        }
                    }
                    mma_commit(&empty[s]);
                    mma_commit(&sum_full[at]);
                    if (++s == L::kStages) { s = 0u; ph ^= 1u; }
                    if (++at == 2u) { at = 0u; aph ^= 1u; }
                }
            }
            if (*abort_flag != 0u) {
                mma_commit(done);
                mbar_drain(done, 0u);
            }
        }
    } else if (warp == 2u && !kQuantize) {
        // --------------------------------------------------------------- factors, a slot at a time
        if (!kSplit && a.b_ready) pdl_wait();
        uint32_t slot = 0u, ph = 0u;
        bool ok = true;
        const uint32_t pitch = (blocks + 3u) & ~3u, b_blocks = blocks_of(a.n);
        for (uint32_t w = first_item; ok && w < total; w += step) {
            const Item it = item_of(w);
            if constexpr (kToken && kSplit) {
                for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb += L::kSlotBlocks) {
                    float f[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint32_t at = min(kb + i, it.kb_end - 1u), route = at / blocks, in = at - route * blocks;
                        const uint32_t group = ids_s[route];
                        f[i] = 0.f;
                        if (group < a.groups) {
                            f[i] = a.a_scales[(uint64_t)route * pitch + in] *
                                   a.b_scales[((uint64_t)group * b_blocks + it.column / kBlock) * blocks + in] * weights_s[route];
                        }
                    }
                    if (!mbar_wait(&factor_empty[slot], ph ^ 1u, abort_flag)) { ok = false; break; }
                    float *to = reinterpret_cast<float *>(base + L::kFactors) + slot * L::kSlotFloats;
                    if (lane < kRows) {
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) to[i * kRows + lane] = f[i];
                    }
                    mbar_arrive(&factor_full[slot]);
                    if (++slot == L::kSlots) { slot = 0u; ph ^= 1u; }
                }
                continue;
            }
            const bool valid = !kToken || it.group < a.groups;
            const uint64_t sb = ((uint64_t)(valid ? it.group : 0u) * b_blocks + it.column / kBlock) * blocks;
            const float *b_row[2] = {a.b_scales + sb, nullptr};
            if (kTiles == 2u) {
                b_row[1] = kEpilogue == kOutActivated ? a.b2_scales + sb
                           : it.column / kBlock + 1u < b_blocks ? b_row[0] + blocks : b_row[0];
            }
            for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb += L::kSlotBlocks) {
                float f[kTiles][4];
#pragma unroll
                for (uint32_t t = 0; t < kTiles; t++) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) f[t][i] = valid ? b_row[t][min(kb + i, blocks - 1u)] : 0.f;
                }
                float x[(kRows + 31u) / 32u][4];
#pragma unroll
                for (uint32_t j = 0; j < (kRows + 31u) / 32u; j++) {
                    // rows past the tile's take the last row's scales: their columns are not kept
                    const float *row = a.a_scales + (uint64_t)(kToken ? 0u : it.row + min(j * kWarp + lane, it.rows - 1u)) * pitch;
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) x[j][i] = row[min(kb + i, blocks - 1u)];
                }
                if (!mbar_wait(&factor_empty[slot], ph ^ 1u, abort_flag)) { ok = false; break; }
                float *to = reinterpret_cast<float *>(base + L::kFactors) + slot * L::kSlotFloats;
#pragma unroll
                for (uint32_t j = 0; j < (kRows + 31u) / 32u; j++) {
                    if (j * kWarp + lane >= kRows) continue;
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
#pragma unroll
                        for (uint32_t t = 0; t < kTiles; t++) to[(i * kTiles + t) * kRows + j * kWarp + lane] = x[j][i] * f[t][i];
                    }
                }
                mbar_arrive(&factor_full[slot]);
                if (++slot == L::kSlots) { slot = 0u; ph ^= 1u; }
            }
        }
    } else if (kQuantize && warp >= 4u + L::kSumWarps) {
        // ------------------ a's rows: a warp takes every fourth block of 128 columns, eight lanes a row's
        const Item it = item_of(0u);
        const uint32_t mine = warp - 4u - L::kSumWarps, in_pass = lane / 8u, first = lane % 8u * 16u;
        const float *sb = a.b_scales + (uint64_t)(it.column / kBlock) * blocks;
        for (uint32_t kb = it.kb_begin + mine; kb < it.kb_end; kb += L::kQuantizeWarps) {
            const uint32_t at = kb - it.kb_begin, s = at % L::kStages, slot = at % L::kSlots;
            uint32_t v[4][8];                                        // 16 bf16 of each of four rows
#pragma unroll
            for (uint32_t p = 0; p < 4u; p++) {
                const uint32_t row = p * 4u + in_pass, c = kb * kBlock + first;
                const uint16_t *from = a.x + (uint64_t)(it.row + row) * a.k + c;
#pragma unroll
                for (uint32_t h = 0; h < 2u; h++) {
                    uint4 q = make_uint4(0u, 0u, 0u, 0u);
                    if (a.x_vector) {
                        if (row < it.rows && c + h * 8u < a.k) q = *reinterpret_cast<const uint4 *>(from + h * 8u);
                    } else if (row < it.rows) {
                        uint32_t e[8];
#pragma unroll
                        for (uint32_t i = 0; i < 8u; i++) e[i] = c + h * 8u + i < a.k ? from[h * 8u + i] : 0u;
                        q = make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
                    }
                    v[p][h * 4u] = q.x; v[p][h * 4u + 1u] = q.y; v[p][h * 4u + 2u] = q.z; v[p][h * 4u + 3u] = q.w;
                }
            }
            const float by = sb[kb];
            if (!mbar_wait(&empty[s], (at / L::kStages & 1u) ^ 1u, abort_flag) ||
                !mbar_wait(&factor_empty[slot], (at / L::kSlots & 1u) ^ 1u, abort_flag)) {
                break;
            }
            unsigned char *to = base + s * L::kStageBytes + kTiles * L::kBTile;
            float *factors = reinterpret_cast<float *>(base + L::kFactors) + slot * L::kSlotFloats;
#pragma unroll
            for (uint32_t p = 0; p < 4u; p++) {
                if (p * 4u >= it.rows) break;                         // what rows past the end hold is not kept
                uint32_t most = 0u;
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) most = max(most, max((v[p][i] << 16) & 0x7fffffffu, v[p][i] & 0x7fff0000u));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float scale = scale_of(most), inverse = inverse_of(scale);
                uint32_t w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    const uint32_t x = v[p][2u * i], y = v[p][2u * i + 1u];
                    w[i] = codes2(quotient(bf16_lo(x), scale, inverse), quotient(bf16_hi(x), scale, inverse)) |
                           (codes2(quotient(bf16_lo(y), scale, inverse), quotient(bf16_hi(y), scale, inverse)) << 16);
                }
                const uint32_t row = p * 4u + in_pass;                // 128-byte rows, 16-byte units swizzled as TMA does
                *reinterpret_cast<uint4 *>(to + row * kBlock + ((lane % 8u) ^ (row % 8u)) * 16u) = make_uint4(w[0], w[1], w[2], w[3]);
                if (lane % 8u == 0u) factors[row] = scale * by;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0u) {
                mbar_arrive(&full[s]);
                mbar_arrive(&factor_full[slot]);
            }
        }
    } else if (warp >= 4u) {
        // --------------------------------------------------------------------------- running sums
        if (!kSplit && a.b_ready) pdl_wait();                        // before the first store
        constexpr uint32_t kMine = kRows < 32u ? kRows : 32u;         // rows of a per warp
        const uint32_t q = warp % 4u, half = (warp - 4u) / 4u;
        const uint32_t lanes = tmem + ((32u * q) << 16) + half * kMine;
        uint32_t at = 0u, aph = 0u, slot = 0u, sph = 0u, lph = 0u;
        bool ok = true;
        for (uint32_t w = first_item; ok && w < total; w += step) {
            const Item it = item_of(w);
            const uint32_t n = it.rows > half * kMine ? min(kMine, it.rows - half * kMine) : 0u;
            uint64_t sum[kTiles][kMine / 2u];
#pragma unroll
            for (uint32_t t = 0; t < kTiles; t++) {
#pragma unroll
                for (uint32_t j = 0; j < kMine / 2u; j++) sum[t][j] = 0ull;
            }
            for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb++) {
                const uint32_t in_slot = (kb - it.kb_begin) % L::kSlotBlocks;
                if ((in_slot == 0u && !mbar_wait(&factor_full[slot], sph, abort_flag)) || !mbar_wait(&sum_full[at], aph, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float *factors = reinterpret_cast<const float *>(base + L::kFactors) + slot * L::kSlotFloats +
                                       in_slot * kTiles * kRows + half * kMine;
                constexpr uint32_t kChunks = kMine / 16u;
                uint32_t r[kTiles][kChunks][16];
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++) {
                    if (c * 16u < n) {
#pragma unroll
                        for (uint32_t t = 0; t < kTiles; t++) tmem_ld_32x16(lanes + at * (kTiles * kRows) + t * kRows + c * 16u, r[t][c]);
                    }
                }
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++) {
#pragma unroll
                    for (uint32_t t = 0; t < kTiles; t++) tmem_ld_wait_for(r[t][c]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0u) mbar_arrive(&sum_empty[at]);
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++) {
                    if (c * 16u < n) {
#pragma unroll
                        for (uint32_t t = 0; t < kTiles; t++) {
                            const ulonglong2 *f = reinterpret_cast<const ulonglong2 *>(factors + t * kRows + c * 16u);
#pragma unroll
                            for (uint32_t j = 0; j < 4u; j++) {
                                const ulonglong2 v = f[j];
                                uint64_t *to = &sum[t][c * 8u + j * 2u];
                                to[0] = fma2(pack2(r[t][c][4u * j], r[t][c][4u * j + 1u]), v.x, to[0]);
                                to[1] = fma2(pack2(r[t][c][4u * j + 2u], r[t][c][4u * j + 3u]), v.y, to[1]);
                            }
                        }
                    }
                }
                if (++at == 2u) { at = 0u; aph ^= 1u; }
                if (in_slot == L::kSlotBlocks - 1u || kb + 1u == it.kb_end) {
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&factor_empty[slot]);
                    if (++slot == L::kSlots) { slot = 0u; sph ^= 1u; }
                }
            }
            if (!ok) break;
            const uint32_t column = 32u * q + lane;                  // of the tile
            auto value = [&](uint32_t t, uint32_t j) { return j & 1u ? hi2(sum[t][j / 2u]) : lo2(sum[t][j / 2u]); };
            if (kSplit) {
                float *part = reinterpret_cast<float *>(base);       // [kRows][128]; every stage has been read
#pragma unroll
                for (uint32_t j = 0; j < kMine; j++) {
                    if (j < n) part[(half * kMine + j) * kBlock + column] = value(0u, j);
                }
            } else if (kEpilogue == kOutActivated) {
                // ---------------------------------- activation, largest of a row's 128 columns, codes
                const bool inside = it.column + column < a.n;
                uint32_t *largest = reinterpret_cast<uint32_t *>(base + L::kLargest) + half * kMine;   // [4][kRows]
                float act[kMine];
                auto activate = [&](auto f) {
#pragma unroll
                    for (uint32_t j = 0; j < kMine; j++) act[j] = j < n && inside ? f(value(0u, j), value(kTiles - 1u, j)) : 0.f;
                };
                if (a.activation == kActSitu) activate(ExpertActivation<true>{a.beta, a.by_beta, a.linear_beta, a.by_linear_beta});
                else activate(ExpertActivation<false>{});
#pragma unroll
                for (uint32_t j = 0; j < kMine; j++) {
                    if (j < n) {
                        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(act[j]) & 0x7fffffffu);
                        if (lane == 0u) largest[q * kRows + j] = most;
                    }
                }
                __syncwarp();
                if (lane == 0u) mbar_arrive(&largest_full[half]);
                if (!mbar_wait(&largest_full[half], lph, abort_flag)) { ok = false; break; }
                lph ^= 1u;
                const uint32_t out_pitch = pitch_of(a.n), scale_pitch = scale_pitch_of(a.n);
#pragma unroll
                for (uint32_t j = 0; j < kMine; j++) {
                    if (j < n) {
                        const uint32_t most = max(max(largest[j], largest[kRows + j]), max(largest[2u * kRows + j], largest[3u * kRows + j]));
                        const float scale = scale_of(most);
                        const uint64_t row = it.row + half * kMine + j;
                        if (q == 0u && lane == 0u) a.out_scales[row * scale_pitch + it.column / kBlock] = scale;
                        if (it.column + column < out_pitch) {
                            ((uint8_t *)a.out)[row * out_pitch + it.column + column] =
                                (uint8_t)codes2(quotient(act[j], scale, inverse_of(scale)), 0.f);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0u) mbar_arrive(&largest_full[half]);     // read: the next item may overwrite it
                if (!mbar_wait(&largest_full[half], lph, abort_flag)) { ok = false; break; }
                lph ^= 1u;
            } else {
#pragma unroll
                for (uint32_t t = 0; t < kTiles; t++) {
                    const uint32_t c = it.column + t * kBlock + column;
                    if (c < a.n) {
#pragma unroll
                        for (uint32_t j = 0; j < kMine; j++) {
                            if (j < n) {
                                ((float *)a.out)[(uint64_t)(it.row + half * kMine + j) * a.n + c] = value(t, j);
                            }
                        }
                    }
                }
            }
        }
    }

    if (kSplit) {
        // the parts' sums, in ascending order of the depth; each block adds its share of the item
        __syncthreads();
        cluster_barrier();
        const Item it = item_of(0u);
        const uint32_t size = cluster_size(), all = it.rows * (kBlock / 4u);        // four columns at a time
        const uint32_t share = (all + size - 1u) / size, begin = cluster_rank() * share, end = min(all, begin + share);
        const float *part = reinterpret_cast<const float *>(base);
        const bool vector = a.n % 4u == 0u && ((uintptr_t)a.out & (kEpilogue == kOutF32 ? 15u : 7u)) == 0u;
        for (uint32_t e = begin + threadIdx.x; e < end; e += L::kThreads) {
            float4 v[kMaxSplits];
#pragma unroll
            for (uint32_t r = 0; r < kMaxSplits; r++) v[r] = r < size ? cluster_load4(part + e * 4u, r) : make_float4(0.f, 0.f, 0.f, 0.f);
            float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (uint32_t r = 1; r < kMaxSplits; r++) {
                if (r < size) {
                    sum[0] += v[r].x;
                    sum[1] += v[r].y;
                    sum[2] += v[r].z;
                    sum[3] += v[r].w;
                }
            }
            const uint32_t c = it.column + e % (kBlock / 4u) * 4u;
            if (c >= a.n) continue;
            const uint64_t to = (uint64_t)(it.row + e / (kBlock / 4u)) * a.n + c;
            if (kEpilogue == kOutF32) {
                float *out = (float *)a.out + to;
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) {
                    if (a.accumulate && c + j < a.n) sum[j] += out[j];
                }
                if (vector) {
                    *reinterpret_cast<float4 *>(out) = make_float4(sum[0], sum[1], sum[2], sum[3]);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        if (c + j < a.n) out[j] = sum[j];
                    }
                }
            } else {
                uint16_t *out = (uint16_t *)a.out + to;
                if (kToken && a.shared) {                             // added as k3_moe_combine does
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        if (c + j < a.n) {
                            sum[j] = bf16_bits_to_float(float_to_bf16_bits(sum[j])) + bf16_bits_to_float(a.shared[c + j]);
                        }
                    }
                }
                if (vector) {
                    *reinterpret_cast<uint2 *>(out) = make_uint2(bf16x2(sum[0], sum[1]), bf16x2(sum[2], sum[3]));
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        if (c + j < a.n) out[j] = float_to_bf16_bits(sum[j]);
                    }
                }
            }
        }
        cluster_barrier();                                           // nobody leaves while its sums are read
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0u) atomicOr(&g_fp8_few_status, 1u);
    if (warp == 1u) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kTmem);
    }
}

FewArgs args_of(const Product &p) {
    FewArgs a{};
    a.out = p.out;
    a.out_scales = (float *)p.out_scales;
    a.a_scales = (const float *)p.a_scales;
    a.b_scales = (const float *)p.b_scales;
    a.b2_scales = (const float *)p.b2_scales;
    a.offsets = p.offsets;
    a.ids = p.ids;
    a.weights = p.weights;
    a.shared = (const uint16_t *)p.shared;
    a.top_k = p.top_k;
    a.groups = p.groups;
    a.rows = p.rows;
    a.n = p.n;
    a.k = p.k;
    a.accumulate = p.accumulate;
    a.activation = p.activation;
    a.beta = p.beta;
    a.linear_beta = p.linear_beta;
    a.by_beta = 1.0f / p.beta;
    a.by_linear_beta = 1.0f / p.linear_beta;
    return a;
}

template <int kEpilogue, bool kQuantize, bool kToken = false>
bool launch_split(const Product &p, const void *x, cudaStream_t stream) {
    constexpr uint32_t kRows = few_linear_rows;
    using L = Layout<1, kRows, true, kQuantize>;
    CUtensorMap a_map{}, b_map;
    if ((!kQuantize && !map_codes(&a_map, p.a, kToken ? p.top_k : p.rows, p.k, kBoxRows)) ||
        !map_codes(&b_map, p.b, (uint64_t)p.groups * p.n, p.k, kBlock)) {
        return false;
    }
    FewArgs a = args_of(p);
    a.x = (const uint16_t *)x;
    a.x_vector = aligned16(x) && p.k % 8u == 0u;
    a.b_ready = p.b_ready && !kQuantize;
    const uint32_t tiles = blocks_of(p.n), row_tiles = (p.rows + kRows - 1u) / kRows;
    const uint32_t blocks = blocks_of(p.k) * (kToken ? p.top_k : 1u);
    if (tiles > 65535u || row_tiles > 65535u) return false;
    auto kernel = fp8_few_kernel<kEpilogue, 1, kRows, true, kQuantize, kToken>;
    if (!set_max_dynamic_smem((const void *)kernel, L::kBytes)) return false;
    // a launch, the first loads and the sums' way through the cluster take as long as 8 steps
    const uint32_t parts = best_parts((uint64_t)tiles * row_tiles, blocks, 1u, 8u,
                                      active_clusters((const void *)kernel, L::kThreads, L::kBytes));
    a.split_blocks = (blocks + parts - 1u) / parts;
    return launch_chained_cluster(kernel, dim3(parts, tiles, row_tiles), L::kThreads, dim3(parts, 1, 1), L::kBytes, stream, a_map,
                                  b_map, b_map, a);
}

template <int kEpilogue, bool kToken = false>
bool launch_grouped(const Product &p, cudaStream_t stream) {
    constexpr uint32_t kRows = kToken ? 16u : kGroupRows, kColumns = kEpilogue == kOutActivated ? kBlock : 2u * kBlock;
    using L = Layout<2, kRows, false, false>;
    CUtensorMap a_map, b_map, b2_map;
    const uint64_t b_rows = (uint64_t)p.groups * p.n;
    if (!map_codes(&a_map, p.a, p.rows, p.k, kBoxRows) || !map_codes(&b_map, p.b, b_rows, p.k, kBlock) ||
        !map_codes(&b2_map, kEpilogue == kOutActivated ? p.b2 : p.b, b_rows, p.k, kBlock)) {
        return false;
    }
    FewArgs a = args_of(p);
    a.b_ready = p.b_ready;
    a.column_items = (p.n + kColumns - 1u) / kColumns;
    const uint64_t items = (kToken ? p.top_k : (uint64_t)(p.rows + kRows - 1u) / kRows + p.groups) * a.column_items;
    if (items > 0x7fffffffull) return false;
    auto kernel = fp8_few_kernel<kEpilogue, 2, kRows, false, false, kToken>;
    return set_max_dynamic_smem((const void *)kernel, L::kBytes) &&
           launch_chained(kernel, (uint32_t)std::min<uint64_t>(items, sm_count()), L::kThreads, L::kBytes, stream, a_map, b_map,
                          b2_map, a);
}

}  // namespace

bool k3::fp8::few_product(const Product &p, cudaStream_t stream) {
    if (p.offsets) return p.epilogue == kOutActivated ? launch_grouped<kOutActivated>(p, stream) : launch_grouped<kOutF32>(p, stream);
    return p.epilogue == kOutF32 ? launch_split<kOutF32, false>(p, nullptr, stream) : launch_split<kOutBf16, false>(p, nullptr, stream);
}

bool k3::fp8::token_gateup(const Product &p, cudaStream_t stream) { return launch_grouped<kOutActivated, true>(p, stream); }

bool k3::fp8::token_down(const Product &p, cudaStream_t stream) {
    return launch_split<kOutBf16, false, true>(p, nullptr, stream);
}

bool k3::fp8::few_linear(const Product &p, const void *x_bf16, cudaStream_t stream) {
    return launch_split<kOutBf16, true>(p, x_bf16, stream);
}

uint32_t k3_fp8_few_status() {
    uint32_t v = 0xffffffffu;
    if (cudaMemcpyFromSymbol(&v, g_fp8_few_status, sizeof(v)) != cudaSuccess) (void)cudaGetLastError();
    return v;
}

bool k3_fp8_few_status_clear() {
    const uint32_t zero = 0u;
    const bool ok = cudaMemcpyToSymbol(g_fp8_few_status, &zero, sizeof(zero)) == cudaSuccess;
    if (!ok) (void)cudaGetLastError();
    return ok;
}
