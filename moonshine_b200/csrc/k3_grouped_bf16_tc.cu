// bf16 products grouped by expert, and their gradients, on tcgen05 (kind::f16).
//
// D[m, c] = sum_r A(m, r) B(c, r), the tensor cores' 128 lanes along m:
//   forward    A = w_g   [n, k], m a feature of the output, c a row of the group, r < k
//   by input   A = w_g^T [k, n], m a feature of the input,  c a row of the group, r < n
//   by weight  A = dy^T  [n, rows], B = x^T [k, rows],      r a row of the group
// A group's rows are the N extent of the first two, which takes any multiple of 16 (pairs of blocks: 32): a group of 130
// rows costs a tile of 144, where rows as lanes would cost 256.  What lies in memory with its depth in neighbouring rows
// (w by input, both operands by weight) goes to shared memory as it is and is read "MN-major".
//
// An item is kHalves x 128 lanes by up to kMaxN columns over the whole depth, 64 of it per stage.  One block per SM:
//   warp 0       loads by TMA
//   warp 1       MMA issuer, owns the tensor memory: two accumulators of kMaxN columns, for the item's two halves or, where
//                it has one, for two items in turn
//   warp 2       draws items from a counter and tells the others, when the loads of the one before come to an end
//                by weight beside a kernel that takes the small groups: every gridDim-th item, where its group is another
//   warp 3       by weight: clears what a group's first stage holds of the rows behind its part of the group
//   warps 4-11   results: lane quadrant warp % 4, every second chunk of 32 columns; the accumulator is free again once
//                it is in registers, before anything is stored
// Items that share a matrix are neighbours in the order, so it is in L2 for all but one of them.  Their results do not
// depend on who draws what.
//
// kCtas 2: a pair of blocks (cta_group::2) shares an item of twice the lanes.  Each loads its lanes and half of the columns,
// which both tensor cores read, so the columns come from L2 once for two SMs; the first block draws, waits and issues.
// A release across the pair waits for the stores of the warp that does it (the weight's gradient of 32 groups of 128 rows, in pairs,
// took 409 us so and 318 without), so warps that store do none.  That the second block's have read an item they tell its warp 2,
// which has no stores and hands it on.  That they have read an accumulator needs no release: what follows it are tcgen05
// operations alone, ordered by tcgen05.wait::ld and the tcgen05 fences on both sides of the arrival.
// kSplit: a cluster of up to eight blocks shares an item's depth and adds its sums through distributed shared memory.
//
// What bounds it.  Large calls: power, and what the last of a group's column tiles leaves empty.  64 groups of 512 rows, 2048 x
// 7168, bf16 forward, 20 in a row after a pause: 676 to 712 us on two B200s = 1350 to 1420 TFLOP/s; for four seconds 854 us = 1130 at
// 989 W and 1065 MHz (the library's plain product of 32768 rows: 1350 TFLOP/s at 993 W and 1312 MHz; it reads 0.5 GB where 64
// matrices are 2.3).  64 groups of 520 rows, which take a third tile, 814 us, of 560 818, of 640 921.  Few rows per group: the
// matrices' bytes, 6.2 to 6.9 TB/s.
//
// Every wait is bounded; on give-up the block raises the status word, waits for its copies and frees its tensor memory.
#include "k3_fp8_ptx.cuh"
#include "k3_grouped.h"
#include "k3_grouped_bf16.h"

#include <algorithm>
#include <cmath>

using namespace k3;
using namespace k3::tc;
using namespace k3::gb;
using k3::fp8::bf16x2;
using k3::fp8::fewer_registers;
using k3::fp8::more_registers;
using k3::fp8::mbar_drain;
using k3::fp8::tensor_map_encoder;

namespace {

constexpr uint32_t kThreads = 384, kResultWarps = 8, kDepth = 64;      // depth of a stage: 128 bytes of bf16
constexpr uint32_t kBox = 64 * kDepth * 2;                             // 8 KB: 64 x 64 elements
constexpr uint32_t kSlots = 4;                                         // items that are known ahead
constexpr uint32_t kMaxParts = 8;                                      // of an item's depth: the portable cluster
constexpr uint32_t kAhead = 6;                                         // stages before an item's last in which the next is drawn
constexpr uint32_t kNoItem = 0xffffffffu;

__device__ uint32_t g_grouped_bf16_status = 0;

// What the kernel in front leaves in the workspace: the counter, the number of row tiles, and of each row tile its
// group, rows, and its group's tiles.
struct Plan {
    uint32_t counter, tiles, pad[2];
};
struct Tile {
    uint32_t group, row, rows, first, count, pad[3];                   // first .. first + count - 1: the group's tiles
};

template <uint32_t kCtas_, uint32_t kHalves_, uint32_t kMaxN_, uint32_t kStages_, bool kSplit_ = false>
struct Shape {
    static constexpr bool kSplit = kSplit_;
    static constexpr uint32_t kCtas = kCtas_, kHalves = kHalves_, kMaxN = kMaxN_, kStages = kStages_;
    static constexpr uint32_t kHalf = 128u * kCtas, kLanes = kHalf * kHalves;
    static constexpr uint32_t kStep = 16u * kCtas;                     // of an MMA's columns
    static constexpr uint32_t kA = kHalves * 2u * kBox, kStage = kA + kMaxN / kCtas * kDepth * 2u;
    static constexpr uint32_t kStore = kStages * kStage;               // 4 KB per result warp
    static constexpr uint32_t kBars = kStore + kResultWarps * 4096u;
    static constexpr uint32_t kBytes = kBars + 512u + 1024u;           // the last: alignment
    static constexpr uint32_t kTmem = 2u * kMaxN;
    // barriers, items, and two words
    static_assert((4u * kStages + 4u + 3u * kSlots + 2u) * 8u + kSlots * 24u + 8u <= 512u, "");
    static_assert(!kSplit || (kCtas == 1u && kLanes * kMaxN * 4u <= kResultWarps * 4096u), "a part's sums take the stores' place");
    static_assert(kBytes <= 232448u && kTmem <= 512u && (kTmem & (kTmem - 1u)) == 0u, "");
};

struct TcArgs {
    void *out;
    const uint32_t *offsets;
    Plan *plan;
    Tile *tiles;
    uint32_t rows, groups, n, k;
    uint32_t lane_tiles;                                               // items side by side along the lanes
    uint32_t column_tiles;                                             // by weight: and along the columns
    uint32_t batch;                                                    // items per draw
    bool single;                                                       // an item per block at most: no plan, nothing is drawn
    uint32_t least;                                                    // by weight: groups of fewer rows are left out
    int accumulate;
};

struct Item {
    uint32_t group, row, rows;                                         // by weight: the group's rows, all of them
    uint32_t lane0, column0;                                           // by weight: column0 of k
    uint32_t draw;                                                     // 1: the last one drawn
};
static_assert(sizeof(Item) == 24u, "what Shape leaves room for");

// Instruction descriptor, kind::f16, as make_idesc_bf16, with bits 15 and 16 for operands whose depth is not what lies
// side by side.
K3_DEVINL constexpr uint32_t idesc_of(uint32_t m, uint32_t n, bool a_by_depth, bool b_by_depth) {
    return make_idesc_bf16(m, n) | (a_by_depth ? 1u << 15 : 0u) | (b_by_depth ? 1u << 16 : 0u);
}
// Shared-memory descriptor of a tile whose rows are its depth: boxes of 64 elements x 64 rows of 128 bytes with the
// 128-byte swizzle, 8 KB apart (the leading offset); groups of 8 rows are 1024 bytes apart (the stride offset).
K3_DEVINL uint64_t make_desc_by_depth(uint32_t smem_addr) {
    return (make_desc_sw128(smem_addr) & ~((uint64_t)0x3fffu << 16)) | ((uint64_t)(kBox >> 4) << 16);
}

// ------------------------------------------------------------------- what a pair of blocks adds
// The place of `p` in the shared memory of block `rank` of the cluster.
K3_DEVINL uint32_t place_in(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
K3_DEVINL void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// The same between tcgen05.fence::before_thread_sync here and ::after_thread_sync there, which order tcgen05 operations; nothing
// else is ordered by it.
K3_DEVINL void arrive_relaxed_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
K3_DEVINL void store_at(uint32_t to, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory"); }
// mbar_wait for arrivals from the other block
K3_DEVINL bool wait_cluster(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag) {
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t spin = 1;; spin++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((spin & 63u) == 0u) {
            if (*abort_flag != 0u) return false;
            if (global_timer_ns() - t0 > kWaitLimitNs) break;
        }
    }
    *abort_flag = 1u;
    return false;
}

// Loads of 2 and 3 dimensions.  kCtas 2: `bar` is the first block's barrier, wherever the copy goes.
template <uint32_t kCtas>
K3_DEVINL void load_2d(void *dst, const void *map, uint32_t bar, int32_t x, int32_t y) {
    if constexpr (kCtas == 2u) {
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(bar), "r"(x), "r"(y)
            : "memory");
    } else {
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
                     "l"(map), "r"(bar), "r"(x), "r"(y)
                     : "memory");
    }
}
template <uint32_t kCtas>
K3_DEVINL void load_3d(void *dst, const void *map, uint32_t bar, int32_t x, int32_t y, int32_t z) {
    if constexpr (kCtas == 2u) {
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    } else {
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                         smem_u32(dst)),
                     "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
                     : "memory");
    }
}
template <uint32_t kCtas>
K3_DEVINL void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kCtas == 2u) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        mma_f16_ss(d, a, b, idesc, accumulate);
    }
}
// `bar`, of both blocks, once every MMA issued so far has run
template <uint32_t kCtas>
K3_DEVINL void commit(uint64_t *bar) {
    if constexpr (kCtas == 2u) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    } else {
        mma_commit(bar);
    }
}
template <uint32_t kCtas>
K3_DEVINL void alloc_tmem(uint32_t *slot, uint32_t columns) {
    if constexpr (kCtas == 2u) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(slot, columns);
        tmem_relinquish();
    }
}
template <uint32_t kCtas>
K3_DEVINL void free_tmem(uint32_t tmem, uint32_t columns) {
    if constexpr (kCtas == 2u) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else tmem_dealloc(tmem, columns);
}

// ------------------------------------------------------------------------------------------- the plan
// Tile i of a group's `count`: as few as there can be of up to max_n rows, equally large but for one step.
K3_DEVINL Tile tile_of(uint32_t group, uint32_t begin, uint32_t end, uint32_t first, uint32_t count, uint32_t i, uint32_t step) {
    const uint32_t steps = (end - begin + step - 1u) / step, each = steps / count, more = steps - each * count;
    const uint32_t row = begin + (each * i + min(i, more)) * step;
    return Tile{group, row, min((each + (i < more ? 1u : 0u)) * step, end - row), first, count, {}};
}

// A call with an item for every block at most and up to kSearched groups needs no plan: a warp looks its item up.  The tile
// that item w of lane_tiles per tile belongs to, its place along the lanes in `lane_tile`; false past the last.
constexpr uint32_t kSearched = 128;
K3_DEVINL bool search_tile(const uint32_t *offsets, uint32_t rows, uint32_t groups, uint32_t max_n, uint32_t step, uint32_t w,
                           uint32_t lane_tiles, Tile &tile, uint32_t &lane_tile) {
    constexpr uint32_t kEach = kSearched / kWarp;
    const uint32_t lane = threadIdx.x % kWarp, t = w / lane_tiles;
    uint32_t begin[kEach], end[kEach], sum = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t g = lane * kEach + i;
        begin[i] = end[i] = 0u;
        if (g < groups) group_rows(offsets, g, rows, begin[i], end[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) sum += (end[i] - begin[i] + max_n - 1u) / max_n;
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= (uint32_t)o) scan += up;
    }
    uint32_t first = scan - sum;
    const uint32_t holder = __ballot_sync(0xffffffffu, t >= first && t < scan);
    if (holder == 0u) return false;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t count = (end[i] - begin[i] + max_n - 1u) / max_n;
        if (t >= first && t < first + count) {
            const uint32_t local = w - first * lane_tiles;
            tile = tile_of(lane * kEach + i, begin[i], end[i], first, count, local % count, step);
            lane_tile = local / count;
        }
        first += count;
    }
    const uint32_t from = __ffs(holder) - 1u;
    tile.group = __shfl_sync(0xffffffffu, tile.group, from);
    tile.row = __shfl_sync(0xffffffffu, tile.row, from);
    tile.rows = __shfl_sync(0xffffffffu, tile.rows, from);
    lane_tile = __shfl_sync(0xffffffffu, lane_tile, from);
    return true;
}

// One thread per group.  Tiles are counted in 64 bits: overlapping groups, where offsets descend, can have more than 2^32, and a
// place that wrapped would be another group's.
__global__ void __launch_bounds__(kMaxGroups) grouped_plan_kernel(Plan *plan, Tile *tiles, const uint32_t *offsets, uint32_t rows,
                                                                  uint32_t groups, uint32_t max_n, uint32_t step, uint32_t capacity) {
    pdl_trigger();
    pdl_wait();
    __shared__ uint64_t sums[kMaxGroups / kWarp];
    const uint32_t g = threadIdx.x, lane = g % kWarp, warp = g / kWarp;
    uint32_t begin = 0u, end = 0u;
    if (g < groups) group_rows(offsets, g, rows, begin, end);
    const uint32_t count = (end - begin + max_n - 1u) / max_n;
    uint64_t scan = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= (uint32_t)o) scan += up;
    }
    if (lane == 31u) sums[warp] = scan;
    __syncthreads();
    uint64_t first = scan - count;
    for (uint32_t w = 0; w < warp; w++) first += sums[w];
    if (count != 0u) {
        const uint32_t held = first < capacity ? min(count, capacity - (uint32_t)first) : 0u;
        for (uint32_t i = 0; i < held; i++) {
            Tile t = tile_of(g, begin, end, (uint32_t)first, count, i, step);
            t.count = held;                                            // (fewer only if offsets descend)
            tiles[first + i] = t;
        }
    }
    if (g == kMaxGroups - 1u) {
        plan->counter = 0u;
        plan->tiles = (uint32_t)min(first + count, (uint64_t)capacity);
    }
}

// by weight: no row tiles
__global__ void grouped_counter_kernel(Plan *plan) {
    pdl_trigger();
    pdl_wait();
    plan->counter = 0u;
}

// ---------------------------------------------------------------------------------------- the product
template <int kForm, bool kF32, typename S>
__global__ void __launch_bounds__(kThreads, 1)
grouped_bf16_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, TcArgs a) {
    constexpr bool kRows = kForm != kByWeight;                         // the columns are rows of the group
    constexpr bool kADepth = kForm != kForward, kBDepth = kForm == kByWeight;
    constexpr uint32_t kCtas = S::kCtas;
    // The tensor cores cut the sums off instead of rounding them, 2^-24 or so of the sum per 16 of the depth, always towards
    // zero: 8e-6 of the result's norm at a depth of 7168.  For f32 results an accumulator therefore takes up to 8 blocks, a
    // segment, and the warps behind it add the segments, rounded: 4.8e-7 at any depth (16 blocks 1.0e-6, 4 2.5e-7).  64 groups of 512
    // rows, 2048 x 7168, in pairs of blocks with one half (Square), 20 in a row: forward 767 us (16 blocks 762, 4 781, without segments
    // 750), by input 821 (818, 857, 810).  Two halves, whose sums no registers would hold, have none; Wide takes 731 us forward.
    constexpr uint32_t kSegment = kF32 && S::kHalves == 1u ? 8u : 0xffffffffu;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(base + S::kBars);    // [kStages]
    uint64_t *empty = full + S::kStages;                               // [kStages]
    uint64_t *acc_full = empty + S::kStages;                           // [2]
    uint64_t *acc_empty = acc_full + 2;                                // [2]
    uint64_t *item_full = acc_empty + 2;                               // [kSlots]
    uint64_t *item_empty = item_full + kSlots;                         // [kSlots]
    uint64_t *wanted = item_empty + kSlots;                            // [1] the loads come to an end
    uint64_t *armed = wanted + 1;                                      // [kStages] a stage that has to be cleared is being loaded
    uint64_t *cleared = armed + S::kStages;                            // [kStages] and its rows behind the group are zeros
    uint64_t *done = cleared + S::kStages;                             // [1] every MMA issued has run
    uint64_t *item_read_here = done + 1;                               // [kSlots] the second block of a pair: its warps have read it
    Item *items = reinterpret_cast<Item *>(item_read_here + kSlots);   // [kSlots]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(items + kSlots);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    const uint32_t warp = warp_index(), lane = threadIdx.x % kWarp;
    const uint32_t rank = kCtas == 2u ? cluster_rank() : 0u;           // the first of a pair issues its MMAs and draws its items
    // the extent along the lanes, the depth, and the output's row length
    const uint32_t lanes = kForm == kByInput ? a.k : a.n;

    if (warp == 0u && elect_one()) {
        *abort_flag = 0u;
        for (uint32_t s = 0; s < S::kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&armed[s], 1);
            mbar_init(&cleared[s], 1);
        }
        for (uint32_t s = 0; s < 2u; s++) {
            mbar_init(&acc_full[s], 1);
            mbar_init(&acc_empty[s], kResultWarps * kCtas);
        }
        for (uint32_t s = 0; s < kSlots; s++) {
            mbar_init(&item_full[s], 1);
            // the MMAs', the loads', the results' and the clearing warp; of a second block the one that hands on
            mbar_init(&item_empty[s], 2u + kResultWarps + (kRows ? 0u : 1u) + (kCtas - 1u));
            mbar_init(&item_read_here[s], 1u + kResultWarps);
        }
        mbar_init(wanted, 1);
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
    }
    if (warp == 1u) alloc_tmem<kCtas>(tmem_slot, S::kTmem);
    tc_fence_before();
    __syncthreads();
    if (kCtas == 2u) cluster_barrier();                                // the other block's barriers are there
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    // for arrivals that may come from the other block
    auto wait_at = [&](uint64_t *bar, uint32_t phase) {
        return kCtas == 2u ? wait_cluster(bar, phase, abort_flag) : mbar_wait(bar, phase, abort_flag);
    };
    // Items one after the other, as every role reads them.
    uint32_t slot = 0u, slot_phase = 0u;
    auto next_item = [&](Item &it) {
        if (!wait_at(&item_full[slot], slot_phase)) return false;
        it = items[slot];
        return it.group != kNoItem;
    };
    // by one thread of a warp that has read an accumulator
    auto accumulator_read = [&](uint32_t acc) {
        if (kCtas == 2u) arrive_relaxed_at(place_in(&acc_empty[acc], 0u));
        else mbar_arrive(&acc_empty[acc]);
    };
    // by one thread of a warp that has read the item
    auto item_read = [&]() { mbar_arrive(rank == 0u ? &item_empty[slot] : &item_read_here[slot]); };
    auto item_done = [&]() {
        if (++slot == kSlots) { slot = 0u; slot_phase ^= 1u; }
    };
    // blocks of the depth: all, or the part of a cluster's block
    const uint32_t split = S::kSplit ? cluster_rank() : 0u, splits = S::kSplit ? cluster_size() : 1u;
    auto range_of = [&](uint32_t blocks, uint32_t &begin, uint32_t &end) {
        const uint32_t each = (blocks + splits - 1u) / splits;
        begin = min(split * each, blocks);
        end = min(begin + each, blocks);
    };
    auto depth_of = [&](const Item &it) { return kForm == kForward ? a.k : kForm == kByInput ? a.n : it.rows; };
    // by weight: the rows of the first block, so that those behind it are whole, and what is behind the group's rows is
    // cleared while the products of the item before still run
    auto first_rows = [](uint32_t depth) { return (depth - 1u) % kDepth + 1u; };
    auto halves_of = [&](const Item &it) { return min(S::kHalves, (lanes - it.lane0 + S::kHalf - 1u) / S::kHalf); };
    auto columns_of = [&](const Item &it) { return kRows ? it.rows : min(S::kMaxN, a.k - it.column0); };
    // of an MMA, and how many of them this block holds
    auto steps_of = [&](uint32_t columns) { return (columns + S::kStep - 1u) / S::kStep * S::kStep; };
    auto boxes_of = [&](uint32_t columns) { return (steps_of(columns) / kCtas + (kRows ? 31u : 63u)) / (kRows ? 32u : 64u); };

    // an accumulator half in registers is 128 of them: 2 x 128 x 232 + 128 x 40 are the 384 x 168 of the launch
    constexpr bool kShares = S::kMaxN == 256u;
    if (kShares && warp < 4u) fewer_registers<40>();
    if (warp == 0u) {
        // ----------------------------------------------------------------------------- loads
        if (elect_one()) {
            uint32_t s = 0u, ph = 0u, issued = 0u;
            bool ok = true;
            Item it;
            while (ok && next_item(it)) {
                item_read();
                item_done();
                const uint32_t halves = halves_of(it), columns = columns_of(it);
                uint32_t begin, end;
                range_of((depth_of(it) + kDepth - 1u) / kDepth, begin, end);
                const uint32_t b_boxes = boxes_of(columns), b_first = rank * (steps_of(columns) / kCtas);
                const uint32_t bytes = halves * 2u * kBox + b_boxes * (kRows ? kBox / 2u : kBox);
                if (rank == 0u && it.draw != 0u && end - begin <= kAhead) mbar_arrive(wanted);
                for (uint32_t kb = begin; kb < end; kb++) {
                    if (rank == 0u && it.draw != 0u && kb + kAhead == end - 1u) mbar_arrive(wanted);
                    if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) { ok = false; break; }
                    unsigned char *at = base + s * S::kStage, *bt = at + S::kA;
                    const int32_t d = (int32_t)(kRows || kb == 0u ? kb * kDepth : first_rows(it.rows) + (kb - 1u) * kDepth), r = (int32_t)it.row;
                    if (rank == 0u) mbar_arrive_expect_tx(&full[s], bytes * kCtas);
                    const uint32_t bar = kCtas == 2u ? place_in(&full[s], 0u) : smem_u32(&full[s]);
                    for (uint32_t h = 0; h < halves; h++) {
                        const int32_t l = (int32_t)(it.lane0 + S::kHalf * h + 128u * rank);
                        unsigned char *to = at + h * 2u * kBox;
                        if (kForm == kForward) {
                            load_3d<kCtas>(to, &map_a, bar, d, l, (int32_t)it.group);
                        } else if (kForm == kByInput) {
                            load_3d<kCtas>(to, &map_a, bar, l, d, (int32_t)it.group);
                            load_3d<kCtas>(to + kBox, &map_a, bar, l + 64, d, (int32_t)it.group);
                        } else {
                            load_2d<kCtas>(to, &map_a, bar, l, r + d);
                            load_2d<kCtas>(to + kBox, &map_a, bar, l + 64, r + d);
                        }
                    }
                    for (uint32_t b = 0; b < b_boxes; b++) {
                        if (kRows) load_2d<kCtas>(bt + b * (kBox / 2u), &map_b, bar, d, r + (int32_t)(b_first + 32u * b));
                        else load_2d<kCtas>(bt + b * kBox, &map_b, bar, (int32_t)(it.column0 + b_first + 64u * b), r + d);
                    }
                    if (!kRows && kb == 0u && it.rows % 16u != 0u) mbar_arrive(&armed[s]);
                    issued++;
                    if (++s == S::kStages) { s = 0u; ph ^= 1u; }
                }
            }
            pdl_trigger();                                             // the blocks of the next kernel may take places as these leave
            if (rank == 0u && *abort_flag != 0u) {                     // nothing may land in a block that has left
                for (uint32_t i = issued > S::kStages ? issued - S::kStages : 0u; i < issued; i++) {
                    mbar_drain(&full[i % S::kStages], (i / S::kStages) & 1u);
                }
            }
        }
    } else if (warp == 1u) {
        // ------------------------------------------------------------------------------- MMA
        if (rank == 0u && elect_one()) {
            uint32_t s = 0u, ph = 0u, clear_phases = 0u, turn = 0u, acc_phase[2] = {1u, 1u};
            bool ok = true;
            Item it;
            while (ok && next_item(it)) {
                item_read();
                item_done();
                const uint32_t depth = depth_of(it), halves = halves_of(it);
                uint32_t begin, end;
                range_of((depth + kDepth - 1u) / kDepth, begin, end);
                const uint32_t idesc = idesc_of(S::kHalf, steps_of(columns_of(it)), kADepth, kBDepth);
                // by weight: the first block has what does not fill one, in the steps of 16 that it takes
                const uint32_t first_steps = kRows ? 4u : (first_rows(depth) + 15u) / 16u;
                auto free = [&](uint32_t acc) {
                    const bool is = wait_at(&acc_empty[acc], acc_phase[acc]);
                    acc_phase[acc] ^= 1u;
                    return is;
                };
                // a stage's products for one half of the lanes
                auto half = [&](uint32_t stage, uint32_t kb, uint32_t h, uint32_t acc) {
                    const uint32_t at = smem_u32(base + stage * S::kStage), ah = at + h * 2u * kBox, d = tmem + acc * S::kMaxN;
                    const uint64_t da = kADepth ? make_desc_by_depth(ah) : make_desc_sw128(ah);
                    const uint64_t db = kBDepth ? make_desc_by_depth(at + S::kA) : make_desc_sw128(at + S::kA);
                    tc_fence_after();
                    const uint32_t steps = kb == 0u ? first_steps : 4u;
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {                // 16 of the depth: 32 bytes on, or 16 rows of 128
                        if (j < steps) mma<kCtas>(d, da + (kADepth ? 128u : 2u) * j, db + (kBDepth ? 128u : 2u) * j, idesc, (kb - begin) % kSegment != 0u || j != 0u);
                    }
                    if (kb + 1u == end || (kb + 1u - begin) % kSegment == 0u) commit<kCtas>(&acc_full[acc]);
                };
                uint32_t ahead = begin;                                // blocks up to this one have run for the first half
                for (uint32_t kb = begin; ok && kb < end; kb++) {
                    const uint32_t acc = S::kHalves == 2u ? 0u : turn;
                    const bool fresh = (kb - begin) % kSegment == 0u;
                    if (kb == begin || kb > ahead) {
                        ok = mbar_wait(&full[s], ph, abort_flag);
                        if (!kRows && ok && kb == 0u && depth % 16u != 0u) {
                            ok = mbar_wait(&cleared[s], (clear_phases >> s) & 1u, abort_flag);
                            clear_phases ^= 1u << s;
                        }
                        if (!ok || (fresh && !(ok = free(acc)))) break;
                        half(s, kb, 0u, acc);
                    }
                    if (S::kHalves == 2u && halves == 2u) {
                        if (kb == begin) {
                            // While the second accumulator is read (its results wait for the first's to be stored) the first half
                            // runs ahead, as far as the ring reaches.
                            uint32_t s2 = s, ph2 = ph;
                            while (ok && ahead + 1u < min(begin + S::kStages, end) && !mbar_test(&acc_empty[1], acc_phase[1])) {
                                if (++s2 == S::kStages) { s2 = 0u; ph2 ^= 1u; }
                                ok = mbar_wait(&full[s2], ph2, abort_flag);
                                if (ok) half(s2, ++ahead, 0u, 0u);
                            }
                            if (!ok || !(ok = free(1u))) break;
                        }
                        half(s, kb, 1u, 1u);
                    }
                    commit<kCtas>(&empty[s]);
                    if (++s == S::kStages) { s = 0u; ph ^= 1u; }
                    if (S::kHalves == 1u && (kb + 1u == end || (kb + 1u - begin) % kSegment == 0u)) turn ^= 1u;
                }
            }
            if (*abort_flag != 0u) {
                commit<kCtas>(done);
                mbar_drain(done, 0u);
            }
        }
    } else if (warp == 2u) {
        // ------------------------------------------------- items, each shortly before its loads
        auto publish = [&](const Item &it) {                           // by one thread
            if (!wait_at(&item_empty[slot], slot_phase ^ 1u)) return false;
            items[slot] = it;
            mbar_arrive(&item_full[slot]);
            if (kCtas == 2u) {
                const uint32_t to = place_in(&items[slot], 1u);
                store_at(to, it.group);
                store_at(to + 4u, it.row);
                store_at(to + 8u, it.rows);
                store_at(to + 12u, it.lane0);
                store_at(to + 16u, it.column0);
                store_at(to + 20u, it.draw);
                arrive_at(place_in(&item_full[slot], 1u));
            }
            item_done();
            return it.group != kNoItem;
        };
        const Item none{kNoItem, 0u, 0u, 0u, 0u, 0u};
        auto weight_item = [&](uint32_t w) {                           // by weight: matrices side by side, then groups
            const uint32_t per = a.lane_tiles * a.column_tiles, g = w / per, at = w - g * per;
            uint32_t begin, end;
            group_rows(a.offsets, g, a.rows, begin, end);
            return Item{g, begin, end - begin, at / a.column_tiles * S::kLanes, at % a.column_tiles * S::kMaxN, 0u};
        };
        uint32_t w = blockIdx.x / (S::kSplit ? splits : kCtas);
        if (kCtas == 2u && rank == 1u) {
            if (elect_one()) {                                         // the block's warps have read an item: on to the first block
                Item it;
                while (next_item(it) && mbar_wait(&item_read_here[slot], slot_phase, abort_flag)) {
                    arrive_at(place_in(&item_empty[slot], 0u));
                    item_done();
                }
            }
        } else if (!kRows && a.least != 0u) {
            // the items of the groups that are this kernel's, 32 looked at together, every gridDim-th the block's
            const uint32_t total = a.groups * a.lane_tiles * a.column_tiles, step = gridDim.x;
            bool more = true;
            for (uint64_t first = blockIdx.x; more && first < total; first += (uint64_t)kWarp * step) {
                const uint64_t at = first + (uint64_t)lane * step;
                const Item it = at < total ? weight_item((uint32_t)at) : none;
                for (uint32_t mask = __ballot_sync(0xffffffffu, at < total && it.rows >= a.least); more && mask != 0u; mask &= mask - 1u) {
                    const uint32_t from = __ffs(mask) - 1u;
                    const Item next{__shfl_sync(0xffffffffu, it.group, from), __shfl_sync(0xffffffffu, it.row, from), __shfl_sync(0xffffffffu, it.rows, from),
                                    __shfl_sync(0xffffffffu, it.lane0, from), __shfl_sync(0xffffffffu, it.column0, from), 0u};
                    if (lane == 0u) more = publish(next);
                    more = __shfl_sync(0xffffffffu, more, 0);
                }
            }
            if (lane == 0u && more) publish(none);
        } else if (rank == 0u && a.single) {
            Item it = none;
            if (kRows) {
                Tile tile{};
                uint32_t lane_tile = 0u;
                if (search_tile(a.offsets, a.rows, a.groups, S::kMaxN, S::kStep, w, a.lane_tiles, tile, lane_tile)) {
                    it = Item{tile.group, tile.row, tile.rows, lane_tile * S::kLanes, 0u, 0u};
                }
            } else if (w < a.groups * a.lane_tiles * a.column_tiles) {
                it = weight_item(w);
            }
            if (elect_one() && publish(it)) publish(none);
        } else if (rank == 0u && elect_one()) {
            const uint32_t total = kRows ? a.plan->tiles * a.lane_tiles : a.groups * a.lane_tiles * a.column_tiles;
            uint32_t left = a.batch, want_phase = 0u;
            w *= a.batch;
            for (;;) {
                Item it = none;
                left--;
                if (w < total) {
                    if (kRows) {
                        const Tile of = a.tiles[w / a.lane_tiles];
                        const uint32_t local = w - of.first * a.lane_tiles, t = local % of.count;
                        const Tile tile = t + of.first == w / a.lane_tiles ? of : a.tiles[of.first + t];
                        it = Item{tile.group, tile.row, tile.rows, local / of.count * S::kLanes, 0u, 0u};
                    } else {
                        it = weight_item(w);
                    }
                    it.draw = left == 0u;
                }
                if (!publish(it)) break;
                if (left != 0u) {
                    w++;
                    continue;
                }
                if (!mbar_wait(wanted, want_phase, abort_flag)) break;
                want_phase ^= 1u;
                left = a.batch;
                w = gridDim.x / kCtas * a.batch + atomicAdd(&a.plan->counter, a.batch);
            }
        }
    } else if (warp == 3u) {
        if (!kRows) {
            // --------------------------------------------------- rows behind the group in its first block
            static_assert(kRows || kCtas == 1u, "a block clears and multiplies its own shared memory");
            uint32_t used = 0u, phases = 0u;                           // stages so far; of armed[], a bit each
            Item it;
            while (next_item(it)) {
                __syncwarp();
                if (lane == 0u) item_read();
                item_done();
                const uint32_t s = used % S::kStages, ph = (used / S::kStages) & 1u;
                used += (it.rows + kDepth - 1u) / kDepth;
                if (it.rows % 16u == 0u || split != 0u) continue;      // the first block is the first part's
                // once the load is under way the stage's barrier is in the phase that this one's parity names
                if (!mbar_wait(&armed[s], (phases >> s) & 1u, abort_flag) || !mbar_wait(&full[s], ph, abort_flag)) break;
                phases ^= 1u << s;
                unsigned char *at = base + s * S::kStage;
                const uint32_t a_boxes = halves_of(it) * 2u, boxes = a_boxes + boxes_of(columns_of(it));
                const uint32_t from = it.rows % kDepth, rows = 16u - from % 16u;
                for (uint32_t e = lane; e < boxes * rows * 8u; e += kWarp) {
                    const uint32_t box = e / (rows * 8u), in = e - box * rows * 8u;
                    unsigned char *to = box < a_boxes ? at + box * kBox : at + S::kA + (box - a_boxes) * kBox;
                    *reinterpret_cast<uint4 *>(to + from * 128u + in * 16u) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0u) mbar_arrive(&cleared[s]);
            }
        }
    } else {
        // --------------------------------------------------------------------------- results
        if (kShares) more_registers<232>();
        const uint32_t q = warp % 4u, part = (warp - 4u) / 4u;
        unsigned char *mine = base + S::kStore + (warp - 4u) * 4096u;
        const uint32_t row_length = kRows ? lanes : a.k;
        uint32_t acc_phase[2] = {0u, 0u}, turn = 0u;
        bool ok = true;
        Item it;
        while (ok && next_item(it)) {
            __syncwarp();
            if (lane == 0u) item_read();
            item_done();
            const uint32_t halves = halves_of(it), columns = columns_of(it);
            uint32_t begin, end;
            range_of((depth_of(it) + kDepth - 1u) / kDepth, begin, end);
            const bool nothing = begin == end;                         // by weight: a group without rows; a part with no blocks
            if (!S::kSplit && nothing && a.accumulate) continue;
            for (uint32_t h = 0; h < halves; h++) {
                const uint32_t acc = S::kHalves == 2u ? h : turn;
                constexpr uint32_t kChunks = S::kMaxN / 64u;           // of 32 columns, for this warp
                uint32_t v[kChunks][32];
                if (!nothing) {
                    if (!mbar_wait(&acc_full[acc], acc_phase[acc], abort_flag)) { ok = false; break; }
                    acc_phase[acc] ^= 1u;
                    tc_fence_after();
                    // columns past those that there are, too: they are in the accumulator
                    auto from = [&](uint32_t at, uint32_t c) { return tmem + at * S::kMaxN + (2u * c + part) * 32u + ((32u * q) << 16); };
#pragma unroll
                    for (uint32_t c = 0; c < kChunks; c++) tmem_ld_32x32(from(acc, c), v[c]);
#pragma unroll
                    for (uint32_t c = 0; c < kChunks; c++) k3::fp8::tmem_ld_wait_for(v[c]);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0u) accumulator_read(acc);
                    for (uint32_t kb = begin; end - kb > kSegment; kb += kSegment) {           // the item's other segments
                        turn ^= 1u;
                        if (!mbar_wait(&acc_full[turn], acc_phase[turn], abort_flag)) { ok = false; break; }
                        acc_phase[turn] ^= 1u;
                        tc_fence_after();
#pragma unroll
                        for (uint32_t c = 0; c < kChunks; c++) {
                            uint32_t more[32];
                            tmem_ld_32x32(from(turn, c), more);
                            k3::fp8::tmem_ld_wait_for(more);
#pragma unroll
                            for (uint32_t i = 0; i < 32u; i++) v[c][i] = __float_as_uint(__uint_as_float(v[c][i]) + __uint_as_float(more[i]));
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0u) accumulator_read(turn);
                    }
                    if (!ok) break;
                } else {
#pragma unroll
                    for (uint32_t c = 0; c < kChunks; c++) {
#pragma unroll
                        for (uint32_t i = 0; i < 32u; i++) v[c][i] = 0u;
                    }
                }
                if (S::kSplit) {
                    // this part's sums where the others read them: of a row of the group [column][128], by weight [128][columns]
                    // in units of 16 bytes permuted by the lane
                    float *sums = reinterpret_cast<float *>(base + S::kStore);
                    const uint32_t at = 32u * q + lane;
                    if (kRows) {
#pragma unroll
                        for (uint32_t i = 0; i < 32u; i++) sums[(part * 32u + i) * 128u + at] = __uint_as_float(v[0][i]);
                    } else {
#pragma unroll
                        for (uint32_t u = 0; u < 8u; u++) {
                            reinterpret_cast<uint4 *>(sums)[at * (S::kMaxN / 4u) + ((part * 8u + u) ^ (at & 7u))] =
                                make_uint4(v[0][4u * u], v[0][4u * u + 1u], v[0][4u * u + 2u], v[0][4u * u + 3u]);
                        }
                    }
                    continue;
                }
                // 32 x 32 at a time through shared memory: rows of the output, units of 16 bytes, permuted by the row.  This
                // thread then stores a unit of every kApart-th row; where that goes is worked out once per half (results of
                // 32 groups of 16 rows by 2048 x 7168, without the stores themselves: 150 us, with the products for the address in
                // every store 280; with them 287, the rate of the memory).
                constexpr uint32_t kUnits = kF32 ? 8u : 4u, kApart = 32u / kUnits, kSize = kF32 ? 4u : 2u;
                auto unit = [&](uint32_t row, uint32_t u) {
                    return mine + row * (kUnits * 16u) + ((u ^ (kF32 ? row & 7u : (row >> 1) & 3u)) * 16u);
                };
                const uint32_t lane0 = it.lane0 + S::kHalf * h + 128u * rank + 32u * q;      // this warp's first lane
                const uint32_t r0 = lane / kUnits, e0 = lane % kUnits * (16u / kSize);
                // the unit's row and column in the output, and how many of its rows and columns there are from there on
                const uint64_t row = kRows ? (uint64_t)it.row + part * 32u + r0 : (uint64_t)it.group * a.n + lane0 + r0;
                const uint32_t column = (kRows ? lane0 : it.column0 + part * 32u) + e0;
                const uint32_t from = (kRows ? part * 32u : lane0) + r0, rows = kRows ? it.rows : a.n;
                const uint64_t pitch = (uint64_t)row_length * kSize;
                char *to = (char *)a.out + row * pitch + (uint64_t)column * kSize;
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++, to += kRows ? 64u * pitch : 64u * kSize) {
                    if ((2u * c + part) * 32u >= columns) break;
                    if (kRows) {                                       // this thread's 32 results go down a column
#pragma unroll
                        for (uint32_t i = 0; i < 32u; i++) {
                            if (kF32) *reinterpret_cast<uint32_t *>(unit(i, lane / 4u) + (lane % 4u) * 4u) = v[c][i];
                            else *reinterpret_cast<uint16_t *>(unit(i, lane / 8u) + (lane % 8u) * 2u) = float_to_bf16_bits(__uint_as_float(v[c][i]));
                        }
                    } else {
#pragma unroll
                        for (uint32_t u = 0; u < kUnits; u++) {
                            uint4 x;
                            if (kF32) {
                                x = make_uint4(v[c][4u * u % 32u], v[c][(4u * u + 1u) % 32u], v[c][(4u * u + 2u) % 32u], v[c][(4u * u + 3u) % 32u]);
                            } else {
                                uint32_t word[4];
#pragma unroll
                                for (uint32_t j = 0; j < 4u; j++) {
                                    word[j] = bf16x2(__uint_as_float(v[c][(8u * u + 2u * j) % 32u]), __uint_as_float(v[c][(8u * u + 2u * j + 1u) % 32u]));
                                }
                                x = make_uint4(word[0], word[1], word[2], word[3]);
                            }
                            *reinterpret_cast<uint4 *>(unit(lane, u)) = x;
                        }
                    }
                    __syncwarp();
                    uint4 x[kUnits];
#pragma unroll
                    for (uint32_t i = 0; i < kUnits; i++) x[i] = *reinterpret_cast<const uint4 *>(unit(i * kApart + r0, lane % kUnits));
                    __syncwarp();
                    if (column + (kRows ? 0u : 64u * c) >= row_length) continue;
                    char *at = to;
#pragma unroll
                    for (uint32_t i = 0; i < kUnits; i++, at += kApart * pitch) {
                        if (from + (kRows ? 64u * c : 0u) + i * kApart >= rows) break;
                        if (kF32 && a.accumulate) {
                            const float4 o = *reinterpret_cast<const float4 *>(at);
                            x[i] = make_uint4(__float_as_uint(o.x + __uint_as_float(x[i].x)), __float_as_uint(o.y + __uint_as_float(x[i].y)),
                                              __float_as_uint(o.z + __uint_as_float(x[i].z)), __float_as_uint(o.w + __uint_as_float(x[i].w)));
                        }
                        *reinterpret_cast<uint4 *>(at) = x[i];
                    }
                }
            }
            if (S::kHalves == 1u && !nothing) turn ^= 1u;
        }
    }

    if (S::kSplit) {
        // the parts' sums in ascending order of the depth; each block adds its share of the item
        __syncwarp();
        cluster_barrier();
        const Item it = items[0];
        if (*abort_flag == 0u && it.group != kNoItem) {
            const uint32_t columns = columns_of(it), units = kRows ? 32u : (columns + 3u) / 4u;
            const uint32_t all = (kRows ? columns : 128u) * units, share = (all + splits - 1u) / splits, past = min(all, (split + 1u) * share);
            for (uint32_t e = split * share + threadIdx.x; e < past; e += kThreads) {
                const uint32_t major = e / units, u = e - major * units;             // of the group [column], by weight [lane]
                const uint32_t row = kRows ? it.row + major : it.lane0 + major, column = (kRows ? it.lane0 : it.column0) + 4u * u;
                if (kRows ? column >= lanes : row >= a.n) continue;
                const float *from = reinterpret_cast<const float *>(base + S::kStore) +
                                    (kRows ? major * 128u + 4u * u : major * S::kMaxN + 4u * (u ^ (major & 7u)));
                float4 x[kMaxParts];                                   // all under way before the first is added
#pragma unroll
                for (uint32_t r = 0; r < kMaxParts; r++) {
                    if (r < splits) x[r] = cluster_load4(from, r);
                }
                float4 sum = x[0];
#pragma unroll
                for (uint32_t r = 1; r < kMaxParts; r++) {
                    if (r < splits) sum = make_float4(sum.x + x[r].x, sum.y + x[r].y, sum.z + x[r].z, sum.w + x[r].w);
                }
                const uint64_t to = ((kRows ? 0u : (uint64_t)it.group * a.n) + row) * (kRows ? lanes : a.k) + column;
                if (kF32) {
                    float4 *out = reinterpret_cast<float4 *>((float *)a.out + to);
                    if (a.accumulate) sum = make_float4(out->x + sum.x, out->y + sum.y, out->z + sum.z, out->w + sum.w);
                    *out = sum;
                } else {
                    *reinterpret_cast<uint2 *>((uint16_t *)a.out + to) = make_uint2(bf16x2(sum.x, sum.y), bf16x2(sum.z, sum.w));
                }
            }
        }
        __syncwarp();
        cluster_barrier();                                             // nobody leaves while its sums are read
    }
    tc_fence_before();
    __syncthreads();
    if (kCtas == 2u) cluster_barrier();                                // nobody leaves while the other may signal here
    if (threadIdx.x == 0 && *abort_flag != 0u) atomicExch(&g_grouped_bf16_status, 1u);
    if (warp == 1u) {
        tc_fence_after();
        free_tmem<kCtas>(tmem, S::kTmem);
    }
}

// ------------------------------------------------------------------------------------------------ host
// bf16 [z, y, x] with boxes of 64 x box_y, 128-byte swizzle; what lies outside reads as zero.
bool make_map(CUtensorMap *map, const void *p, uint32_t x, uint64_t y, uint32_t z, uint32_t box_y) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[3] = {x, y, z};
    const cuuint64_t strides[2] = {(cuuint64_t)x * 2u, (cuuint64_t)x * y * 2u};
    const cuuint32_t box[3] = {64u, box_y, 1u}, steps[3] = {1u, 1u, 1u};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, z != 0u ? 3 : 2, const_cast<void *>(p), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr uint64_t plan_bytes(uint32_t tiles) { return sizeof(Plan) + (uint64_t)tiles * sizeof(Tile); }
// The most row tiles of up to max_n that the groups can have.
uint32_t most_tiles(uint32_t rows, uint32_t groups, uint32_t max_n) {
    return (uint32_t)((rows + (uint64_t)(max_n - 1u) * std::min(rows, groups)) / max_n);
}

constexpr uint32_t kFewRows = 64;
using Wide = Shape<2, 2, 256, 4>;
using Square = Shape<2, 1, 256, 6>;
using Middle = Shape<1, 1, 128, 6>;
using Few = Shape<1, 1, kFewRows, 8>;
using FewSplit = Shape<1, 1, kFewRows, 8, true>;
using WideWeight = Shape<1, 2, 256, 3>;
using DeepWeight = Shape<1, 1, 256, 4>;

// Items of a call, at most.
template <int kForm, typename S>
uint64_t items_of(const Product &p) {
    const uint64_t lanes = ((kForm == kByInput ? p.k : p.n) + S::kLanes - 1u) / S::kLanes;
    return lanes * (kForm == kByWeight ? (uint64_t)p.groups * ((p.k + S::kMaxN - 1u) / S::kMaxN) : most_tiles(p.rows, p.groups, S::kMaxN));
}

// Items per draw.  A draw takes about 1.3 us from the wish to the item, which items of a few stages do not cover; four at a
// time where every SM has 16 of them or more.
template <int kForm, typename S>
uint32_t batch_of(const Product &p) {
    const uint32_t depth = kForm == kForward ? p.k : kForm == kByInput ? p.n : p.rows / p.groups;
    return !S::kSplit && depth <= 4u * kDepth && items_of<kForm, S>(p) >= 16u * (uint64_t)sm_count() / S::kCtas ? 4u : 1u;
}

// parts: blocks that share an item's depth (S::kSplit); least: as TcArgs
template <int kForm, bool kF32, typename S>
bool launch(const Product &p, cudaStream_t stream, uint32_t parts = 1u, uint32_t least = 0u) {
    constexpr bool kRows = kForm != kByWeight;
    auto kernel = grouped_bf16_kernel<kForm, kF32, S>;
    CUtensorMap ma, mb;
    if (kForm == kForward) {
        if (!make_map(&ma, p.b, p.k, p.n, p.groups, 128u) || !make_map(&mb, p.a, p.k, p.rows, 0u, 32u)) return false;
    } else if (kForm == kByInput) {
        if (!make_map(&ma, p.b, p.k, p.n, p.groups, 64u) || !make_map(&mb, p.a, p.n, p.rows, 0u, 32u)) return false;
    } else {
        if (!make_map(&ma, p.a, p.n, p.rows, 0u, 64u) || !make_map(&mb, p.b, p.k, p.rows, 0u, 64u)) return false;
    }
    const uint32_t lanes = kForm == kByInput ? p.k : p.n, tiles = most_tiles(p.rows, p.groups, S::kMaxN);
    const uint64_t items = items_of<kForm, S>(p), places = S::kSplit ? items : (uint64_t)sm_count() / S::kCtas;
    const bool single = items <= places && (!kRows || p.groups <= kSearched);
    const TcArgs a{p.out, p.offsets, (Plan *)p.workspace, (Tile *)((Plan *)p.workspace + 1), p.rows, p.groups, p.n, p.k,
                   (lanes + S::kLanes - 1u) / S::kLanes, (p.k + S::kMaxN - 1u) / S::kMaxN, batch_of<kForm, S>(p), single, least, p.accumulate};
    if (items * parts > 0x7fffffffull || (S::kSplit && !single) || !set_max_dynamic_smem((const void *)kernel, S::kBytes)) return false;
    const uint32_t cluster = S::kSplit ? parts : S::kCtas;
    const bool planned = single || least != 0u || (kRows ? launch_chained(grouped_plan_kernel, 1, kMaxGroups, 0, stream, a.plan, a.tiles, p.offsets, p.rows,
                                                           p.groups, S::kMaxN, S::kStep, tiles)
                                          : launch_chained(grouped_counter_kernel, 1, 1, 0, stream, a.plan));
    return planned && launch_chained_cluster(kernel, (uint32_t)std::min(items, places) * cluster, kThreads, dim3(cluster, 1, 1), S::kBytes, stream,
                                             ma, mb, a);
}

template <int kForm, typename S>
bool launch_typed(const Product &p, cudaStream_t stream, uint32_t parts = 1u, uint32_t least = 0u) {
    return p.f32 ? launch<kForm, true, S>(p, stream, parts, least) : launch<kForm, false, S>(p, stream, parts, least);
}

// Which shape.  The host knows the rows and groups of a call, not how they are spread: it takes a third of the groups to hold
// all rows, each equally many, which lies between even loads and loads by Zipf's law, whose rows lie in groups of four times
// the mean; and of the shapes the one with the shortest time by what was measured on a B200 (us, and ns per stage of 64 of
// the depth): `fixed` for a call, `item` for an item's results, and per stage base + column x columns, alone in a single round
// of items, full where the SMs share memory and power over several.  Over 176 calls of 1 to 64 even groups of 1 to 2048 rows
// at 2048 x 7168, 7168 x 2048, 2048 x 1024 and 512 x 512 the shape that this takes is 2.4 % from the best on average, over
// eight of 16 to 896 uneven groups 3.2 % (with all groups holding rows 0.8 and 13.6 %).  What each is for:
//   Few      up to 64 rows per group: bound by the matrices' bytes, 6.4 TB/s at 64 groups of 8 rows of 2048 x 7168 (274 us; Middle 294)
//   Middle   up to 128, or too few items for larger ones (4 groups of 256 rows: 35 us; Few 53, Square 43)
//   Square   pairs of blocks with two accumulators (16 groups of 256 rows of 7168 x 2048: 107 us; Wide 115, Middle 134)
//   Wide     least traffic per product, so least power, which bounds large calls (64 groups of 512 rows of 2048 x 7168, forward, bf16,
//            712 us 20 in a row and 848 for 0.8 s; Square 735 and 876)
struct Cost {
    double fixed, item, alone, alone_column, full, full_column;
};
template <typename S>
double time_of(const Cost &c, double items, double stages, double columns) {
    const double rounds = items / ((double)sm_count() / S::kCtas);
    if (rounds <= 1.0) return c.fixed + c.item + stages * (c.alone + c.alone_column * columns) * 1e-3;
    return c.fixed + (rounds + 0.4) * (c.item + stages * (c.full + c.full_column * columns) * 1e-3);
}
constexpr Cost kFewCost = {4.5, 0.0, 225, 0.1, 240, 0.6}, kMiddleCost = {5, 1, 232, 0.12, 245, 0.5}, kSquareCost = {6, 1.5, 210, 0.5, 165, 1.33},
               kWideCost = {8, 8, 120, 1.9, 380, 2.06};
constexpr Cost kFewWeight = {2.8, 1, 190, 0.1, 240, 0.6}, kMiddleWeight = {3, 1.2, 200, 0.4, 245, 0.5}, kWideWeight = {3, 4, 350, 1.2, 400, 1.2};

// Few items: the blocks that share the depth of each, as many as there are SMs for.  The parts' way through the cluster costs
// about 6.5 us and 0.05 per column; one group of 8 rows of 2048 x 7168 takes 9.6 us in eight parts, 25.9 in one.
template <int kForm>
uint32_t parts_of(const Product &p, uint32_t stages, double columns, double shortest) {
    const uint64_t items = items_of<kForm, FewSplit>(p);
    if (items * 2u > (uint64_t)sm_count() || (kForm != kByWeight && p.groups > kSearched)) return 1u;
    auto kernel = grouped_bf16_kernel<kForm, true, FewSplit>;
    if (!set_max_dynamic_smem((const void *)kernel, FewSplit::kBytes)) return 1u;
    const ActiveClusters active = active_clusters((const void *)kernel, kThreads, FewSplit::kBytes);
    uint32_t parts = std::max(1u, std::min(kMaxParts, stages));
    while (parts > 1u && active.of_size[parts] < items) parts--;
    return 6.5 + 0.05 * columns + 0.23 * ((stages + parts - 1u) / parts) < shortest ? parts : 1u;
}

template <int kForm>
bool rows_product(const Product &p, cudaStream_t stream) {
    const uint32_t stages = ((kForm == kForward ? p.k : p.n) + kDepth - 1u) / kDepth;
    const double rows = std::min(3.0 * p.rows / std::min(p.rows, p.groups), (double)p.rows), groups = p.rows / rows;
    auto time = [&](auto shape, const Cost &c) {
        using S = decltype(shape);
        const double tiles = std::ceil(rows / S::kMaxN), lanes = (double)(((kForm == kByInput ? p.k : p.n) + S::kLanes - 1u) / S::kLanes);
        return time_of<S>(c, groups * tiles * lanes, stages, rows / tiles);
    };
    const double few = time(Few{}, kFewCost), middle = time(Middle{}, kMiddleCost), square = time(Square{}, kSquareCost);
    const bool deep = p.f32 && stages > 8u;                           // Wide has no segments
    const double wide = deep ? INFINITY : time(Wide{}, kWideCost), shortest = rows <= kFewRows ? few : std::min({few, middle, square, wide});
    const uint32_t parts = parts_of<kForm>(p, stages, std::min(rows, (double)kFewRows), shortest);
    if (parts > 1u) return launch_typed<kForm, FewSplit>(p, stream, parts);
    if (shortest == few) return launch_typed<kForm, Few>(p, stream);
    if (shortest == middle) return launch_typed<kForm, Middle>(p, stream);
    return shortest == square ? launch_typed<kForm, Square>(p, stream) : launch_typed<kForm, Wide>(p, stream);
}

// By weight the lanes and columns are the matrices', the depth the rows; one block per item, for pairs multiply two operands
// that lie by their depth 10 % more slowly (4096 rows of 8 groups, without the stores: 669 us, pairs 729).
bool weight_product(const Product &p, cudaStream_t stream) {
    if (p.rows <= kOuterRows) return product_outer(p, stream);
    const uint32_t stages = std::max(1u, (p.rows / p.groups + kDepth - 1u) / kDepth);
    auto time = [&](auto shape, const Cost &c) {
        using S = decltype(shape);
        return time_of<S>(c, (double)items_of<kByWeight, S>(p), stages, std::min(p.k, S::kMaxN));
    };
    const double few = time(Few{}, kFewWeight), middle = time(Middle{}, kMiddleWeight), wide = time(WideWeight{}, kWideWeight);
    const double shortest = std::min({few, middle, wide});
    const uint32_t parts = parts_of<kByWeight>(p, stages, std::min(p.k, kFewRows), shortest);
    if (parts > 1u) return launch_typed<kByWeight, FewSplit>(p, stream, parts);
    // Few rows per group: those of up to 16 rows go to the other kernel, whose time is its stores, and what this one then takes to
    // look the groups over.  bf16 and f32, us, here alone / both: 896 groups of 3 rows, 264 x 520 143 / 68 and 156 / 96, by
    // Zipf's law 119 / 74 and 139 / 104; 32 groups of 8, 2048 x 7168 197 / 168 and 317 / 287, of 12 195 / 180 and 320 / 295, of 16 195 /
    // 195 and 320 / 313; 128 groups of 3, 512 x 1024 39 / 35 and 53 / 55, so f32 stays here.
    const double bytes = (double)p.groups * p.n * p.k * (p.f32 ? 4.0 : 2.0), stores = 3.0 + bytes / 6.1e6, both = 10.0 + bytes / 6.9e6;
    const bool outer = p.rows <= 12u * (uint64_t)p.groups && both < std::max(shortest, stores);
    if (outer && !product_outer(p, stream)) return false;
    const uint32_t least = outer ? kOuterRows + 1u : 0u;
    if (shortest == few) return launch_typed<kByWeight, Few>(p, stream, 1u, least);
    if (shortest == middle) return launch_typed<kByWeight, Middle>(p, stream, 1u, least);
    if (!p.f32) return launch<kByWeight, false, WideWeight>(p, stream, 1u, least);
    // f32 in segments, so items of one half, whatever the group's size: 4.7e-7 of the gradient's norm from 64 bits where two halves
    // without segments are 2.3e-7 at 256 rows, 1.0e-6 at 1024 and 4.4e-6 at 4096.  Longest where all groups hold some 1000 rows: 32 of
    // 1024 rows, 2048 x 7168, 980 us, 898 without segments; 32 of 512 607 and 580, of 256 421 and 424, of 2000 1660 either way; 32 of
    // 512 rows by Zipf's law, 512 x 1024, 38 us, 57 with larger groups in a launch of their own (20 calls in a row).  The shape is
    // the one that the times of two halves give, on average 2 % from the best of the three over 193 calls.
    return launch<kByWeight, true, DeepWeight>(p, stream, 1u, least);
}

}  // namespace

uint64_t k3::gb::tc_workspace_bytes(uint32_t rows, uint32_t groups) { return plan_bytes(most_tiles(rows, groups, kFewRows)); }

bool k3::gb::product_tc(const Product &p, cudaStream_t stream) {
    if (p.form == kByWeight) return weight_product(p, stream);
    return p.form == kForward ? rows_product<kForward>(p, stream) : rows_product<kByInput>(p, stream);
}

uint32_t k3_grouped_bf16_status() {
    uint32_t v = 0xffffffffu;
    if (cudaMemcpyFromSymbol(&v, g_grouped_bf16_status, sizeof(v)) != cudaSuccess) (void)cudaGetLastError();
    return v;
}

bool k3_grouped_bf16_status_clear() {
    const uint32_t zero = 0u;
    const bool ok = cudaMemcpyToSymbol(g_grouped_bf16_status, &zero, sizeof(zero)) == cudaSuccess;
    if (!ok) (void)cudaGetLastError();
    return ok;
}
