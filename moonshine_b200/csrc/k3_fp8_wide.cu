// Products of E4M3 matrices with many rows on tcgen05 (kind::f8f6f4).
//
//   out[m, n] = sum_kb sa[m, kb] sb[n, kb] sum_{k in kb} a[m, k] b[n, k]
//
// The scales are f32, so no MMA kind applies them: the tensor cores sum one block of 128 columns into
// tensor memory, and warps with the running f32 sums in registers read it, scale it and add it while the
// tensor cores sum the next block into the other half of tensor memory.  a's rows are the lanes, so a
// thread's row scale is one register, and 128 of b's rows share a block scale: one packed FMA per two
// elements and block is all the arithmetic there is.
//
// One work item = 128 rows x 256 columns over the whole depth (kOutActivated: 128 columns of gate and
// the same 128 of up).  One block per SM, items in a static order:
//   warp 0        loads by TMA: a stage is 128 columns of 128 rows of a and 256 rows of b, 48 KB
//   warp 1        MMA issuer, owns the tensor memory
//   warp 2        scales, four blocks ahead: a row's times the block's, where the adding warps read them
//   warps 4-11    running sums: lane quadrant warp % 4, columns in two halves (kOutActivated: warps 4-19, quarters)
// kSplit (one matrix, fewer items than SMs, or the items that are left over when every SM has had as many as
// the others): an item is a cluster of up to 8 blocks with a part of the depth each, which add their sums
// through distributed shared memory in ascending order of the depth.
// The warpgroups of running sums take registers over from the first one: with 128 sums per thread
// 2 x 128 x 232 + 128 x 40 are the 384 x 168 of the launch, with 64 (kOutActivated) 4 x 128 x 112 + 128 x 32 the
// 640 x 96.  Four warps per scheduler instead of two hide more of the activations' chains, but the stores of the
// other epilogues take longer: gate/up of 4096 tokens (16 of 64 experts, 7168 x 2048) 2.09 ms back to back against
// 2.40, 8192 x 7168 x 7168 386 us against 364.
//
// Every wait is bounded; on give-up the block raises the status word, waits for its copies and frees its
// tensor memory.
//
// Measured, 8192 x 7168 x 7168: 374 us = 2.25 PFLOP/s in a burst at 1965 MHz, 436 us = 1.93 back to back,
// where the power limit holds the clock at 1410 MHz.  With half of the reads and adds left out (a wrong
// result) it takes 331 and 388 us: power bounds what is left.  Pairs of blocks (cta_group::2), which halve
// b's way from L2, take the same time with arrivals across the pair that carry no release, and twice as
// long with release.  Loads of 64 columns at once, or the next block's before the last adds, change
// nothing or cost 5 %.
#include "k3_fp8_ptx.cuh"
#include "k3_grouped.h"
#include "k3_moe_layer.h"

#include <algorithm>

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t BM = 128, BN = 256;
constexpr uint32_t kATile = BM * kBlock, kBTile = BN * kBlock;       // 16 KB, 32 KB
constexpr uint32_t kStageBytes = kATile + kBTile;
// Column parts of an item, and threads: a warp of running sums has a quarter of the rows and one part of the columns.
// Four parts where the epilogue is the activation, two elsewhere.
template <int kEpilogue>
constexpr uint32_t kParts = kEpilogue == kOutActivated ? 4u : 2u;
template <int kEpilogue>
constexpr uint32_t kThreads = 128u + 128u * kParts<kEpilogue>;
constexpr uint32_t kStoreBytes = 8u * 32u * 64u;                     // 8 warps: 32 rows of 64 bytes on their way out
constexpr uint32_t kMaxGroups = 1024;
constexpr uint32_t kMaxSplits = 8;                                   // of the depth: the portable cluster
constexpr uint32_t kScaleSlots = 2, kSlotBlocks = 4;                 // scales travel four blocks at a time

template <bool kColumnScales>
struct Layout {
    // a block's scales: of the 128 rows for each half of the columns, or of the rows and of the 256 columns
    static constexpr uint32_t kBlockScales = kColumnScales ? BM + BN : 2u * BM;
    static constexpr uint32_t kSlotFloats = kSlotBlocks * kBlockScales;
    static constexpr uint32_t kStages = kColumnScales ? 3u : 4u;     // the columns' scales take the fourth stage's place
    static constexpr uint32_t kStore = kStages * kStageBytes;
    static constexpr uint32_t kScales = kStore + kStoreBytes;
    static constexpr uint32_t kLargest = kScales + kScaleSlots * kSlotFloats * 4u;   // f32 bits [2][4][128]: the parts' largest activations
    static constexpr uint32_t kPrefix = kLargest + 8u * BM * 4u;
    static constexpr uint32_t kBars = (kPrefix + (kMaxGroups + 1u) * 4u + 15u) / 16u * 16u;
    static constexpr uint32_t kBytes = kBars + 256u + 1024u;         // the last: alignment
    static_assert(kBytes <= 232448u, "shared memory of a block");
};

__device__ uint32_t g_fp8_wide_status = 0;

struct WideArgs {
    void *out;
    float *out_scales;
    const float *a_scales, *b_scales, *b2_scales;
    const uint32_t *offsets;
    uint32_t groups, rows, n, k;
    uint32_t column_items;
    uint32_t items;                                                  // one matrix: items of this launch
    uint32_t first_item;                                             // kSplit: and the first of them
    uint32_t split_blocks;                                           // kSplit: blocks of 128 per part, a multiple of 4
    bool b_ready;                                                    // Product::b_ready
    int accumulate;
    int activation;
    float beta, by_beta, linear_beta, by_linear_beta;                // by_: the reciprocals
};

struct Item {
    uint32_t group, row, rows, column, kb_begin, kb_end;
};

// the largest of a and the magnitudes of b and c; NaN if one of them is
K3_DEVINL float largest_of(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The first half of the pairs of sums (gate) and the other half (up) to the negatives of the activations in the first,
// zero past `left`; the largest magnitude's bits, or a NaN's.
template <bool kSitu, uint32_t kPairs>
K3_DEVINL uint32_t activate(uint64_t (&sum)[kPairs], uint32_t left, const ExpertActivation<kSitu> &act) {
    float most = 0.f;
#pragma unroll
    for (uint32_t j = 0; j < kPairs / 2u; j++) {
        sum[j] = negative_activation2(act, sum[j], sum[kPairs / 2u + j]);
        if (left < kPairs) sum[j] = pack2(2u * j < left ? lo2(sum[j]) : 0.f, 2u * j + 1u < left ? hi2(sum[j]) : 0.f);
        most = largest_of(most, lo2(sum[j]), hi2(sum[j]));
    }
    return __float_as_uint(most);
}

// four neighbouring results at `out`, of which `left` columns exist
K3_DEVINL void store4(float *out, const float (&sum)[4], uint32_t left, bool vector, int accumulate) {
    float v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4u; j++) v[j] = accumulate && j < left ? out[j] + sum[j] : sum[j];
    if (vector) {
        *reinterpret_cast<float4 *>(out) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) {
            if (j < left) out[j] = v[j];
        }
    }
}
K3_DEVINL void store4(uint16_t *out, const float (&sum)[4], uint32_t left, bool vector, int) {
    if (vector) {
        *reinterpret_cast<uint2 *>(out) = make_uint2(bf16x2(sum[0], sum[1]), bf16x2(sum[2], sum[3]));
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4u; j++) {
            if (j < left) out[j] = float_to_bf16_bits(sum[j]);
        }
    }
}

template <int kEpilogue, bool kColumnScales, bool kSplit>
__global__ void __launch_bounds__(kThreads<kEpilogue>, 1)
fp8_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_b2, WideArgs a) {
    using L = Layout<kColumnScales>;
    constexpr uint32_t kSumWarps = 4u * kParts<kEpilogue>, kPairs = BN / kParts<kEpilogue> / 2u;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t *full = reinterpret_cast<uint64_t *>(base + L::kBars);  // [kStages]
    uint64_t *empty = full + L::kStages;                             // [kStages]
    uint64_t *sum_full = empty + L::kStages;                         // [2] a block's products are in tensor memory
    uint64_t *sum_empty = sum_full + 2;                              // [2] and have been read
    uint64_t *scale_full = sum_empty + 2;                            // [kScaleSlots]
    uint64_t *scale_empty = scale_full + kScaleSlots;                // [kScaleSlots]
    uint64_t *largest_full = scale_empty + kScaleSlots;              // [1]
    uint64_t *done = largest_full + 1;                               // [1] every MMA issued has run
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    uint32_t *total_s = tmem_slot + 2;
    uint32_t *prefix = reinterpret_cast<uint32_t *>(base + L::kPrefix);
    const uint32_t warp = warp_index(), lane = threadIdx.x % kWarp;
    const uint32_t blocks = blocks_of(a.k);
    constexpr uint32_t kColumns = kEpilogue == kOutActivated ? kBlock : BN;

    auto item_of = [&](uint32_t w) {
        Item it;
        it.kb_begin = 0u;
        it.kb_end = blocks;
        if (kSplit) {
            w = a.first_item + blockIdx.y;
            it.kb_begin = blockIdx.x * a.split_blocks;
            it.kb_end = min(blocks, it.kb_begin + a.split_blocks);
        }
        const uint32_t tile = w / a.column_items;
        it.column = (w - tile * a.column_items) * kColumns;
        if (a.offsets == nullptr) {
            it.group = 0u;
            it.row = tile * BM;
            it.rows = min(BM, a.rows - it.row);
            return it;
        }
        uint32_t lo = 0u, hi = a.groups;                             // the last group whose first tile is at most `tile`
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (prefix[mid] <= tile) lo = mid; else hi = mid;
        }
        it.group = lo;
        it.row = a.offsets[lo] + (tile - prefix[lo]) * BM;
        it.rows = min(BM, a.offsets[lo + 1u] - it.row);
        return it;
    };
    // b's 256 rows of a stage; the barrier waits for a's 128 as well
    auto load_b = [&](const Item &it, uint32_t stage, uint32_t kb) {
        unsigned char *st = base + stage * kStageBytes + kATile;
        const int32_t x = (int32_t)(kb * kBlock), y = (int32_t)(it.group * a.n + it.column);
        mbar_arrive_expect_tx(&full[stage], kStageBytes);
        tma_load_2d(st, &map_b, &full[stage], x, y);
        if (kEpilogue == kOutActivated) tma_load_2d(st + kBTile / 2u, &map_b2, &full[stage], x, y);
        else tma_load_2d(st + kBTile / 2u, &map_b, &full[stage], x, y + (int32_t)kBlock);
    };

    if (warp == 0u && elect_one()) {
        *abort_flag = 0u;
        for (uint32_t s = 0; s < L::kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t s = 0; s < 2u; s++) {
            mbar_init(&sum_full[s], 1);
            mbar_init(&sum_empty[s], kSumWarps);
        }
        for (uint32_t s = 0; s < kScaleSlots; s++) {
            mbar_init(&scale_full[s], kWarp);
            mbar_init(&scale_empty[s], kSumWarps);
        }
        mbar_init(largest_full, kSumWarps);
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
        if (kEpilogue == kOutActivated) prefetch_tensormap(&map_b2);
        if (kSplit) {                                                // b's first stages, before anyone waits for anyone
            if (!a.b_ready) pdl_wait();
            const Item it = item_of(0u);
            for (uint32_t i = 0; i < min(L::kStages, it.kb_end - it.kb_begin); i++) load_b(it, i, it.kb_begin + i);
        }
    }
    if (warp == 1u) {
        tmem_alloc(tmem_slot, 512u);
        tmem_relinquish();
    }
    if (!a.b_ready) pdl_wait();                                      // otherwise every role waits for itself
    if (a.offsets != nullptr) {
        // exclusive prefix of the groups' row tiles, one warp, 32 groups at a time
        if (warp == 2u) {
            uint32_t before = 0u;
            for (uint32_t g0 = 0; g0 < a.groups; g0 += kWarp) {
                const uint32_t g = g0 + lane;
                const uint32_t n = g < a.groups ? (a.offsets[g + 1u] - a.offsets[g] + BM - 1u) / BM : 0u;
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
    } else if (threadIdx.x == 0) {
        *total_s = kSplit ? 1u : a.items;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot, total = *total_s;
    const uint32_t first_item = kSplit ? 0u : blockIdx.x, step = kSplit ? 1u : gridDim.x;

    if (warp < 4u) {
        fewer_registers<kPairs == 64u ? 40u : 32u>();
        if (warp == 0u) {
            // ------------------------------------------------------------------------- loads
            if (elect_one()) {
                uint32_t s = 0u, ph = 0u, issued = 0u, early = 0u;
                bool ok = true;
                if (kSplit) {
                    const Item it = item_of(0u);
                    early = min(L::kStages, it.kb_end - it.kb_begin);
                } else if (a.b_ready && first_item < total) {
                    const Item it = item_of(first_item);
                    early = min(L::kStages, blocks);
                    for (uint32_t i = 0; i < early; i++) load_b(it, i, i);
                }
                if (a.b_ready) pdl_wait();
                for (uint32_t w = first_item; ok && w < total; w += step) {
                    const Item it = item_of(w);
                    for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb++) {
                        if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) { ok = false; break; }
                        if (issued >= early) load_b(it, s, kb);
                        tma_load_2d(base + s * kStageBytes, &map_a, &full[s], (int32_t)(kb * kBlock), (int32_t)it.row);
                        issued++;
                        if (++s == L::kStages) { s = 0u; ph ^= 1u; }
                    }
                }
                pdl_trigger();                                       // the blocks of the next kernel may take places as these leave
                if (*abort_flag != 0u) {                             // nothing may land in a block that has left
                    issued = max(issued, early);
                    for (uint32_t i = issued > L::kStages ? issued - L::kStages : 0u; i < issued; i++) {
                        mbar_drain(&full[i % L::kStages], (i / L::kStages) & 1u);
                    }
                }
            }
        } else if (warp == 1u) {
            // --------------------------------------------------------------------------- MMA
            if (elect_one()) {
                constexpr uint32_t idesc = make_idesc_e4m3(BM, BN);
                uint32_t s = 0u, ph = 0u, at = 0u, aph = 0u;
                bool ok = true;
                for (uint32_t w = first_item; ok && w < total; w += step) {
                    const uint32_t n = kSplit ? item_of(w).kb_end - item_of(w).kb_begin : blocks;
                    for (uint32_t kb = 0; kb < n; kb++) {
                        if (!mbar_wait(&full[s], ph, abort_flag) || !mbar_wait(&sum_empty[at], aph ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t addr = smem_u32(base + s * kStageBytes), d = tmem + at * BN;
                        const uint64_t da = make_desc_sw128(addr), db = make_desc_sw128(addr + kATile);
#pragma unroll
                        for (uint32_t j = 0; j < 4u; j++) mma_e4m3_ss(d, da + 2u * j, db + 2u * j, idesc, j != 0u);
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
        } else if (warp == 2u) {
            // ------------------------------------------------------------- scales, a slot at a time
            if (a.b_ready) pdl_wait();
            uint32_t slot = 0u, ph = 0u;
            bool ok = true;
            const uint32_t pitch = (blocks + 3u) & ~3u, b_blocks = blocks_of(a.n);
            for (uint32_t w = first_item; ok && w < total; w += step) {
                const Item it = item_of(w);
                // b's rows of block scales: of the two halves of the columns, or gate's and up's
                const uint64_t sb = ((uint64_t)it.group * b_blocks + it.column / kBlock) * blocks;
                const float *b0 = a.b_scales + sb;
                const float *b1 = kEpilogue == kOutActivated ? a.b2_scales + sb
                                  : it.column / kBlock + 1u < b_blocks ? b0 + blocks : b0;
                for (uint32_t kb = it.kb_begin; kb < it.kb_end; kb += kSlotBlocks) {
                    if (!mbar_wait(&scale_empty[slot], ph ^ 1u, abort_flag)) { ok = false; break; }
                    float *to = reinterpret_cast<float *>(base + L::kScales) + slot * L::kSlotFloats;
                    float f0[4], f1[4];
                    if (!kColumnScales) {
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) {
                            f0[i] = b0[min(kb + i, blocks - 1u)];
                            f1[i] = b1[min(kb + i, blocks - 1u)];
                        }
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        const uint32_t r = j * kWarp + lane;
                        const float4 v = *reinterpret_cast<const float4 *>(
                            a.a_scales + (uint64_t)min(it.row + r, a.rows - 1u) * pitch + kb);
                        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (uint32_t i = 0; i < 4u; i++) {
                            to[i * L::kBlockScales + r] = kColumnScales ? x[i] : x[i] * f0[i];
                            if (!kColumnScales) to[i * L::kBlockScales + BM + r] = x[i] * f1[i];
                        }
                    }
                    if (kColumnScales) {
#pragma unroll
                        for (uint32_t j = 0; j < 8u; j++) {
                            const uint32_t c = j * kWarp + lane;
                            const float4 v = *reinterpret_cast<const float4 *>(
                                a.b_scales + (uint64_t)min(it.column + c, a.n - 1u) * pitch + kb);
                            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (uint32_t i = 0; i < 4u; i++) to[i * L::kBlockScales + BM + c] = x[i];
                        }
                    }
                    mbar_arrive(&scale_full[slot]);
                    if (++slot == kScaleSlots) { slot = 0u; ph ^= 1u; }
                }
            }
        }
        if (kSplit) {                                                // the other warps' two barriers, see below
            __syncwarp();
            cluster_barrier();
            cluster_barrier();
        }
    } else {
        // ---------------------------------------------------------------------- running sums
        more_registers<kPairs == 64u ? 232u : 112u>();
        if (a.b_ready) pdl_wait();                                   // before the first store
        const uint32_t q = warp % 4u, part = (warp - 4u) / 4u;
        // half of a thread's sums are columns first, first + 1, .. of the tile, the other half those from second
        const uint32_t first = part * (kEpilogue == kOutActivated ? kPairs : 2u * kPairs);
        const uint32_t second = first + (kEpilogue == kOutActivated ? kBlock : kPairs);
        const uint32_t lanes = tmem + ((32u * q) << 16);
        const uint32_t row_in = 32u * q + lane;
        uint32_t at = 0u, aph = 0u, slot = 0u, sph = 0u, lph = 0u;
        bool ok = true;
        for (uint32_t w = first_item; ok && w < total; w += step) {
            const uint32_t kb_begin = kSplit ? blockIdx.x * a.split_blocks : 0u;
            const uint32_t kb_end = kSplit ? min(blocks, kb_begin + a.split_blocks) : blocks;
            uint64_t sum[kPairs];
#pragma unroll
            for (uint32_t i = 0; i < kPairs; i++) sum[i] = 0ull;
            for (uint32_t kb = kb_begin; kb < kb_end; kb++) {
                if (kb % kSlotBlocks == 0u && !mbar_wait(&scale_full[slot], sph, abort_flag)) { ok = false; break; }
                const float *scales = reinterpret_cast<const float *>(base + L::kScales) + slot * L::kSlotFloats +
                                      kb % kSlotBlocks * L::kBlockScales;
                float s0, s1;
                if (kColumnScales) {
                    s0 = s1 = scales[row_in];
                } else if (kEpilogue == kOutActivated) {
                    s0 = scales[row_in];
                    s1 = scales[BM + row_in];
                } else {
                    s0 = s1 = scales[first / kBlock * BM + row_in];
                }
                if (!mbar_wait(&sum_full[at], aph, abort_flag)) { ok = false; break; }
                tc_fence_after();
                // with registers for it the next 32 columns are on their way while these are added
                constexpr uint32_t kChunks = kPairs / 16u, kAhead = kPairs == 64u ? 1u : 0u;
                auto column_of = [&](uint32_t c) { return (c < kChunks / 2u ? first : second) + c % (kChunks / 2u) * 32u; };
                uint32_t r[kAhead + 1u][32];
                if (kAhead) tmem_ld_32x32(lanes + at * BN + first, r[0]);
#pragma unroll
                for (uint32_t c = 0; c < kChunks; c++) {
                    const uint32_t column = column_of(c);
                    uint32_t (&v)[32] = r[c & kAhead];
                    if (!kAhead) tmem_ld_32x32(lanes + at * BN + column, v);
                    tmem_ld_wait_for(v);
                    if (c < kChunks - 1u) {
                        if (kAhead) tmem_ld_32x32(lanes + at * BN + column_of(c + 1u), r[(c + 1u) & kAhead]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0u) mbar_arrive(&sum_empty[at]);
                    }
                    const uint64_t s2 = both2(c < kChunks / 2u ? s0 : s1);
                    if (kColumnScales) {
                        const ulonglong2 *by = reinterpret_cast<const ulonglong2 *>(scales + BM + column);
#pragma unroll
                        for (uint32_t j = 0; j < 8u; j++) {
                            const ulonglong2 b = by[j];
                            const uint32_t p = c * 16u + j * 2u;
                            sum[p] = fma2(mul2(pack2(v[4u * j], v[4u * j + 1u]), s2), b.x, sum[p]);
                            sum[p + 1u] = fma2(mul2(pack2(v[4u * j + 2u], v[4u * j + 3u]), s2), b.y, sum[p + 1u]);
                        }
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 16u; j++) {
                            sum[c * 16u + j] = fma2(pack2(v[2u * j], v[2u * j + 1u]), s2, sum[c * 16u + j]);
                        }
                    }
                }
                if (++at == 2u) { at = 0u; aph ^= 1u; }
                if (kb % kSlotBlocks == kSlotBlocks - 1u || kb + 1u == kb_end) {
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&scale_empty[slot]);
                    if (++slot == kScaleSlots) { slot = 0u; sph ^= 1u; }
                }
            }
            if (!ok) break;
            const Item it = item_of(w);                              // looked up here: the loop above has no registers to spare
            if (kSplit) {
                // [128][64] units of 16 bytes in the ring's place (every stage has been read), swizzled by the row
                float4 *part = reinterpret_cast<float4 *>(base) + row_in * (BN / 4u);
#pragma unroll
                for (uint32_t j = 0; j < kPairs / 2u; j++) {
                    const uint32_t unit = (j < kPairs / 4u ? first : second) / 4u + j % (kPairs / 4u);
                    part[unit ^ (row_in & 7u)] = make_float4(lo2(sum[2u * j]), hi2(sum[2u * j]), lo2(sum[2u * j + 1u]), hi2(sum[2u * j + 1u]));
                }
            } else if (kEpilogue == kOutActivated) {
                // ------------------------------------------ activation, largest of the row's 128, codes
                const uint32_t left = it.column + first < a.n ? a.n - it.column - first : 0u;       // of the thread's columns, those that exist
                const uint32_t most_here = a.activation == kActSitu
                    ? activate<true>(sum, left, {a.beta, a.by_beta, a.linear_beta, a.by_linear_beta})
                    : activate<false>(sum, left, {});
                // one of two buffers in turn: a warp is here again only when all have read what it wrote two items ago
                uint32_t *largest = reinterpret_cast<uint32_t *>(base + L::kLargest) + lph * 4u * BM;
                largest[part * BM + row_in] = most_here;
                __syncwarp();
                if (lane == 0u) mbar_arrive(largest_full);
                if (!mbar_wait(largest_full, lph, abort_flag)) { ok = false; break; }
                lph ^= 1u;
                uint32_t most = most_here;
#pragma unroll
                for (uint32_t i = 1; i < kParts<kEpilogue>; i++) most = max(most, largest[(part ^ i) * BM + row_in]);
                const float scale = scale_of(most);
                const uint64_t by = both2(scale * lift_of(scale)), inverse = both2(-inverse_of(scale));
                if (lift_of(scale) != 1.0f) {
#pragma unroll
                    for (uint32_t j = 0; j < kPairs / 2u; j++) sum[j] = mul2(sum[j], both2(lift_of(scale)));
                }
                if (row_in < it.rows) {
                    const uint64_t row = it.row + row_in;
                    const uint32_t out_pitch = pitch_of(a.n), scale_pitch = scale_pitch_of(a.n);
                    if (part == 0u) a.out_scales[row * scale_pitch + it.column / kBlock] = scale;
                    uint8_t *to = (uint8_t *)a.out + row * out_pitch + it.column + first;
#pragma unroll
                    for (uint32_t c = 0; c < kPairs / 16u; c++) {
                        uint32_t word[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4u; j++) {
                            const uint64_t x = divided2(sum[c * 8u + 2u * j], by, inverse);
                            const uint64_t y = divided2(sum[c * 8u + 2u * j + 1u], by, inverse);
                            word[j] = codes2(lo2(x), hi2(x)) | (codes2(lo2(y), hi2(y)) << 16);
                        }
                        if (it.column + first + c * 16u < out_pitch) {
                            *reinterpret_cast<uint4 *>(to + c * 16u) = make_uint4(word[0], word[1], word[2], word[3]);
                        }
                    }
                }
            } else {
                // ---------------------- rows of 64 bytes through shared memory: a warp then stores 8 rows at once
                constexpr uint32_t kBytesEach = kEpilogue == kOutF32 ? 4u : 2u;
                constexpr uint32_t kPer = 64u / kBytesEach;            // elements per pass
                unsigned char *mine = base + L::kStore + (warp - 4u) * (kStoreBytes / kSumWarps);
                const bool vector = (a.n * kBytesEach) % 16u == 0u && ((uintptr_t)a.out & 15u) == 0u;
#pragma unroll
                for (uint32_t pass = 0; pass < 128u / kPer; pass++) {
#pragma unroll
                    for (uint32_t c = 0; c < 4u; c++) {
                        uint4 v;
                        if (kEpilogue == kOutF32) {
                            const uint64_t x = sum[pass * 8u + c * 2u], y = sum[pass * 8u + c * 2u + 1u];
                            v = make_uint4((uint32_t)x, (uint32_t)(x >> 32), (uint32_t)y, (uint32_t)(y >> 32));
                        } else {
                            const uint64_t *p = sum + pass * 16u + c * 4u;
                            v = make_uint4(bf16x2(lo2(p[0]), hi2(p[0])), bf16x2(lo2(p[1]), hi2(p[1])),
                                           bf16x2(lo2(p[2]), hi2(p[2])), bf16x2(lo2(p[3]), hi2(p[3])));
                        }
                        *reinterpret_cast<uint4 *>(mine + lane * 64u + ((c ^ ((lane >> 1) & 3u)) * 16u)) = v;
                    }
                    __syncwarp();
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) {
                        const uint32_t r = i * 8u + lane / 4u, c = lane % 4u;
                        const uint4 v = *reinterpret_cast<const uint4 *>(mine + r * 64u + ((c ^ ((r >> 1) & 3u)) * 16u));
                        const uint32_t column = it.column + first + pass * kPer + c * (16u / kBytesEach);
                        if (32u * q + r >= it.rows || column >= a.n) continue;
                        const uint64_t to = (uint64_t)(it.row + 32u * q + r) * a.n + column;
                        if (kEpilogue == kOutF32) {
                            float *out = (float *)a.out + to;
                            const float f[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
                            if (vector) {
                                float4 o = a.accumulate ? *reinterpret_cast<const float4 *>(out) : make_float4(0.f, 0.f, 0.f, 0.f);
                                if (a.accumulate) o = make_float4(o.x + f[0], o.y + f[1], o.z + f[2], o.w + f[3]);
                                else o = make_float4(f[0], f[1], f[2], f[3]);
                                *reinterpret_cast<float4 *>(out) = o;
                            } else {
#pragma unroll
                                for (uint32_t j = 0; j < 4u; j++) {
                                    if (column + j < a.n) out[j] = a.accumulate ? out[j] + f[j] : f[j];
                                }
                            }
                        } else {
                            uint16_t *out = (uint16_t *)a.out + to;
                            if (vector) {
                                *reinterpret_cast<uint4 *>(out) = v;
                            } else {
                                const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (uint32_t j = 0; j < 8u; j++) {
                                    if (column + j < a.n) out[j] = (uint16_t)(word[j / 2u] >> (16u * (j & 1u)));
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (kSplit) {
            // the parts' sums, in ascending order of the depth; each block adds its share of the item
            __syncwarp();
            cluster_barrier();
            const Item it = item_of(0u);
            constexpr uint32_t kUnits = BN / 4u;
            const uint32_t size = cluster_size(), all = it.rows * kUnits;
            const uint32_t share = (all + size - 1u) / size, begin = cluster_rank() * share, end = min(all, begin + share);
            const bool vector = a.n % 4u == 0u && ((uintptr_t)a.out & (kEpilogue == kOutF32 ? 15u : 7u)) == 0u;
            for (uint32_t e = begin + threadIdx.x - 4u * kWarp; e < end; e += kSumWarps * kWarp) {
                const uint32_t row = e / kUnits, unit = e % kUnits, c = it.column + unit * 4u;
                if (c >= a.n) continue;
                const float *part = reinterpret_cast<const float *>(base) + (row * kUnits + (unit ^ (row & 7u))) * 4u;
                float4 v[kMaxSplits];
#pragma unroll
                for (uint32_t r = 0; r < kMaxSplits; r++) v[r] = r < size ? cluster_load4(part, r) : make_float4(0.f, 0.f, 0.f, 0.f);
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
                const uint64_t to = (uint64_t)(it.row + row) * a.n + c;
                if (kEpilogue == kOutF32) store4((float *)a.out + to, sum, a.n - c, vector, a.accumulate);
                else store4((uint16_t *)a.out + to, sum, a.n - c, vector, 0);
            }
            cluster_barrier();                                           // nobody leaves while its sums are read
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag != 0u) atomicExch(&g_fp8_wide_status, 1u);
    if (warp == 1u) {
        tc_fence_after();
        tmem_dealloc(tmem, 512u);
    }
}

WideArgs args_of(const Product &p, uint32_t columns) {
    WideArgs a{};
    a.out = p.out;
    a.out_scales = (float *)p.out_scales;
    a.a_scales = (const float *)p.a_scales;
    a.b_scales = (const float *)p.b_scales;
    a.b2_scales = (const float *)p.b2_scales;
    a.offsets = p.offsets;
    a.groups = p.groups;
    a.rows = p.rows;
    a.n = p.n;
    a.k = p.k;
    a.column_items = (p.n + columns - 1u) / columns;
    a.b_ready = p.b_ready;
    a.accumulate = p.accumulate;
    a.activation = p.activation;
    a.beta = p.beta;
    a.linear_beta = p.linear_beta;
    a.by_beta = 1.0f / p.beta;
    a.by_linear_beta = 1.0f / p.linear_beta;
    return a;
}

struct Maps {
    CUtensorMap a, b, b2;
    bool make(const Product &p) {
        const uint64_t b_rows = (uint64_t)p.groups * p.n;
        return map_codes(&a, p.a, p.rows, p.k, BM) && map_codes(&b, p.b, b_rows, p.k, kBlock) &&
               map_codes(&b2, p.b2 ? p.b2 : p.b, b_rows, p.k, kBlock);
    }
};

template <int kEpilogue>
bool launch_grouped(const Product &p, cudaStream_t stream) {
    Maps m;
    if (!m.make(p)) return false;
    const WideArgs a = args_of(p, kEpilogue == kOutActivated ? kBlock : BN);
    const uint64_t items = ((uint64_t)(p.rows + BM - 1u) / BM + p.groups) * a.column_items;
    auto kernel = fp8_wide_kernel<kEpilogue, false, false>;
    constexpr uint32_t kBytes = Layout<false>::kBytes;
    return items <= 0x7fffffffull && set_max_dynamic_smem((const void *)kernel, kBytes) &&
           launch_chained(kernel, (uint32_t)std::min<uint64_t>(items, sm_count()), kThreads<kEpilogue>, kBytes, stream, m.a, m.b, m.b2, a);
}

// One matrix.  Every SM takes the same number of whole items; what is left, or all where there are fewer items than SMs,
// is split along the depth if that is sooner done than one more round of whole items.  A step takes 0.44 us where few
// blocks run, and the sums' way through the cluster 3 us (7 steps).  Measured, without / with: 128 rows of 7168 x 7168
// 26.1 / 17.1 us, 512 of 2048 x 7168 26.4 / 15.6.
template <int kEpilogue, bool kColumnScales>
bool launch_whole(const Product &p, cudaStream_t stream) {
    Maps m;
    if (!m.make(p)) return false;
    auto whole = fp8_wide_kernel<kEpilogue, kColumnScales, false>, split = fp8_wide_kernel<kEpilogue, kColumnScales, true>;
    constexpr uint32_t kBytes = Layout<kColumnScales>::kBytes, kFixed = 7u;
    if (!set_max_dynamic_smem((const void *)whole, kBytes) || !set_max_dynamic_smem((const void *)split, kBytes)) return false;
    WideArgs a = args_of(p, BN);
    const uint32_t sms = (uint32_t)sm_count(), blocks = blocks_of(p.k);
    const uint64_t items = (uint64_t)((p.rows + BM - 1u) / BM) * a.column_items;
    if (items > 0x7fffffffull) return false;
    const uint32_t left = (uint32_t)(items % sms);
    uint32_t parts = 1u;
    if (left != 0u && left * 2u <= sms) {          // two rounds of clusters take longer than they should: 384 rows of 7168 x 7168 34.3 us, whole 28.2
        parts = best_parts(left, blocks, kSlotBlocks, kFixed, active_clusters((const void *)split, kThreads<kEpilogue>, kBytes));
    }
    a.split_blocks = ((blocks + parts - 1u) / parts + kSlotBlocks - 1u) / kSlotBlocks * kSlotBlocks;
    const bool cut = parts > 1u && a.split_blocks + kFixed < blocks;
    a.items = (uint32_t)items - (cut ? left : 0u);
    if (a.items != 0u) {
        if (!launch_chained(whole, std::min(a.items, sms), kThreads<kEpilogue>, kBytes, stream, m.a, m.b, m.b2, a)) return false;
        a.b_ready = true;                          // the launch in front is then the one above
    }
    a.first_item = a.items;
    return !cut || launch_chained_cluster(split, dim3(parts, left), kThreads<kEpilogue>, dim3(parts, 1, 1), kBytes, stream, m.a, m.b, m.b2, a);
}

}  // namespace

bool k3::fp8::wide_product(const Product &p, cudaStream_t stream) {
    if (p.epilogue == kOutActivated) return launch_grouped<kOutActivated>(p, stream);
    if (p.offsets) return launch_grouped<kOutF32>(p, stream);
    if (p.b_scale_layout == K3_MOE_FP8_ROWS) {
        return p.epilogue == kOutF32 ? launch_whole<kOutF32, true>(p, stream) : launch_whole<kOutBf16, true>(p, stream);
    }
    return p.epilogue == kOutF32 ? launch_whole<kOutF32, false>(p, stream) : launch_whole<kOutBf16, false>(p, stream);
}

uint32_t k3_fp8_wide_status() {
    uint32_t v = 0xffffffffu;
    if (cudaMemcpyFromSymbol(&v, g_fp8_wide_status, sizeof(v)) != cudaSuccess) (void)cudaGetLastError();
    return v;
}

bool k3_fp8_wide_status_clear() {
    const uint32_t zero = 0u;
    const bool ok = cudaMemcpyToSymbol(g_fp8_wide_status, &zero, sizeof(zero)) == cudaSuccess;
    if (!ok) (void)cudaGetLastError();
    return ok;
}
