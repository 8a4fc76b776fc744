// Expert load, balance loss and the router's gradient (include/k3_moe_balance.h has the formulas).
//
// All three are one pass over logits f32 [tokens, experts], so HBM bounds them; 32768 x 896 takes 31 us forward (3.8 TB/s), where
// the exponentials' chains stand beside the loads, and 50 us backward (4.7 TB/s).  A warp takes a token's
// row: lane l holds experts 4 l .. 4 l + 3 of every 128 (or l of every 32 where rows are not whole 16-byte
// units), so the row's sums are shuffles, and in the forward pass the sums over tokens stay in the same
// registers from token to token.
//
// Sums over tokens have a fixed order.  Block b takes tokens [b C, (b + 1) C); at the end of its range
// and at each end of a sequence inside it the block writes what it has as a partial row.  Block b and
// sequence s share the partial row b + s: along the tokens each step raises one of the two, so no two
// pairs meet in a row and there are at most blocks + sequences of them.  A second kernel adds a
// sequence's partial rows, in ascending order, and forms the loss.
#include "k3_common.cuh"
#include "k3_grouped.h"
#include "k3_moe_balance.h"

#include <algorithm>

using namespace k3;

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / kWarp;
constexpr uint32_t kMaxExperts = 1024;
constexpr float kTiny = 1e-20f;
constexpr uint32_t kForwardStages = 3, kBackwardStages = 2;   // rows of a warp in shared memory

__device__ uint32_t g_balance_status = 0;          // 2: an expert id >= experts

// Blocks of the backward pass on an SM, two in the forward pass.  30000 x 160 in one sequence, us with two / three / four:
// backward 19.6 / 18.0 / 18.1, forward 10.0 / 10.1 / 25.7, and its second stage, which has a partial row for each
// block, 13.3 / 18.8 / 23.8.  32768 x 896 in 16: forward 31 / 38 / 41, second stage 7.2 / 6.5 / 7.1.
constexpr uint32_t kForwardPerSm = 2;
constexpr uint32_t backward_per_sm(uint32_t groups) { return groups <= 4u ? 3u : 2u; }

struct Shape {
    uint32_t tokens, sequences, experts, top_k;
    uint32_t chunk;                                // tokens per block
    int softmax;
};

// Scores with the fast base-2 exponential and reciprocal: 6e-7 of a score down to 2^-126, below which it is 0.  The
// exponent's product with log2 e would be off by 2^-24 of itself, 5e-6 of a score at a logit of -80, so what it rounds
// away goes into the result as a factor (5 us of 78 at 32768 x 896).  With expf, a rounded quotient and single
// operations the pass over the logits was bound by its instructions, 32768 x 896 forward and backward 198 us.
constexpr float kLn2 = 0.693147181f;
// a, but 200 where it is larger (e^-200 is 0, and an infinity would leave no remainder); NaN stays
K3_DEVINL float bounded(float a) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(200.0f));
    return r;
}
// e^-a of 0 <= a <= 200
K3_DEVINL float exp_negative(float a) {
    const float t = __fmul_rn(a, kLog2E), rest = fmaf(a, -kLog2ELow, fmaf(a, -kLog2E, t)), e = exp2_fast(-t);
    return fmaf(e * kLn2, rest, e);
}
K3_DEVINL uint64_t exp_negative2(uint64_t a) {
    const uint64_t t = mul2(a, both2(kLog2E)), rest = fma2(a, both2(-kLog2ELow), fma2(a, both2(-kLog2E), t));
    const uint64_t e = pack2(exp2_fast(-lo2(t)), exp2_fast(-hi2(t)));
    return fma2(mul2(e, both2(kLn2)), rest, e);
}
K3_DEVINL float sigmoid(float x) {
    const float e = exp_negative(bounded(fabsf(x))), r = reciprocal_fast(1.0f + e);
    return x > 0.0f ? r : e * r;
}

template <int kBytes>
K3_DEVINL void copy_async(float *to, const float *from) {
    const uint32_t addr = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(addr), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(addr), "l"(from) : "memory");
}
K3_DEVINL void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
K3_DEVINL void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

struct Softmax {
    float top, over;                               // a score is exp(logit - top) * over
};

// A warp's row: kV groups of four experts per lane, neighbours (kVector) or 32 apart, two to a register pair.
template <uint32_t kV, bool kVector>
struct Row {
    uint64_t v[kV * 2u];
    // expert of element i of this lane
    static K3_DEVINL uint32_t expert(uint32_t i, uint32_t lane) {
        return kVector ? (i / 4u) * 128u + lane * 4u + i % 4u : i * 32u + lane;
    }
    // group g (elements 4 g .. 4 g + 3) of a row in memory, and back
    template <typename T>
    static K3_DEVINL void get(uint64_t (&to)[2], const T *row, uint32_t experts, uint32_t lane, uint32_t g, float fill) {
        float q[4];
        if (kVector) {
            const uint32_t e = expert(4u * g, lane);
            uint4 bits = make_uint4(0u, 0u, 0u, 0u);
            if (e < experts) bits = *reinterpret_cast<const uint4 *>(row + e);
            q[0] = e < experts ? value(bits.x, row) : fill;
            q[1] = e < experts ? value(bits.y, row) : fill;
            q[2] = e < experts ? value(bits.z, row) : fill;
            q[3] = e < experts ? value(bits.w, row) : fill;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) q[j] = expert(4u * g + j, lane) < experts ? (float)row[expert(4u * g + j, lane)] : fill;
        }
        to[0] = pack2(q[0], q[1]);
        to[1] = pack2(q[2], q[3]);
    }
    static K3_DEVINL void put(float *row, const uint64_t (&from)[2], uint32_t experts, uint32_t lane, uint32_t g) {
        const float q[4] = {lo2(from[0]), hi2(from[0]), lo2(from[1]), hi2(from[1])};
        if (kVector) {
            const uint32_t e = expert(4u * g, lane);
            if (e < experts) *reinterpret_cast<float4 *>(row + e) = make_float4(q[0], q[1], q[2], q[3]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) {
                if (expert(4u * g + j, lane) < experts) row[expert(4u * g + j, lane)] = q[j];
            }
        }
    }
    // The same row by asynchronous copies into shared memory (kV * 128 floats; what lies past the experts stays).
    // A lane copies what it reads itself.
    static K3_DEVINL void fetch(float *to, const float *row, uint32_t experts, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < kV * 4u; i += kVector ? 4u : 1u) {
            const uint32_t e = expert(i, lane);
            if (e < experts) copy_async<kVector ? 16 : 4>(to + e, row + e);
        }
    }
    template <typename T>
    K3_DEVINL void load(const T *row, uint32_t experts, uint32_t lane, float fill) {
#pragma unroll
        for (uint32_t g = 0; g < kV; g++) {
            uint64_t q[2];
            get(q, row, experts, lane, g, fill);
            v[2u * g] = q[0];
            v[2u * g + 1u] = q[1];
        }
    }
    K3_DEVINL void store(float *row, uint32_t experts, uint32_t lane) const {
#pragma unroll
        for (uint32_t g = 0; g < kV; g++) {
            const uint64_t q[2] = {v[2u * g], v[2u * g + 1u]};
            put(row, q, experts, lane, g);
        }
    }
    static K3_DEVINL float value(uint32_t bits, const float *) { return __uint_as_float(bits); }
    static K3_DEVINL float value(uint32_t bits, const uint32_t *) { return (float)bits; }
    K3_DEVINL void fill(float x) {
#pragma unroll
        for (uint32_t i = 0; i < kV * 2u; i++) v[i] = pack2(x, x);
    }
    K3_DEVINL void scale(float x) {
        const uint64_t by = pack2(x, x);
#pragma unroll
        for (uint32_t i = 0; i < kV * 2u; i++) v[i] = mul2(v[i], by);
    }
    K3_DEVINL float sum() const {
        uint64_t s = v[0];
#pragma unroll
        for (uint32_t i = 1; i < kV * 2u; i++) s = add2(s, v[i]);
        return warp_sum(lo2(s) + hi2(s));
    }
    // logits -> scores; experts past the end have the logit -inf and get the score 0.  kSmaller: of a sigmoid s the
    // smaller of s and 1 - s, negative (-0 too) where that is 1 - s: the derivative s (1 - s) of a score near 1 has no
    // bits left in s.
    template <bool kSmaller>
    K3_DEVINL Softmax scores(int softmax) {
        Softmax f{0.f, 0.f};
        if (!softmax) {
#pragma unroll
            for (uint32_t i = 0; i < kV * 2u; i++) {
                const float x = lo2(v[i]), y = hi2(v[i]);
                const uint64_t e = exp_negative2(pack2(bounded(fabsf(x)), bounded(fabsf(y)))), d = add2(e, both2(1.0f));
                const uint64_t r = pack2(reciprocal_fast(lo2(d)), reciprocal_fast(hi2(d))), small = mul2(e, r);
                v[i] = kSmaller ? pack2(x > 0.0f ? -lo2(small) : lo2(small), y > 0.0f ? -hi2(small) : hi2(small))
                                : pack2(x > 0.0f ? lo2(r) : lo2(small), y > 0.0f ? hi2(r) : hi2(small));
            }
            return f;
        }
        f.top = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < kV * 2u; i++) f.top = fmaxf(f.top, fmaxf(lo2(v[i]), hi2(v[i])));
        f.top = warp_max(f.top);
        if (f.top == -INFINITY) {                  // every logit is -inf, or NaN, which fmaxf drops
            float s = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < kV * 2u; i++) {
                const float a = lo2(v[i]), b = hi2(v[i]);
                s += (a != a ? a : 0.f) + (b != b ? b : 0.f);
            }
            f.top = 0.f;
            f.over = warp_sum(s);                  // 0, or NaN
            fill(f.over);
            return f;
        }
#pragma unroll
        for (uint32_t i = 0; i < kV * 2u; i++) {
            const uint64_t less = fma2(v[i], both2(-1.0f), both2(f.top));
            v[i] = exp_negative2(pack2(bounded(lo2(less)), bounded(hi2(less))));
        }
        f.over = 1.0f / sum();
        scale(f.over);
        return f;
    }
};

// Sigmoids of what scores<true>() gives for them, and their derivatives
K3_DEVINL float sigmoid_of(float smaller) { return (int32_t)__float_as_uint(smaller) < 0 ? 1.0f + smaller : smaller; }
K3_DEVINL uint64_t sigmoid_of2(uint64_t smaller) { return pack2(sigmoid_of(lo2(smaller)), sigmoid_of(hi2(smaller))); }
K3_DEVINL uint64_t derivative_of2(uint64_t smaller) {
    const uint64_t y = smaller & 0x7fffffff7fffffffull;
    return mul2(y, fma2(y, both2(-1.0f), both2(1.0f)));
}

// the sequence that holds `token`: the last one that starts at or before it (sequences - 1 at most)
K3_DEVINL uint32_t sequence_of(const uint32_t *offsets, uint32_t sequences, uint32_t token) {
    if (offsets == nullptr) return 0u;
    uint32_t lo = 0u, hi = sequences;              // offsets[lo] <= token < offsets[hi]
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (offsets[mid] <= token) lo = mid; else hi = mid;
    }
    return lo;
}
K3_DEVINL uint32_t begin_of(const uint32_t *offsets, uint32_t s) { return offsets ? offsets[s] : 0u; }
K3_DEVINL uint32_t end_of(const uint32_t *offsets, uint32_t s, uint32_t tokens) {
    return offsets ? min(offsets[s + 1u], tokens) : tokens;
}

// ---------------------------------------------------------------------------------------- forward
// Shared memory of a block: counts u32 [kPitch], then rows of logits [kWarps][kForwardStages][kPitch], whose place the
// warps' sums [kWarps][kPitch] take at the end.
//
// The block's tokens first + warp, first + warp + stride, .. below `end`: their routes into counts, the sums of their
// scores over Z into the warps' sums.  All threads of the block; a barrier stands at the end.
template <uint32_t kV, bool kVector>
K3_DEVINL void sum_tokens(float *rows_s, const float *logits, const uint32_t *ids, uint32_t first, uint32_t stride, uint32_t end,
                          const Shape &a) {
    constexpr uint32_t kPitch = kV * 128u;
    uint32_t *counts_s = reinterpret_cast<uint32_t *>(rows_s);
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    float *mine = rows_s + kPitch + warp * (kForwardStages * kPitch), *sums_s = rows_s + kPitch;
    auto fetch = [&](uint32_t u, uint32_t stage) {
        if (u < end) Row<kV, kVector>::fetch(mine + stage * kPitch, logits + (uint64_t)u * a.experts, a.experts, lane);
        copies_commit();
    };
    Row<kV, kVector> acc;
    acc.fill(0.f);
    const uint32_t t = first + warp;
    if (logits) {
#pragma unroll
        for (uint32_t g = 0; g + 1u < kForwardStages; g++) fetch(t + g * stride, g);
        for (uint32_t e = a.experts + lane; e < kPitch; e += kWarp) {
            for (uint32_t g = 0; g < kForwardStages; g++) mine[g * kPitch + e] = -INFINITY;
        }
    }
    for (uint32_t e = threadIdx.x; e < a.experts; e += kThreads) counts_s[e] = 0u;
    __syncthreads();
    uint32_t stage = 0u, next_id = t < end && lane < a.top_k ? ids[(uint64_t)t * a.top_k + lane] : 0u;
    for (uint32_t u = t; u < end; u += stride) {
        const uint32_t id = next_id;
        if (u + stride < end && lane < a.top_k) next_id = ids[(uint64_t)(u + stride) * a.top_k + lane];
        if (logits) {
            fetch(u + (kForwardStages - 1u) * stride, stage == 0u ? kForwardStages - 1u : stage - 1u);
            copies_wait<kForwardStages - 1>();
            Row<kV, kVector> p;
            p.load(mine + stage * kPitch, kPitch, lane, 0.f);
            p.template scores<false>(a.softmax);
            const float r = a.softmax ? 1.0f : reciprocal_fast(kTiny + p.sum());
            const uint64_t r2 = pack2(r, r);
#pragma unroll
            for (uint32_t i = 0; i < kV * 2u; i++) acc.v[i] = fma2(p.v[i], r2, acc.v[i]);
            if (++stage == kForwardStages) stage = 0u;
        }
        if (lane < a.top_k) {
            if (id < a.experts) atomicAdd(&counts_s[id], 1u);
            else g_balance_status = 2u;
        }
    }
    if (logits) {
        copies_wait<0>();
        __syncthreads();                           // everyone's rows have been read: the sums take their place
        acc.store(sums_s + warp * kPitch, kPitch, lane);
    }
    __syncthreads();
}

template <uint32_t kV, bool kVector>
__global__ void __launch_bounds__(kThreads, kForwardPerSm)
balance_tokens_kernel(float *part_sums, uint32_t *part_counts, const float *logits, const uint32_t *ids, const uint32_t *offsets,
                      Shape a) {
    constexpr uint32_t kPitch = kV * 128u;
    extern __shared__ __align__(16) float rows_s[];
    pdl_wait();
    uint32_t t = blockIdx.x * a.chunk;
    const uint32_t last = min(a.tokens, t + a.chunk);
    uint32_t s = sequence_of(offsets, a.sequences, t);
    for (; t < last && s < a.sequences; s++) {
        const uint32_t end = min(last, end_of(offsets, s, a.tokens));
        if (end <= t) continue;                    // an empty sequence, or tokens past the last one
        sum_tokens<kV, kVector>(rows_s, logits, ids, t, kWarps, end, a);
        pdl_trigger();                             // the second stage's blocks may take places as these leave
        const uint64_t to = (uint64_t)(blockIdx.x + s) * a.experts;
        for (uint32_t e = threadIdx.x; e < a.experts; e += kThreads) {
            part_counts[to + e] = reinterpret_cast<uint32_t *>(rows_s)[e];
            if (logits) {
                float sum = 0.f;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; w++) sum += rows_s[(1u + w) * kPitch + e];
                part_sums[to + e] = sum;
            }
        }
        __syncthreads();
        t = end;
    }
}

// Few tokens: one cluster of eight blocks per sequence does both stages, with the blocks' partial rows in shared memory.
// The second launch takes longer than that while few tokens are each warp's: 257 tokens x 160 experts 4.6 us instead of
// 3.7 + 3.8, but 1000 tokens x 896 experts in one sequence 19.2 instead of 3.5 + 8.5.
constexpr uint32_t kFewTokens = 512, kFewSequences = 64, kCluster = 8;

template <uint32_t kV, bool kVector>
__global__ void __launch_bounds__(kThreads, 2)
balance_few_kernel(uint32_t *counts, float *loss, float *means, const float *logits, const uint32_t *ids, const uint32_t *offsets,
                   Shape a, float coefficient) {
    constexpr uint32_t kPitch = kV * 128u;
    extern __shared__ __align__(16) float rows_s[];
    __shared__ float part[kPitch], total[4], mine;
    __shared__ uint32_t part_counts[kPitch];
    pdl_wait();
    pdl_trigger();
    const uint32_t s = blockIdx.y, rank = cluster_rank(), begin = begin_of(offsets, s), end = end_of(offsets, s, a.tokens);
    const uint32_t length = end > begin ? end - begin : 0u;
    sum_tokens<kV, kVector>(rows_s, logits, ids, begin + rank * kWarps, kCluster * kWarps, begin + length, a);
    for (uint32_t e = threadIdx.x; e < a.experts; e += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t w = 0; logits && w < kWarps; w++) sum += rows_s[(1u + w) * kPitch + e];
        part[e] = sum;
        part_counts[e] = reinterpret_cast<uint32_t *>(rows_s)[e];
    }
    __syncthreads();
    cluster_barrier();
    if (threadIdx.x < 128u) {                      // block `rank` has experts rank * 128 .. of the sequence
        const uint32_t e = rank * 128u + threadIdx.x;
        float product = 0.f;
        if (e < a.experts) {
            uint32_t n = 0u;
            float sum = 0.f;
#pragma unroll
            for (uint32_t r = 0; r < kCluster; r++) {
                n += __float_as_uint(cluster_load(reinterpret_cast<const float *>(part_counts) + e, r));
                if (logits) sum += cluster_load(part + e, r);
            }
            const float mean = length ? sum / (float)length : 0.f;
            counts[(uint64_t)s * a.experts + e] = n;
            if (logits) means[(uint64_t)s * a.experts + e] = mean;
            product = (float)n * mean;
        }
        product = warp_sum(product);
        if (threadIdx.x % kWarp == 0u) total[threadIdx.x / kWarp] = product;
    }
    __syncthreads();
    if (threadIdx.x == 0u) mine = total[0] + total[1] + total[2] + total[3];
    __syncthreads();
    cluster_barrier();
    if (logits && rank == 0u && threadIdx.x == 0u) {
        float all = 0.f;
        for (uint32_t r = 0; r < kCluster; r++) all += cluster_load(&mine, r);
        loss[s] = length ? coefficient * all * ((float)a.experts / ((float)a.top_k * (float)length)) : 0.f;
    }
    cluster_barrier();                             // nobody leaves while its sums are read
}

// A cluster of blocks per sequence, 128 experts each; eight groups of threads take every eighth partial row.
__global__ void __launch_bounds__(1024)
balance_sequences_kernel(uint32_t *counts, float *loss, float *means, const float *part_sums, const uint32_t *part_counts,
                         const uint32_t *offsets, Shape a, float coefficient) {
    __shared__ float sums_s[8][128];
    __shared__ uint32_t counts_s[8][128];
    __shared__ float total[4], mine;
    pdl_wait();
    pdl_trigger();
    const uint32_t s = blockIdx.y, begin = begin_of(offsets, s), end = end_of(offsets, s, a.tokens);
    const uint32_t length = end > begin ? end - begin : 0u;
    const uint32_t column = threadIdx.x % 128u, group = threadIdx.x / 128u, e = blockIdx.x * 128u + column;
    uint32_t n = 0u;
    float sum = 0.f;
    if (length && e < a.experts) {
        const uint32_t last = (end - 1u) / a.chunk;
#pragma unroll 4
        for (uint32_t b = begin / a.chunk + group; b <= last; b += 8u) {
            const uint64_t at = (uint64_t)(b + s) * a.experts + e;
            n += part_counts[at];
            if (means) sum += part_sums[at];
        }
    }
    sums_s[group][column] = sum;
    counts_s[group][column] = n;
    __syncthreads();
    if (threadIdx.x < 128u) {
#pragma unroll
        for (uint32_t g = 1; g < 8u; g++) {
            n += counts_s[g][column];
            sum += sums_s[g][column];
        }
        const float mean = length ? sum / (float)length : 0.f;
        if (e < a.experts) {
            counts[(uint64_t)s * a.experts + e] = n;
            if (means) means[(uint64_t)s * a.experts + e] = mean;
        }
        const float part = warp_sum((float)n * mean);              // an expert past the end has none
        if (threadIdx.x % kWarp == 0u) total[threadIdx.x / kWarp] = part;
    }
    if (!means) return;
    __syncthreads();
    if (threadIdx.x == 0u) mine = total[0] + total[1] + total[2] + total[3];
    __syncthreads();
    cluster_barrier();
    if (cluster_rank() == 0u && threadIdx.x == 0u) {
        float all = 0.f;
        for (uint32_t r = 0; r < cluster_size(); r++) all += cluster_load(&mine, r);
        loss[s] = length ? coefficient * all * ((float)a.experts / ((float)a.top_k * (float)length)) : 0.f;
    }
    cluster_barrier();                             // nobody leaves while its sum is read
}

// --------------------------------------------------------------------------------------- backward
// A warp's tokens follow one another, so a sequence's shares f stay in registers while it lasts.
template <uint32_t kV, bool kVector>
__global__ void __launch_bounds__(kThreads, backward_per_sm(kV))
router_backward_kernel(float *d_logits, const float *logits, const uint32_t *ids, const uint32_t *counts, const uint32_t *offsets,
                       const float *d_loss, const float *d_weights, Shape a, float coefficient, float route_scale) {
    constexpr uint32_t kPitch = kV * 128u;
    // per warp: kBackwardStages rows of logits, and a row of zeros but for the chosen of the token at hand
    extern __shared__ __align__(16) float rows_s[];
    const uint32_t warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    float *mine = rows_s + warp * ((kBackwardStages + 1u) * kPitch), *row_s = mine + kBackwardStages * kPitch;
    for (uint32_t e = lane; e < kPitch; e += kWarp) {
        row_s[e] = 0.f;
        for (uint32_t g = 0; e >= a.experts && g < kBackwardStages; g++) mine[g * kPitch + e] = -INFINITY;
    }
    __syncwarp();
    pdl_wait();
    const uint32_t first = (blockIdx.x * kWarps + warp) * a.chunk;
    if (first >= a.tokens) return;
    const uint32_t last = min(a.tokens, first + a.chunk);
    uint32_t s = 0u, end = first;
    Row<kV, kVector> f;
    float c = 0.f;
    uint32_t next_id = 0xffffffffu;
    float next_w = 0.f;
    // a token's row, and what lane r needs of its r-th choice
    auto fetch = [&](uint32_t t, uint32_t stage) {
        if (t < last) Row<kV, kVector>::fetch(mine + stage * kPitch, logits + (uint64_t)t * a.experts, a.experts, lane);
        copies_commit();
    };
    auto fetch_choice = [&](uint32_t t) {          // neither load waits for the other; the id is looked at when its token comes
        if (d_weights && t < last && lane < a.top_k) {
            next_id = ids[(uint64_t)t * a.top_k + lane];
            next_w = d_weights[(uint64_t)t * a.top_k + lane];
        }
    };
#pragma unroll
    for (uint32_t g = 0; g + 1u < kBackwardStages; g++) fetch(first + g, g);
    fetch_choice(first);
    uint32_t stage = 0u;
    for (uint32_t t = first; t < last; t++) {
        fetch(t + kBackwardStages - 1u, stage == 0u ? kBackwardStages - 1u : stage - 1u);
        const uint32_t id = next_id;
        const float w = id < a.experts ? next_w : 0.f;
        fetch_choice(t + 1u);
        copies_wait<kBackwardStages - 1>();
        __syncwarp();                              // the lanes' chosen lie in one another's copies
        const float l = id < a.experts ? mine[stage * kPitch + id] : 0.f;
        Row<kV, kVector> p;
        p.load(mine + stage * kPitch, kPitch, lane, 0.f);
        if (++stage == kBackwardStages) stage = 0u;
        if (d_loss && t >= end) {
            s = sequence_of(offsets, a.sequences, t);
            const uint32_t begin = begin_of(offsets, s);
            end = end_of(offsets, s, a.tokens);
            if (t >= end) {                        // past the last sequence: no loss
                end = a.tokens;
                c = 0.f;
                f.fill(0.f);
            } else {
                const float length = (float)(end - begin), scale = (float)a.experts / ((float)a.top_k * length);
                c = coefficient * d_loss[s] / length;
                f.load(counts + (uint64_t)s * a.experts, a.experts, lane, 0.f);
                f.scale(scale);
            }
        }
        const Softmax soft = p.template scores<true>(a.softmax);
        // the loss by a score is by (f - mean)
        float by = c, mean = 0.f;
        if (d_loss && !a.softmax) {
            uint64_t z = pack2(0.f, 0.f), fp = z;
#pragma unroll
            for (uint32_t i = 0; i < kV * 2u; i++) {
                const uint64_t score = sigmoid_of2(p.v[i]);
                z = add2(z, score);
                fp = fma2(f.v[i], score, fp);
            }
            const float r = reciprocal_fast(kTiny + warp_sum(lo2(z) + hi2(z)));
            mean = warp_sum(lo2(fp) + hi2(fp)) * r;
            by = c * r;
        }
        const bool chosen = id < a.experts;
        if (d_weights) {
            if (lane < a.top_k && !chosen) g_balance_status = 2u;
            // the weights' share at the chosen, through shared memory to the lanes that hold them
            const float si = !chosen ? 0.f : a.softmax ? exp_negative(bounded(soft.top - l)) * soft.over : sigmoid(l);
            // (w - sum w s / D) / D with D = tiny + sum s, of the weights' gradients less that of the largest score: where
            // they are equal, as a single choice is with itself, the difference is 0 and w tiny / D is left
            const uint32_t bits = __float_as_uint(si), most = __reduce_max_sync(0xffffffffu, bits);
            const uint32_t holders = __ballot_sync(0xffffffffu, chosen && bits == most);
            const float w0 = holders ? __shfl_sync(0xffffffffu, w, __ffs(holders) - 1) : 0.f, more = chosen ? w - w0 : 0.f;
            const float all = warp_sum(si), weighted = warp_sum(more * si);
            const float under = reciprocal_fast(kTiny + all);
            const float share = route_scale * (more - weighted * under + w0 * (kTiny * under)) * under;
            // an expert named twice keeps one of the lanes' numbers (with __match_any_sync for this 30000 x 160 took 32 us
            // instead of 20)
            if (chosen) row_s[id] = __uint_as_float(lane);
            __syncwarp();
            const bool other = chosen && __float_as_uint(row_s[id]) != lane;
            if (!__any_sync(0xffffffffu, other)) {
                if (chosen) row_s[id] = share;
            } else {                               // one after the other
                if (chosen) row_s[id] = 0.f;
                __syncwarp();
                for (uint32_t r = 0; r < a.top_k; r++) {
                    if (lane == r && chosen) row_s[id] += share;
                    __syncwarp();
                }
            }
            __syncwarp();
        }
        // by the scores of group g
        const uint64_t by2 = pack2(by, by), less = pack2(-mean, -mean);
        auto by_scores = [&](uint64_t (&d)[2], uint32_t g) {
            if (d_weights) {
                Row<kV, kVector>::get(d, row_s, kPitch, lane, g, 0.f);
            } else {
                d[0] = d[1] = pack2(0.f, 0.f);
            }
            if (d_loss) {
                d[0] = fma2(by2, add2(f.v[2u * g], less), d[0]);
                d[1] = fma2(by2, add2(f.v[2u * g + 1u], less), d[1]);
            }
        };
        // softmax: p (d - sum d p) of the d less that of the largest score, so that a score near 1 keeps the small sum of
        // the others'.  The largest have the exponential 1, and so the score `over`.
        uint64_t shift = pack2(0.f, 0.f), dp = shift;
        if (a.softmax) {
            float top = -INFINITY;
#pragma unroll
            for (uint32_t g = 0; g < kV; g++) {
                uint64_t d[2];
                by_scores(d, g);
#pragma unroll
                for (uint32_t j = 0; j < 2u; j++) {
                    if (lo2(p.v[2u * g + j]) == soft.over) top = fmaxf(top, lo2(d[j]));
                    if (hi2(p.v[2u * g + j]) == soft.over) top = fmaxf(top, hi2(d[j]));
                }
            }
            shift = both2(-warp_max(top));
#pragma unroll
            for (uint32_t g = 0; g < kV; g++) {
                uint64_t d[2];
                by_scores(d, g);
                dp = fma2(add2(d[0], shift), p.v[2u * g], fma2(add2(d[1], shift), p.v[2u * g + 1u], dp));
            }
            dp = both2(-warp_sum(lo2(dp) + hi2(dp)));
        }
        float *out = d_logits + (uint64_t)t * a.experts;
#pragma unroll
        for (uint32_t g = 0; g < kV; g++) {
            uint64_t d[2];
            by_scores(d, g);
#pragma unroll
            for (uint32_t j = 0; j < 2u; j++) {
                const uint64_t q = p.v[2u * g + j];
                d[j] = a.softmax ? mul2(q, add2(add2(d[j], shift), dp)) : mul2(d[j], derivative_of2(q));
            }
            Row<kV, kVector>::put(out, d, a.experts, lane, g);
        }
        __syncwarp();
        if (d_weights && chosen) row_s[id] = 0.f;
        __syncwarp();                              // the zeros are back before the next token's shares
    }
}

bool shape_ok(uint32_t tokens, uint32_t sequences, uint32_t experts, uint32_t top_k, int score, const void *offsets) {
    return tokens != 0u && tokens <= (1u << 26) && sequences != 0u && sequences <= 65535u && (offsets || sequences == 1u) &&
           experts != 0u && experts <= kMaxExperts && top_k != 0u && top_k <= 32u && top_k <= experts &&
           (score == K3_MOE_SCORE_SIGMOID || score == K3_MOE_SCORE_SOFTMAX);
}

constexpr uint32_t groups_of(uint32_t experts) { return (experts + 127u) / 128u; }

// Blocks of the forward pass's first stage (148 SMs whatever the device: the same partial sums on any), and tokens per
// block: one per warp at least.
constexpr uint32_t kForwardBlocks = 148u * kForwardPerSm;
uint32_t forward_chunk(uint32_t tokens) { return std::max((tokens + kForwardBlocks - 1u) / kForwardBlocks, kWarps); }

struct BalanceWorkspace {
    uint64_t rows;
    size_t sums, total;
    BalanceWorkspace(uint32_t tokens, uint32_t sequences, uint32_t experts) {
        rows = std::min((tokens + kWarps - 1u) / kWarps, kForwardBlocks) + (uint64_t)sequences;   // never less for more tokens
        sums = (size_t)(rows * experts * sizeof(float) + 255u) / 256u * 256u;
        total = sums + (size_t)(rows * experts * sizeof(uint32_t));
    }
};

// The instance for a number of experts: one to eight groups of 128.
template <template <uint32_t, bool> class Pick, uint32_t kV = 1, typename... A>
bool pick(uint32_t experts, bool vector, A... args) {
    if constexpr (kV < 8u) {
        if (experts > kV * 128u) return pick<Pick, kV + 1u>(experts, vector, args...);
    }
    return vector ? Pick<kV, true>::go(args...) : Pick<kV, false>::go(args...);
}

template <uint32_t kV, bool kVector>
struct Forward {
    static bool go(float *sums, uint32_t *counts, const float *logits, const uint32_t *ids, const uint32_t *offsets, Shape a,
                   cudaStream_t stream) {
        const size_t smem = (1u + (logits ? kWarps * kForwardStages : 0u)) * kV * 128u * sizeof(float);
        return set_max_dynamic_smem((const void *)balance_tokens_kernel<kV, kVector>, smem) &&
               launch_chained(balance_tokens_kernel<kV, kVector>, (a.tokens + a.chunk - 1u) / a.chunk, kThreads, smem, stream,
                              sums, counts, logits, ids, offsets, a);
    }
};

template <uint32_t kV, bool kVector>
struct Few {
    static bool go(uint32_t *counts, float *loss, float *means, const float *logits, const uint32_t *ids, const uint32_t *offsets,
                   Shape a, float coefficient, cudaStream_t stream) {
        const size_t smem = (1u + (logits ? kWarps * kForwardStages : 0u)) * kV * 128u * sizeof(float);
        return set_max_dynamic_smem((const void *)balance_few_kernel<kV, kVector>, smem) &&
               launch_chained_cluster(balance_few_kernel<kV, kVector>, dim3(kCluster, a.sequences), kThreads, dim3(kCluster, 1, 1), smem,
                                      stream, counts, loss, means, logits, ids, offsets, a, coefficient);
    }
};

template <uint32_t kV, bool kVector>
struct Backward {
    static bool go(float *d_logits, const float *logits, const uint32_t *ids, const uint32_t *counts, const uint32_t *offsets,
                   const float *d_loss, const float *d_weights, Shape a, float coefficient, float route_scale,
                   cudaStream_t stream) {
        const size_t smem = kWarps * (kBackwardStages + 1u) * kV * 128u * sizeof(float);
        const uint32_t warps = (a.tokens + a.chunk - 1u) / a.chunk;
        return set_max_dynamic_smem((const void *)router_backward_kernel<kV, kVector>, smem) &&
               launch_chained(router_backward_kernel<kV, kVector>, (warps + kWarps - 1u) / kWarps, kThreads, smem, stream,
                              d_logits, logits, ids, counts, offsets, d_loss, d_weights, a, coefficient, route_scale);
    }
};

bool words_ok(const void *p) { return ((uintptr_t)p & 3u) == 0u; }

}  // namespace

uint32_t k3_balance_status() {
    uint32_t v = 0xffffffffu;
    if (cudaMemcpyFromSymbol(&v, g_balance_status, sizeof(v)) != cudaSuccess) (void)cudaGetLastError();
    return v;
}

bool k3_balance_status_clear() {
    const uint32_t zero = 0u;
    const bool ok = cudaMemcpyToSymbol(g_balance_status, &zero, sizeof(zero)) == cudaSuccess;
    if (!ok) (void)cudaGetLastError();
    return ok;
}

extern "C" size_t k3_moe_balance_workspace_bytes(uint32_t tokens, uint32_t sequences, uint32_t experts) {
    if (!shape_ok(tokens, sequences, experts, 1u, K3_MOE_SCORE_SIGMOID, &tokens)) return 0;
    return BalanceWorkspace(tokens, sequences, experts).total;
}

extern "C" bool k3_moe_balance(void *counts, void *loss, void *means, const void *logits, const void *ids, const void *offsets,
                               uint32_t tokens, uint32_t sequences, uint32_t experts, uint32_t top_k, int score,
                               float coefficient, void *workspace, size_t workspace_bytes, void *stream_pointer) {
    if (!shape_ok(tokens, sequences, experts, top_k, score, offsets) || !counts || !ids || !workspace ||
        (logits != nullptr) != (loss != nullptr) || (logits != nullptr) != (means != nullptr) || ((uintptr_t)workspace & 15u) != 0u ||
        !words_ok(counts) || !words_ok(loss) || !words_ok(means) || !words_ok(logits) || !words_ok(ids) || !words_ok(offsets)) {
        return false;
    }
    const BalanceWorkspace w(tokens, sequences, experts);
    if (workspace_bytes < w.total) return false;
    cudaStream_t stream = (cudaStream_t)stream_pointer;
    const Shape a{tokens, sequences, experts, top_k, forward_chunk(tokens), score};
    float *sums = (float *)workspace;
    uint32_t *part_counts = (uint32_t *)((char *)workspace + w.sums);
    const bool vector = experts % 4u == 0u && ((uintptr_t)logits & 15u) == 0u;
    if (tokens <= kFewTokens && sequences <= kFewSequences) {
        return pick<Few>(experts, vector, (uint32_t *)counts, (float *)loss, (float *)means, (const float *)logits, (const uint32_t *)ids,
                         (const uint32_t *)offsets, a, coefficient, stream);
    }
    const uint32_t slices = groups_of(experts);
    return pick<Forward>(experts, vector, sums, part_counts, (const float *)logits, (const uint32_t *)ids, (const uint32_t *)offsets,
                         a, stream) &&
           launch_chained_cluster(balance_sequences_kernel, dim3(slices, sequences), 1024, dim3(slices, 1, 1), 0, stream, (uint32_t *)counts, (float *)loss, (float *)means,
                          (const float *)sums, (const uint32_t *)part_counts, (const uint32_t *)offsets, a, coefficient);
}

extern "C" bool k3_moe_router_backward(void *d_logits, const void *logits, const void *ids, const void *counts,
                                       const void *offsets, const void *d_loss, const void *d_weights, uint32_t tokens,
                                       uint32_t sequences, uint32_t experts, uint32_t top_k, int score, float coefficient,
                                       float route_scale, void *stream) {
    if (!shape_ok(tokens, sequences, experts, top_k, score, offsets) || !d_logits || !logits || (!d_loss && !d_weights) ||
        (d_loss && !counts) || (d_weights && (!ids || !(route_scale > 0.0f))) || !words_ok(d_logits) || !words_ok(logits) ||
        !words_ok(ids) || !words_ok(counts) || !words_ok(offsets) || !words_ok(d_loss) || !words_ok(d_weights)) {
        return false;
    }
    const uint32_t warps = (uint32_t)sm_count() * backward_per_sm(groups_of(experts)) * kWarps;
    const Shape a{tokens, sequences, experts, top_k, std::max((tokens + warps - 1u) / warps, 1u), score};
    const bool vector = experts % 4u == 0u && (((uintptr_t)logits | (uintptr_t)d_logits | (uintptr_t)counts) & 15u) == 0u;
    return pick<Backward>(experts, vector, (float *)d_logits, (const float *)logits, (const uint32_t *)ids, (const uint32_t *)counts,
                          (const uint32_t *)offsets, (const float *)d_loss, (const float *)d_weights, a, coefficient, route_scale,
                          (cudaStream_t)stream);
}
