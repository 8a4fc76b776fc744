// RMS norm with the residual's addition in front, E4M3 codes behind, and its gradient (include/k3_moe_norm.h).
//
//   s = x + residual,  rstd = (mean s^2 + epsilon)^(-1/2),  y = s rstd w
//   dx = d_sum + rstd (w dy - s rstd^2 mean(w dy s)),  dw = sum over rows of dy s rstd
//
// Bound by memory: a row is read once, kept in registers over the row's sum, and written once.  A row belongs to a
// warp (up to 1024 columns) or to a block of 256 or 1024 threads; a thread holds vectors of 8 neighbouring columns,
// so the 16 lanes of half a warp hold a block of 128, whose largest magnitude is four shuffles away.  The gradient of
// many rows goes through a ring in shared memory (below).  8192 x 7168 bf16: forward with sum, bf16 rows and codes 84 us 20 times
// over the same arrays, 90 over others, 6.3 and 5.9 TB/s; backward with the weight's gradient 79 us, 5.9 TB/s.  The gradient of more than
// 8192 columns, 1024 threads to a row, spills 132 to 272 bytes of registers.
#include "k3_common.cuh"
#include "k3_fp8_ptx.cuh"
#include "k3_grouped.h"
#include "k3_moe_norm.h"

#include <algorithm>

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kMaxHidden = 16384;

// Eight elements of a row as they lie in memory.  kVector: neighbours, c .. c + 7, of rows that start on 16 bytes and are
// whole vectors.  Otherwise (matrices that start elsewhere) c, c + 16, .. c + 112: the half warp still holds a block of 128, and its 16 lanes read
// neighbours (rows of 3583 f32: the gradient of 1021 rows 20.7 us, 30.8 with eight neighbours per thread).
template <bool kVector>
K3_DEVINL constexpr uint32_t column_of(uint32_t c, uint32_t i) { return kVector ? c + i : c + 16u * i; }
// the first column of a thread's vector: thread `at` of those that lie along the row
template <bool kVector>
K3_DEVINL constexpr uint32_t first_column(uint32_t at) { return kVector ? at * 8u : at / 16u * kBlock + at % 16u; }

template <bool kF32>
struct Eight {
    static constexpr uint32_t kWords = kF32 ? 8u : 4u;
    uint32_t w[kWords];

    // zeros past the row's end
    template <bool kVector>
    K3_DEVINL void load(const void *row, uint32_t c, uint32_t columns) {
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) w[i] = 0u;
        if (kVector) {
            if (c >= columns) return;
#pragma unroll
            for (uint32_t h = 0; h < kWords / 4u; h++) {
                const uint4 q = *reinterpret_cast<const uint4 *>((const char *)row + (uint64_t)c * (kF32 ? 4u : 2u) + h * 16u);
                w[4u * h] = q.x; w[4u * h + 1u] = q.y; w[4u * h + 2u] = q.z; w[4u * h + 3u] = q.w;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                if (column_of<kVector>(c, i) >= columns) continue;
                if (kF32) w[i % kWords] = ((const uint32_t *)row)[column_of<kVector>(c, i)];
                else w[i / 2u] |= (uint32_t)((const uint16_t *)row)[column_of<kVector>(c, i)] << (16u * (i & 1u));
            }
        }
    }
    template <bool kVector>
    K3_DEVINL void store(void *row, uint32_t c, uint32_t columns) const {
        if (kVector) {
            if (c >= columns) return;
#pragma unroll
            for (uint32_t h = 0; h < kWords / 4u; h++) {
                *reinterpret_cast<uint4 *>((char *)row + (uint64_t)c * (kF32 ? 4u : 2u) + h * 16u) =
                    make_uint4(w[4u * h], w[4u * h + 1u], w[4u * h + 2u], w[4u * h + 3u]);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                if (column_of<kVector>(c, i) >= columns) continue;
                if (kF32) ((uint32_t *)row)[column_of<kVector>(c, i)] = w[i % kWords];
                else ((uint16_t *)row)[column_of<kVector>(c, i)] = (uint16_t)(w[i / 2u] >> (16u * (i & 1u)));
            }
        }
    }
    // Of a matrix of `total` elements on 16 bytes those from `at` on, a multiple of 8, of which the first is in column c of the row
    // (below 0: in the row in front).  In two steps, so that no branch stands between the loads of several: the matrix's last
    // elements and zeros for those of other rows come second.
    K3_DEVINL void fetch(const void *matrix, uint64_t at, uint64_t total, int32_t c, int32_t columns) {
        load<true>((const char *)matrix + at * (kF32 ? 4u : 2u), 0u, c > -8 && c < columns && at + 8u <= total ? 8u : 0u);
    }
    K3_DEVINL void finish(const void *matrix, uint64_t at, uint64_t total, int32_t c, int32_t columns) {
        if (c <= -8 || c >= columns || (c >= 0 && c + 8 <= columns)) return;
        if (at + 8u > total) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                if (at + i >= total) continue;
                if (kF32) w[i % kWords] = ((const uint32_t *)matrix)[at + i];
                else w[i / 2u] |= (uint32_t)((const uint16_t *)matrix)[at + i] << (16u * (i & 1u));
            }
        }
#pragma unroll
        for (int32_t i = 0; i < 8; i++) {
            if (c + i >= 0 && c + i < columns) continue;
            if (kF32) w[i % kWords] = 0u;
            else w[i / 2] &= i & 1 ? 0xffffu : 0xffff0000u;
        }
    }
    K3_DEVINL void store_flat(void *matrix, uint64_t at, int32_t c, int32_t columns) const {
        if (c >= 0 && c + 8 <= columns) {
            store<true>((char *)matrix + at * (kF32 ? 4u : 2u), 0u, 8u);
            return;
        }
#pragma unroll
        for (int32_t i = 0; i < 8; i++) {
            if (c + i < 0 || c + i >= columns) continue;
            if (kF32) ((uint32_t *)matrix)[at + i] = w[i % kWords];
            else ((uint16_t *)matrix)[at + i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
    // elements by .. by + 7 of two neighbours, by < 8
    K3_DEVINL void between(const Eight &first, const Eight &second, uint32_t by) {
        uint32_t v[2u * kWords];
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) {
            v[i] = first.w[i];
            v[kWords + i] = second.w[i];
        }
#pragma unroll
        for (uint32_t bit = 4u; bit > (kF32 ? 0u : 1u); bit /= 2u) {
            const uint32_t words = kF32 ? bit : bit / 2u;
#pragma unroll
            for (uint32_t i = 0; i + words < 2u * kWords; i++) v[i] = by & bit ? v[i + words] : v[i];
        }
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) w[i] = kF32 || (by & 1u) == 0u ? v[i] : __byte_perm(v[i], v[i + 1u], 0x5432);
    }
    K3_DEVINL float value(uint32_t i) const {
        if (kF32) return __uint_as_float(w[i % kWords]);
        return i & 1u ? bf16_hi(w[i / 2u]) : bf16_lo(w[i / 2u]);
    }
    K3_DEVINL void set(const float (&v)[8]) {
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) w[i] = kF32 ? __float_as_uint(v[i]) : bf16x2(v[(2u * i) % 8u], v[(2u * i + 1u) % 8u]);
    }
};

// Sum over the threads of a row, the same in all of them.  `scratch`: one float per warp of the block and a place
// for the next call; called by all threads of the block.
template <uint32_t kTeam>
K3_DEVINL float team_sum(float v, float *scratch) {
    v = warp_sum(v);
    if (kTeam == kWarp) return v;
    constexpr uint32_t kWarps = kTeam / kWarp;
    if (threadIdx.x % kWarp == 0u) scratch[threadIdx.x / kWarp] = v;
    __syncthreads();
    v = threadIdx.x % kWarp < kWarps ? scratch[threadIdx.x % kWarp] : 0.0f;
    return warp_sum(v);
}

constexpr uint32_t threads_of(uint32_t team) { return team == 1024u ? 1024u : 256u; }

struct NormArgs {
    void *sum;
    uint16_t *y;
    uint8_t *codes;
    float *scales, *rstd;
    const void *x, *residual;
    const uint16_t *weight;
    uint32_t rows, hidden;
    float epsilon;
};

// Two neighbouring elements as f32.
template <bool kF32>
K3_DEVINL uint64_t pair_of(const Eight<kF32> &e, uint32_t i) { return pack2(e.value(2u * i), e.value(2u * i + 1u)); }

constexpr uint32_t kSigns = 0x80008000u;                             // of two bf16
K3_DEVINL void negate(Eight<false> &w) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) w.w[i] ^= kSigns;
}
// the largest of a and the magnitudes of b and c; NaN if one of them is
K3_DEVINL float largest_of(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The normalised elements of a thread's vectors to y, and to codes with the largest magnitude of the half warp's block.
// All lanes of a warp call it; `live`: the row exists; kPartial: a vector may
// lie across the row's end, and y is not asked for.  minus_w: the weight's negatives, for the quotients want -y.  Two
// elements at a time and the vectors side by side through every step, 8192 x 7168 to codes alone takes 59 us; element by
// element, and one vector after the other with its shuffles and its reciprocal, it took 78.
//
// Codes of bf16 rows: with rstd = f m, f a power of two, and p = s f w, y is p m, the scale max |p| m / 448 and y / scale therefore
// 448 p / max |p|.  p and 448 p are exact and the quotient is rounded once, so that those in the middle between two codes, one in
// some thousands, go to the even one; by way of y the last bit of rstd decided (8192 x 7168 with both outputs 83 us, now 84).
// Of f32 rows p is y.
template <bool kF32, bool kVector, bool kPartial = false, uint32_t kVectors, typename First>
K3_DEVINL void put_normed(const NormArgs &a, const Eight<kF32> (&s)[kVectors], const Eight<false> (&minus_w)[kVectors], float rstd, uint64_t row,
                          First first, bool live) {
    const uint32_t hidden = a.hidden, pitch = pitch_of(hidden);
    uint64_t p[kVectors][4];                                         // negative
    auto scale_rows = [&](float by) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) p[v][i] = mul2(mul2(pair_of(s[v], i), both2(by)), pair_of(minus_w[v], i));
        }
    };
    if (kF32) scale_rows(rstd);
    if (!kPartial && a.y != nullptr) {
        const uint64_t rstd2 = both2(rstd);
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            Eight<false> out;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint64_t y = kF32 ? p[v][i] : mul2(mul2(pair_of(s[v], i), rstd2), pair_of(minus_w[v], i));
                out.w[i] = bf16x2(lo2(y), hi2(y)) ^ kSigns;
            }
            out.template store<kVector>(a.y + row * hidden, first(v), live ? hidden : 0u);
        }
    }
    if (a.codes == nullptr) return;
    const float m = kF32 ? 1.0f : __uint_as_float((__float_as_uint(rstd) & 0x7fffffu) | 0x3f800000u);
    if (!kF32) scale_rows(__uint_as_float(__float_as_uint(rstd) & 0x7f800000u));
    uint32_t most[kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        const uint32_t c = first(v);
        float largest = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            if (!kVector || kPartial) {                              // past the row's end: no part of the block, whatever rstd is
                p[v][i] = pack2(column_of<kVector>(c, 2u * i) < hidden ? lo2(p[v][i]) : 0.0f,
                                column_of<kVector>(c, 2u * i + 1u) < hidden ? hi2(p[v][i]) : 0.0f);
            }
            largest = largest_of(largest, lo2(p[v][i]), hi2(p[v][i]));
        }
        most[v] = kVector && c >= hidden ? 0u : __float_as_uint(largest);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) most[v] = max(most[v], __shfl_xor_sync(0xffffffffu, most[v], o));
    }
    uint2 codes[kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        const float largest = __uint_as_float(most[v]), scale = scale_of(__float_as_uint(largest * m));
        // (the smallest scale: as if `largest` were what it is for; the lift keeps remainders normal and 448 p finite)
        const float divisor = kF32 ? scale : scale == 0x1p-126f ? 448.0f * 0x1p-126f * reciprocal_fast(m) : largest;
        const float lift = !kF32 && divisor > 0x1p100f ? 0x1p-64f : lift_of(divisor);
        const uint64_t by = both2(divisor * lift), inverse = both2(-inverse_of(divisor * lift)), factor = both2(kF32 ? lift : 448.0f * lift);
        uint32_t h[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            const uint64_t q = divided2(mul2(p[v][i], factor), by, inverse);
            h[i] = codes2(lo2(q), hi2(q));
        }
        codes[v] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        if (kVector && first(v) >= hidden) codes[v] = make_uint2(0u, 0u);            // zeros in the padding: the quotient is one of 0, or NaN
        if (kPartial && first(v) < hidden && hidden - first(v) < 8u) {
            const uint64_t mask = (1ull << (8u * (hidden - first(v)))) - 1u;
            codes[v] = make_uint2(codes[v].x & (uint32_t)mask, codes[v].y & (uint32_t)(mask >> 32));
        }
        most[v] = __float_as_uint(scale);
    }
    if (!live) return;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        const uint32_t c = first(v);
        uint8_t *to = a.codes + row * pitch;
        if (kVector) {
            if (c < pitch) *reinterpret_cast<uint2 *>(to + c) = codes[v];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const uint32_t at = column_of<kVector>(c, i);
                if (at < pitch) to[at] = at < hidden ? (uint8_t)((i < 4u ? codes[v].x : codes[v].y) >> (8u * (i & 3u))) : 0u;
            }
        }
        if (c < hidden && (c & 127u) == 0u) a.scales[row * scale_pitch_of(hidden) + c / kBlock] = __uint_as_float(most[v]);
    }
}
// The scales' row behind its blocks.  t: a thread's place in the row's team.
K3_DEVINL void put_scale_padding(const NormArgs &a, uint64_t row, uint32_t t) {
    const uint32_t blocks = blocks_of(a.hidden), pitch = scale_pitch_of(a.hidden);
    if (a.codes != nullptr && t < pitch - blocks) a.scales[row * pitch + blocks + t] = 0.0f;
}

// kTeam threads per row, kVectors vectors of 8 columns each.
template <bool kF32, bool kVector, uint32_t kTeam, uint32_t kVectors>
__global__ void __launch_bounds__(threads_of(kTeam)) norm_kernel(NormArgs a) {
    pdl_wait();
    __shared__ float scratch[32];
    constexpr uint32_t kTeams = threads_of(kTeam) / kTeam, kSize = kF32 ? 4u : 2u;
    const uint32_t t = threadIdx.x % kTeam;
    const uint64_t task = (uint64_t)blockIdx.x * kTeams + threadIdx.x / kTeam;
    const bool live = task < a.rows;                                 // the shuffles want every lane
    const uint64_t row = live ? task : 0u;
    const uint32_t columns = live ? a.hidden : 0u;
    auto first = [&](uint32_t v) { return first_column<kVector>(v * kTeam + t); };
    const char *x = (const char *)a.x + row * a.hidden * kSize;
    const char *residual = (const char *)a.residual + row * a.hidden * kSize;
    Eight<kF32> s[kVectors], r[kVectors];
    Eight<false> w[kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) s[v].template load<kVector>(x, first(v), columns);
    if (a.residual != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) r[v].template load<kVector>(residual, first(v), columns);
    }
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) w[v].template load<kVector>(a.weight, first(v), columns);
    if (a.residual != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            float f[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) f[i] = s[v].value(i) + r[v].value(i);
            s[v].set(f);
        }
    }
    if (a.sum != nullptr) {
        char *sum = (char *)a.sum + row * a.hidden * kSize;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) s[v].template store<kVector>(sum, first(v), columns);
    }
    float squares = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) squares = fmaf(s[v].value(i), s[v].value(i), squares);
    }
    squares = team_sum<kTeam>(squares, scratch);
    const float rstd = 1.0f / sqrtf(squares / (float)a.hidden + a.epsilon);
    if (live && t == 0u && a.rstd != nullptr) a.rstd[row] = rstd;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) negate(w[v]);
    put_normed<kF32, kVector>(a, s, w, rstd, row, first, live);
    if (live) put_scale_padding(a, row, t);
    pdl_trigger();
}

// Rows whose length is no multiple of 8 start anywhere in a vector.  A thread's vectors are then those of the matrix as a whole, and
// hold the row from column -o on, o the row's place modulo 8: loads and stores are whole but at a row's ends.  The weight's
// vectors lie across these, as do codes and their blocks, for which the row goes through shared memory.  20 times over the same arrays:
// 4096 x 7001 bf16 forward with both outputs 76 us, element by element 108, of 7008 columns 44; backward 85, 209 and 43; f32 forward 107,
// 103 and 68, backward 102, 144 and 66; 2048 x 3583 f32 forward 26, 25 and 17, backward 25, 29 and 24.
K3_DEVINL Eight<false> weight_from(const uint16_t *weight, int32_t c, uint32_t o, uint32_t hidden) {
    const int32_t at = o != 0u ? c + (int32_t)o - 8 : c;
    Eight<false> first, second;
    first.fetch(weight, (uint64_t)(int64_t)at, hidden, at, (int32_t)hidden);
    second.fetch(weight, (uint64_t)(at + 8), hidden, at + 8, (int32_t)hidden);
    first.finish(weight, (uint64_t)(int64_t)at, hidden, at, (int32_t)hidden);
    second.finish(weight, (uint64_t)(at + 8), hidden, at + 8, (int32_t)hidden);
    first.between(first, second, (8u - o) & 7u);
    return first;
}
constexpr uint32_t flat_units(uint32_t hidden) { return (hidden + 7u) / 8u + 1u; }

template <bool kF32, uint32_t kTeam, uint32_t kVectors>
__global__ void __launch_bounds__(threads_of(kTeam), kTeam == 256u && kVectors == 4u && !kF32 ? 4 : 0) norm_flat_kernel(NormArgs a) {
    pdl_wait();
    __shared__ float scratch[32];
    extern __shared__ __align__(16) unsigned char row_smem[];             // codes only: [kTeams][flat_units] vectors
    constexpr uint32_t kTeams = threads_of(kTeam) / kTeam, kUnit = kF32 ? 32u : 16u;
    const uint32_t t = threadIdx.x % kTeam, units = flat_units(a.hidden);
    const uint64_t task = (uint64_t)blockIdx.x * kTeams + threadIdx.x / kTeam, total = (uint64_t)a.rows * a.hidden;
    const bool live = task < a.rows;
    const uint64_t row = live ? task : 0u, from = row * a.hidden / 8u * 8u;
    const uint32_t o = (uint32_t)(row * a.hidden - from);
    const int32_t columns = live ? (int32_t)a.hidden : -8;
    auto unit = [&](uint32_t v) { return v * kTeam + t; };
    auto column = [&](uint32_t v) { return (int32_t)(unit(v) * 8u) - (int32_t)o; };
    Eight<kF32> s[kVectors], r[kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) s[v].fetch(a.x, from + unit(v) * 8u, total, column(v), columns);
    if (a.residual != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) r[v].fetch(a.residual, from + unit(v) * 8u, total, column(v), columns);
    }
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) s[v].finish(a.x, from + unit(v) * 8u, total, column(v), columns);
    if (a.residual != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            r[v].finish(a.residual, from + unit(v) * 8u, total, column(v), columns);
            float f[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) f[i] = s[v].value(i) + r[v].value(i);
            s[v].set(f);
        }
    }
    if (a.sum != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) s[v].store_flat(a.sum, from + unit(v) * 8u, column(v), columns);
    }
    float squares = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) squares = fmaf(s[v].value(i), s[v].value(i), squares);
    }
    unsigned char *mine = row_smem + threadIdx.x / kTeam * units * kUnit;
    if (a.codes != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) s[v].template store<true>(mine, unit(v) * 8u, units * 8u);
    }
    squares = team_sum<kTeam>(squares, scratch);                     // the row is in shared memory behind it
    const float rstd = 1.0f / sqrtf(squares / (float)a.hidden + a.epsilon);
    if (live && t == 0u && a.rstd != nullptr) a.rstd[row] = rstd;
    if (a.y != nullptr) {
        const uint64_t rstd2 = both2(rstd);
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            const Eight<false> w = weight_from(a.weight, column(v), o, a.hidden);
            Eight<false> out;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint64_t y = mul2(mul2(pair_of(s[v], i), rstd2), pair_of(w, i));
                out.w[i] = bf16x2(lo2(y), hi2(y));
            }
            out.store_flat(a.y, from + unit(v) * 8u, column(v), columns);
        }
    }
    if (a.codes != nullptr) {
        if (kTeam == kWarp) __syncwarp();
        Eight<false> w[kVectors];
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            Eight<kF32> first, second;
            const uint32_t c = unit(v) * 8u;
            first.template load<true>(mine, c, units * 8u);
            second.template load<true>(mine, c + 8u, units * 8u);
            s[v].between(first, second, o);
            w[v].fetch(a.weight, c, a.hidden, (int32_t)c, (int32_t)a.hidden);
        }
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            w[v].finish(a.weight, unit(v) * 8u, a.hidden, (int32_t)(unit(v) * 8u), (int32_t)a.hidden);
            negate(w[v]);
        }
        put_normed<kF32, true, true>(a, s, w, rstd, row, [&](uint32_t v) { return unit(v) * 8u; }, live);
        if (live) put_scale_padding(a, row, t);
    }
    pdl_trigger();
}

// -------------------------------------------------------------------------------------------- gradient
struct NormGradArgs {
    void *dx;
    float *partial;                  // [blocks, hidden], or null
    const uint16_t *dy, *weight;
    const void *sum, *d_sum;
    const float *rstd;
    uint32_t rows, hidden;
};

// A vector's part of the row's sum of w dy s rstd, and of the weight's gradient, two elements at a time.
template <bool kF32>
K3_DEVINL uint64_t add_products(const Eight<false> &dy, const Eight<kF32> &s, const Eight<false> &w, uint64_t rstd, uint64_t dot, uint64_t (&dw)[4]) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
        const uint64_t g = pair_of(dy, i), h = mul2(pair_of(s, i), rstd);
        dot = fma2(mul2(g, pair_of(w, i)), h, dot);
        dw[i] = fma2(g, h, dw[i]);
    }
    return dot;
}
// A vector of dx; minus_mean: the negative of the mean of w dy s rstd over the row.
template <bool kF32>
K3_DEVINL Eight<kF32> input_gradient(const Eight<false> &dy, const Eight<kF32> &s, const Eight<false> &w, const Eight<kF32> &d, bool with_d,
                                     uint64_t rstd, uint64_t minus_mean) {
    float f[8];
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) {
        const uint64_t x = fma2(mul2(pair_of(s, i), rstd), minus_mean, mul2(pair_of(dy, i), pair_of(w, i)));
        const uint64_t r = with_d ? fma2(x, rstd, pair_of(d, i)) : mul2(x, rstd);
        f[2u * i] = lo2(r);
        f[2u * i + 1u] = hi2(r);
    }
    Eight<kF32> out;
    out.set(f);
    return out;
}

// Rows team, team + teams, ..; the weight's gradient stays in registers over all of them.
template <bool kF32, bool kVector, uint32_t kTeam, uint32_t kVectors>
__global__ void __launch_bounds__(threads_of(kTeam)) norm_backward_kernel(NormGradArgs a) {
    pdl_wait();
    constexpr uint32_t kThreads = threads_of(kTeam), kTeams = kThreads / kTeam, kSize = kF32 ? 4u : 2u;
    __shared__ float scratch[2][32];
    extern __shared__ float shared_dw[];                             // [kTeams][hidden], several teams only
    const uint32_t t = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
    auto first = [&](uint32_t v) { return first_column<kVector>(v * kTeam + t); };
    Eight<false> w[kVectors];
    uint64_t dw[kVectors][4];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        w[v].template load<kVector>(a.weight, first(v), a.hidden);
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) dw[v][i] = 0ull;
    }
    uint32_t turn = 0u;
    for (uint64_t at = (uint64_t)blockIdx.x * kTeams; at < a.rows; at += (uint64_t)gridDim.x * kTeams, turn ^= 1u) {
        const bool live = at + team < a.rows;
        const uint64_t row = live ? at + team : 0u;
        const uint32_t columns = live ? a.hidden : 0u;
        Eight<false> dy[kVectors];
        Eight<kF32> s[kVectors], d[kVectors];
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            dy[v].template load<kVector>(a.dy + row * a.hidden, first(v), columns);
            s[v].template load<kVector>((const char *)a.sum + row * a.hidden * kSize, first(v), columns);
            if (a.d_sum != nullptr) d[v].template load<kVector>((const char *)a.d_sum + row * a.hidden * kSize, first(v), columns);
        }
        const float rstd = live ? a.rstd[row] : 0.0f;                // with it zeros in the rows that do not exist
        uint64_t dots = 0ull;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) dots = add_products<kF32>(dy[v], s[v], w[v], both2(rstd), dots, dw[v]);
        const float mean = team_sum<kTeam>(lo2(dots) + hi2(dots), scratch[turn]) / (float)a.hidden;
        char *dx = (char *)a.dx + row * a.hidden * kSize;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            input_gradient<kF32>(dy[v], s[v], w[v], d[v], a.d_sum != nullptr, both2(rstd), both2(-mean)).template store<kVector>(dx, first(v), columns);
        }
    }
    if (a.partial == nullptr) return;
    float *to = a.partial + (uint64_t)blockIdx.x * a.hidden;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
            const uint32_t c = column_of<kVector>(first(v), i);
            if (c < a.hidden) (kTeams == 1u ? to : shared_dw + team * a.hidden)[c] = i & 1u ? hi2(dw[v][i / 2u]) : lo2(dw[v][i / 2u]);
        }
    }
    if (kTeams > 1u) {
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < a.hidden; c += kThreads) {
            float sum = shared_dw[c];
            for (uint32_t i = 1; i < kTeams; i++) sum += shared_dw[i * a.hidden + c];
            to[c] = sum;
        }
    }
}

// norm_backward_kernel by the matrix's vectors.  Rows that a team takes are a multiple of 8 apart, so their places modulo 8 are
// the same, and the columns of its weight gradient too.
template <bool kF32, uint32_t kTeam, uint32_t kVectors>
__global__ void __launch_bounds__(threads_of(kTeam)) norm_backward_flat_kernel(NormGradArgs a) {
    pdl_wait();
    constexpr uint32_t kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
    __shared__ float scratch[2][32];
    extern __shared__ float shared_dw[];                             // [kTeams][hidden]
    const uint32_t t = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
    const uint64_t total = (uint64_t)a.rows * a.hidden;
    const uint32_t o = (uint32_t)(((uint64_t)blockIdx.x * kTeams + team) * a.hidden % 8u);
    auto column = [&](uint32_t v) { return (int32_t)((v * kTeam + t) * 8u) - (int32_t)o; };
    Eight<false> w[kVectors];
    uint64_t dw[kVectors][4];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        w[v] = weight_from(a.weight, column(v), o, a.hidden);
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) dw[v][i] = 0ull;
    }
    uint32_t turn = 0u;
    for (uint64_t at = (uint64_t)blockIdx.x * kTeams; at < a.rows; at += (uint64_t)gridDim.x * kTeams, turn ^= 1u) {
        const bool live = at + team < a.rows;
        const uint64_t from = live ? (at + team) * a.hidden - o : 0u;
        const int32_t columns = live ? (int32_t)a.hidden : -8;
        Eight<false> dy[kVectors];
        Eight<kF32> s[kVectors], d[kVectors];
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            const uint64_t f = from + (v * kTeam + t) * 8u;
            dy[v].fetch(a.dy, f, total, column(v), columns);
            s[v].fetch(a.sum, f, total, column(v), columns);
            if (a.d_sum != nullptr) d[v].fetch(a.d_sum, f, total, column(v), columns);
        }
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            const uint64_t f = from + (v * kTeam + t) * 8u;
            dy[v].finish(a.dy, f, total, column(v), columns);
            s[v].finish(a.sum, f, total, column(v), columns);
            if (a.d_sum != nullptr) d[v].finish(a.d_sum, f, total, column(v), columns);
        }
        const float rstd = live ? a.rstd[at + team] : 0.0f;
        uint64_t dots = 0ull;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) dots = add_products<kF32>(dy[v], s[v], w[v], both2(rstd), dots, dw[v]);
        const float mean = team_sum<kTeam>(lo2(dots) + hi2(dots), scratch[turn]) / (float)a.hidden;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            input_gradient<kF32>(dy[v], s[v], w[v], d[v], a.d_sum != nullptr, both2(rstd), both2(-mean))
                .store_flat(a.dx, from + (v * kTeam + t) * 8u, column(v), columns);
        }
    }
    if (a.partial == nullptr) return;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
        for (int32_t i = 0; i < 8; i++) {
            const int32_t c = column(v) + i;
            if (c >= 0 && c < (int32_t)a.hidden) shared_dw[team * a.hidden + c] = i & 1 ? hi2(dw[v][i / 2]) : lo2(dw[v][i / 2]);
        }
    }
    __syncthreads();
    float *to = a.partial + (uint64_t)blockIdx.x * a.hidden;
    for (uint32_t c = threadIdx.x; c < a.hidden; c += kThreads) {
        float sum = shared_dw[c];
        for (uint32_t i = 1; i < kTeams; i++) sum += shared_dw[i * a.hidden + c];
        to[c] = sum;
    }
}

// d_weight from the blocks' partial rows: 32 columns per block, eight parts of the rows, added in ascending order.
__global__ void __launch_bounds__(256) norm_weight_kernel(float *d_weight, const float *partial, uint32_t parts, uint32_t hidden,
                                                          int accumulate) {
    pdl_wait();
    __shared__ float sums[8][33];
    const uint32_t lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp, c = blockIdx.x * kWarp + lane;
    const uint32_t each = (parts + 7u) / 8u, end = min(parts, (warp + 1u) * each);
    float sum = 0.0f;
    if (c < hidden) {
#pragma unroll 8
        for (uint32_t p = warp * each; p < end; p++) sum += partial[(uint64_t)p * hidden + c];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0u && c < hidden) {
        sum = accumulate ? d_weight[c] : 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) sum += sums[i][lane];
        d_weight[c] = sum;
    }
}

// ------------------------------------------------------------------------------------- rows through a ring
// The gradient of many rows of more than 1024 columns: one block per SM, in one or two teams that take a row each in turn, so
// that the weight's gradient stays in registers, from a ring of stages in shared memory with whole rows, up to 192 KB per
// block, so that memory is never waited for while a row's sum goes around the team.  A thread of the team fills the ring: a
// stage is free once its row's sum is there.  (A seventeenth warp for that would leave 96 registers per thread instead of 128:
// 8192 x 7168 96 us; without a ring 136.)  Forward nothing stays from row to row, and a block per row needs no ring.
constexpr uint32_t kRingThreads = 512, kRingBytes = 196608, kRingHidden = 8192, kMaxStages = 8;

__device__ uint32_t g_norm_status = 0;

K3_DEVINL void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// Up to three arrays' rows, side by side in a stage.
struct RowSources {
    const char *at[3];
    uint32_t bytes[3];
};

// A ring of stages; its k-th row is first + k step.
struct Ring {
    // a stage and the parity of its use
    struct Turn {
        uint32_t s, ph;
        K3_DEVINL void advance(uint32_t by, uint32_t stages) {
            s += by;
            if (s >= stages) { s -= stages; ph ^= 1u; }
        }
    };
    unsigned char *base;
    uint64_t *full;
    volatile uint32_t *abort_flag;
    uint32_t stages, stage_bytes;
    Turn next;                               // of the thread that loads
    uint64_t first, step, next_row, rows;

    // ring `at` of `rings` in the block; all threads of the block
    K3_DEVINL void init(unsigned char *smem, uint32_t stages_, uint32_t stage_bytes_, uint32_t at, uint32_t rings, uint64_t rows_) {
        stages = stages_;
        stage_bytes = stage_bytes_;
        full = reinterpret_cast<uint64_t *>(smem) + at * stages;
        abort_flag = reinterpret_cast<uint32_t *>(smem + 8u * kMaxStages);
        base = smem + 256u + at * stages * stage_bytes;
        next = {0u, 0u};
        first = next_row = blockIdx.x + (uint64_t)at * gridDim.x;
        step = (uint64_t)rings * gridDim.x;
        rows = rows_;
        if (threadIdx.x == 0u) {
            *abort_flag = 0u;
            for (uint32_t s = 0; s < stages * rings; s++) mbar_init(&full[s], 1);
            fence_barrier_init();
        }
        __syncthreads();
    }
    // one thread: the next row, if there is one, into its stage, which is free
    K3_DEVINL void load_next(const RowSources &from) {
        if (next_row >= rows || *abort_flag != 0u) return;
        unsigned char *to = base + next.s * stage_bytes;
        mbar_arrive_expect_tx(&full[next.s], stage_bytes);
#pragma unroll
        for (uint32_t i = 0; i < 3u; i++) {
            if (from.bytes[i] == 0u) continue;
            bulk_load(to, from.at[i] + next_row * from.bytes[i], from.bytes[i], &full[next.s]);
            to += from.bytes[i];
        }
        next.advance(1u, stages);
        next_row += step;
    }
    // a row is in its stage; false: given up
    K3_DEVINL bool wait(const Turn &t) { return mbar_wait(&full[t.s], t.ph, abort_flag); }
    K3_DEVINL const unsigned char *place(const Turn &t) const { return base + t.s * stage_bytes; }
    // the thread that loads, at its end: nothing may land in a block that has left.  The last use of each stage.
    K3_DEVINL void drain() {
        if (*abort_flag == 0u) return;
        for (uint32_t s = 0; s < stages; s++) {
            const uint32_t last = s < next.s ? next.ph : next.ph ^ 1u;
            if (s < next.s || next_row >= first + stages * step) mbar_drain(&full[s], last);
        }
    }
};

// Sum over the kTeam threads of a row; `scratch`, a float per warp of the team, alternates between two rows.
template <uint32_t kTeam>
K3_DEVINL float ring_sum(float v, float *scratch) {
    constexpr uint32_t kWarps = kTeam / kWarp;
    v = warp_sum(v);
    if (threadIdx.x % kWarp == 0u) scratch[threadIdx.x % kTeam / kWarp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1u + threadIdx.x / kTeam), "n"(kTeam) : "memory");
    v = scratch[threadIdx.x % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A ring for each team: a stage's rows are all of one team, which has taken out a stage's row before it waits for the next
// one there, so that a wait by parity never meets a phase that another team's row has yet to end.
template <bool kF32, uint32_t kVectors, uint32_t kTeam>
__global__ void __launch_bounds__(kRingThreads, 1) norm_backward_ring_kernel(NormGradArgs a, uint32_t stages) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr uint32_t kTeams = kRingThreads / kTeam;
    __shared__ float scratch[kTeams][2][kTeam / kWarp];
    const uint32_t t = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
    const uint32_t bytes = a.hidden * (kF32 ? 4u : 2u), more = a.d_sum != nullptr ? bytes : 0u;
    const RowSources from = {{(const char *)a.dy, (const char *)a.sum, (const char *)a.d_sum}, {a.hidden * 2u, bytes, more}};
    Ring ring;
    ring.init(smem, stages, a.hidden * 2u + bytes + more, team, kTeams, a.rows);
    pdl_wait();
    if (t == 0u) {
        for (uint32_t i = 0; i < stages; i++) ring.load_next(from);
    }
    auto first = [&](uint32_t v) { return (v * kTeam + t) * 8u; };
    Eight<false> w[kVectors];
    uint64_t dw[kVectors][4];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        w[v].template load<true>(a.weight, first(v), a.hidden);
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) dw[v][i] = 0ull;
    }
    bool ok = true;
    uint32_t turn = 0u;
    Ring::Turn at{0u, 0u};
    float next_rstd = ring.first < a.rows ? a.rstd[ring.first] : 0.0f;               // on its way while the row before is worked on
    for (uint64_t row = ring.first; row < a.rows; row += ring.step, turn ^= 1u) {
        const float rstd = next_rstd;
        if (row + ring.step < a.rows) next_rstd = a.rstd[row + ring.step];
        ok = ok && ring.wait(at);
        const unsigned char *in = ring.place(at);
        at.advance(1u, stages);
        Eight<false> dy[kVectors];
        Eight<kF32> s[kVectors], d[kVectors];
        uint64_t dots = 0ull;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            dy[v].template load<true>(in, first(v), a.hidden);
            s[v].template load<true>(in + a.hidden * 2u, first(v), a.hidden);
            if (more != 0u) d[v].template load<true>(in + a.hidden * 2u + bytes, first(v), a.hidden);
        }
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) dots = add_products<kF32>(dy[v], s[v], w[v], both2(rstd), dots, dw[v]);
        const float mean = ring_sum<kTeam>(lo2(dots) + hi2(dots), scratch[team][turn]) / (float)a.hidden;
        if (t == 0u) ring.load_next(from);
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            input_gradient<kF32>(dy[v], s[v], w[v], d[v], more != 0u, both2(rstd), both2(-mean))
                .template store<true>((char *)a.dx + row * bytes, first(v), a.hidden);
        }
    }
    if (a.partial != nullptr) {
        float *to = a.partial + ((uint64_t)blockIdx.x * kTeams + team) * a.hidden;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            if (first(v) >= a.hidden) continue;
            *reinterpret_cast<ulonglong2 *>(to + first(v)) = make_ulonglong2(dw[v][0], dw[v][1]);
            *reinterpret_cast<ulonglong2 *>(to + first(v) + 4u) = make_ulonglong2(dw[v][2], dw[v][3]);
        }
    }
    if (t == 0u) ring.drain();
    pdl_trigger();
    __syncthreads();
    if (threadIdx.x == 0u && *ring.abort_flag != 0u) atomicExch(&g_norm_status, 1u);
}

// ------------------------------------------------------------------------------------------------ host
bool aligned(const void *p, uint32_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }

// Threads of a row and vectors of 8 columns per thread: a warp up to 1024 columns, then a block.
template <typename F>
bool by_size(uint32_t hidden, F &&launch) {
    using std::integral_constant;
#define K3_SIZE(team, vectors) launch(integral_constant<uint32_t, team>{}, integral_constant<uint32_t, vectors>{})
    if (hidden <= 256u) return K3_SIZE(32u, 1u);
    if (hidden <= 512u) return K3_SIZE(32u, 2u);
    if (hidden <= 1024u) return K3_SIZE(32u, 4u);
    if (hidden <= 2048u) return K3_SIZE(256u, 1u);
    if (hidden <= 4096u) return K3_SIZE(256u, 2u);
    if (hidden <= 8192u) return K3_SIZE(256u, 4u);
    return K3_SIZE(1024u, 2u);
#undef K3_SIZE
}
// Vectors of 8 columns per thread where 512 threads share a row.
template <typename F>
bool by_ring_size(uint32_t hidden, F &&launch) {
    using std::integral_constant;
    return hidden <= 4096u ? launch(integral_constant<uint32_t, 1u>{}) : launch(integral_constant<uint32_t, 2u>{});
}
// Stages for each of `teams`.
uint32_t team_stages(uint32_t stage_bytes, uint32_t teams) { return std::min(kRingBytes / stage_bytes, kMaxStages) / teams; }

template <typename K, typename A>
bool launch_ring(K kernel, const A &a, uint32_t stage_bytes, uint32_t rings, uint32_t stages, cudaStream_t stream) {
    const uint32_t bytes = 256u + rings * stages * stage_bytes;
    return set_max_dynamic_smem((const void *)kernel, 256u + kRingBytes) &&
           launch_chained(kernel, (uint32_t)sm_count(), kRingThreads, bytes, stream, a, stages);
}

// The ring pays once every SM has a row (us, with / without: 148 x 7168 14 / 16, 250 x 7168 16 / 20, 290 x 7168 16 / 22, 250 x 4104
// 14 / 16, f32 250 x 2048 14 / 14).
bool ring_suits(uint32_t rows, uint32_t hidden, bool vector) {
    return vector && hidden > 1024u && hidden <= kRingHidden && rows >= (uint32_t)sm_count();
}

// Rows by the matrix's vectors: no whole vectors, and places for one more.
bool flat_suits(uint32_t hidden) { return hidden % 8u != 0u && hidden + 7u <= kMaxHidden; }

template <bool kF32>
bool launch_norm(const NormArgs &a, bool on_16, cudaStream_t stream) {
    const bool vector = on_16 && a.hidden % 8u == 0u;
    if (on_16 && flat_suits(a.hidden)) {
        return by_size(a.hidden + 7u, [&](auto team, auto vectors) {
            constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
            auto kernel = norm_flat_kernel<kF32, kTeam, decltype(vectors)::value>;
            const uint32_t bytes = a.codes != nullptr ? kTeams * flat_units(a.hidden) * (kF32 ? 32u : 16u) : 0u;
            return set_max_dynamic_smem((const void *)kernel, kTeams * flat_units(kTeams > 1u ? 1024u : kMaxHidden) * 32u) &&
                   launch_chained(kernel, (a.rows + kTeams - 1u) / kTeams, kThreads, bytes, stream, a);
        });
    }
    return by_size(a.hidden, [&](auto team, auto vectors) {
        constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
        auto kernel = vector ? norm_kernel<kF32, true, kTeam, decltype(vectors)::value> : norm_kernel<kF32, false, kTeam, decltype(vectors)::value>;
        return launch_chained(kernel, (a.rows + kTeams - 1u) / kTeams, kThreads, 0, stream, a);
    });
}

// Blocks of the gradient, each with a partial row of the weight's: up to two per SM.
uint32_t most_grad_blocks(uint32_t rows, uint32_t hidden) {
    const uint32_t teams = (hidden % 8u != 0u ? hidden + 7u : hidden) <= 1024u ? 8u : 1u;
    return std::min((rows + teams - 1u) / teams, 2u * (uint32_t)sm_count());
}
// A multiple of 8 where a block takes several rows.
uint32_t grad_blocks(uint32_t rows, uint32_t hidden) {
    const uint32_t most = most_grad_blocks(rows, hidden);
    return most == 2u * (uint32_t)sm_count() ? most / 8u * 8u : most;
}

template <bool kF32>
bool launch_backward(const NormGradArgs &a, bool on_16, uint32_t &blocks, cudaStream_t stream) {
    const bool vector = on_16 && a.hidden % 8u == 0u;
    const uint32_t stage = a.hidden * (2u + (kF32 ? 4u : 2u) * (a.d_sum ? 2u : 1u));
    blocks = grad_blocks(a.rows, a.hidden);
    // two rows at a time up to 4096 columns of bf16 where there are as many; more, and f32, have no registers for it (8192 x 7168 133 us, one 91)
    const uint32_t teams = !kF32 && a.hidden <= 4096u && a.rows >= 2u * (uint32_t)sm_count() ? 2u : 1u, stages = team_stages(stage, teams);
    if (ring_suits(a.rows, a.hidden, vector) && stages >= 2u) {
        blocks = teams * (uint32_t)sm_count();
        if constexpr (!kF32) {
            if (teams == 2u) {
                return launch_ring(norm_backward_ring_kernel<kF32, 2u, kRingThreads / 2u>, a, stage, 2u, stages, stream);
            }
        }
        return by_ring_size(a.hidden, [&](auto vectors) {
            return launch_ring(norm_backward_ring_kernel<kF32, decltype(vectors)::value, kRingThreads>, a, stage, 1u, stages, stream);
        });
    }
    if (on_16 && flat_suits(a.hidden)) {
        return by_size(a.hidden + 7u, [&](auto team, auto vectors) {
            constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
            auto kernel = norm_backward_flat_kernel<kF32, kTeam, decltype(vectors)::value>;
            return set_max_dynamic_smem((const void *)kernel, kTeams * (kTeams > 1u ? 1024u : kMaxHidden) * 4u) &&
                   launch_chained(kernel, blocks, kThreads, kTeams * a.hidden * 4u, stream, a);
        });
    }
    return by_size(a.hidden, [&](auto team, auto vectors) {
        constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
        auto kernel = vector ? norm_backward_kernel<kF32, true, kTeam, decltype(vectors)::value>
                             : norm_backward_kernel<kF32, false, kTeam, decltype(vectors)::value>;
        return launch_chained(kernel, blocks, kThreads, kTeams > 1u ? kTeams * a.hidden * 4u : 0u, stream, a);
    });
}

bool sizes_ok(uint32_t rows, uint32_t hidden, int type) {
    return rows <= (1u << 30) && hidden != 0u && hidden <= kMaxHidden && (type == K3_MOE_NORM_BF16 || type == K3_MOE_NORM_F32);
}

}  // namespace

extern "C" bool k3_moe_norm(void *sum, void *y, void *codes, void *scales, void *rstd, const void *x, const void *residual,
                            const void *weight, uint32_t rows, uint32_t hidden, int type, float epsilon, void *stream) {
    if (!x || !weight || (!y && !codes) || (!codes) != (!scales) || rows == 0u || !sizes_ok(rows, hidden, type)) return false;
    if (!(epsilon > 0.0f)) return false;
    const bool f32 = type == K3_MOE_NORM_F32;
    const uint32_t size = f32 ? 4u : 2u;
    if (!aligned(sum, size) || !aligned(x, size) || !aligned(residual, size) || !aligned(weight, 2u) || !aligned(y, 2u) ||
        !aligned(rstd, 4u) || !aligned(codes, 16u) || !aligned(scales, 16u)) {
        return false;
    }
    const NormArgs a{sum, (uint16_t *)y, (uint8_t *)codes, (float *)scales, (float *)rstd, x, residual, (const uint16_t *)weight, rows,
                     hidden, epsilon};
    const bool on_16 = aligned(sum, 16u) && aligned(x, 16u) && aligned(residual, 16u) && aligned(weight, 16u) && aligned(y, 16u);
    return f32 ? launch_norm<true>(a, on_16, (cudaStream_t)stream) : launch_norm<false>(a, on_16, (cudaStream_t)stream);
}

extern "C" size_t k3_moe_norm_workspace_bytes(uint32_t rows, uint32_t hidden) {
    if (rows == 0u || !sizes_ok(rows, hidden, K3_MOE_NORM_F32)) return 0;
    return ((size_t)most_grad_blocks(rows, hidden) * hidden * 4u + 15u) / 16u * 16u;
}

extern "C" bool k3_moe_norm_backward(void *dx, void *d_weight, const void *dy, const void *sum, const void *rstd, const void *d_sum,
                                     const void *weight, uint32_t rows, uint32_t hidden, int type, int accumulate, void *workspace,
                                     size_t workspace_bytes, void *stream) {
    if (!sizes_ok(rows, hidden, type) || !aligned(d_weight, 4u)) return false;
    if (rows == 0u) {
        if (!d_weight || accumulate) return true;
        if (cudaMemsetAsync(d_weight, 0, (size_t)hidden * 4u, (cudaStream_t)stream) == cudaSuccess) return true;
        (void)cudaGetLastError();
        return false;
    }
    if (!dx || !dy || !sum || !rstd || !weight) return false;
    const bool f32 = type == K3_MOE_NORM_F32;
    const uint32_t size = f32 ? 4u : 2u;
    if (!aligned(dx, size) || !aligned(dy, 2u) || !aligned(sum, size) || !aligned(rstd, 4u) || !aligned(d_sum, size) ||
        !aligned(weight, 2u)) {
        return false;
    }
    if (d_weight && (!workspace || !aligned(workspace, 16u) || workspace_bytes < k3_moe_norm_workspace_bytes(rows, hidden))) return false;
    const NormGradArgs a{dx, d_weight ? (float *)workspace : nullptr, (const uint16_t *)dy, (const uint16_t *)weight, sum, d_sum,
                         (const float *)rstd, rows, hidden};
    const bool on_16 = aligned(dx, 16u) && aligned(dy, 16u) && aligned(sum, 16u) && aligned(d_sum, 16u) && aligned(weight, 16u);
    uint32_t blocks = 0u;
    const bool ok = f32 ? launch_backward<true>(a, on_16, blocks, (cudaStream_t)stream) : launch_backward<false>(a, on_16, blocks, (cudaStream_t)stream);
    if (!ok || !d_weight) return ok;
    return launch_chained(norm_weight_kernel, (hidden + 31u) / 32u, 256, 0, (cudaStream_t)stream, (float *)d_weight,
                          (const float *)workspace, blocks, hidden, accumulate);
}

uint32_t k3_norm_status() {
    uint32_t v = 0xffffffffu;
    if (cudaMemcpyFromSymbol(&v, g_norm_status, sizeof(v)) != cudaSuccess) (void)cudaGetLastError();
    return v;
}

bool k3_norm_status_clear() {
    const uint32_t zero = 0u;
    const bool ok = cudaMemcpyToSymbol(g_norm_status, &zero, sizeof(zero)) == cudaSuccess;
    if (!ok) (void)cudaGetLastError();
    return ok;
}
