// RMS norm with the residual's addition in front, E4M3 codes behind, and its gradient (include/k3_moe_norm.h).
//
//   s = x + residual,  rstd = (mean s^2 + epsilon)^(-1/2),  y = s rstd w
//   dx = d_sum + rstd (w dy - s rstd^2 mean(w dy s)),  dw = sum over rows of dy s rstd
//
// Bound by memory: a row is read once, kept in registers over the row's sum, and written once.  A row belongs to a
// warp (up to 1024 columns) or to a block of 256 or 1024 threads; a thread holds vectors of 8 neighbouring columns,
// so the 16 lanes of half a warp hold a block of 128, whose largest magnitude is four shuffles away.
#include "k3_common.cuh"
#include "k3_fp8_ptx.cuh"
#include "k3_moe_norm.h"

#include <algorithm>

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kMaxHidden = 65536;

// Eight neighbouring elements as they lie in memory.
template <bool kF32>
struct Eight {
    static constexpr uint32_t kWords = kF32 ? 8u : 4u;
    uint32_t w[kWords];

    // elements c .. c + 7 of a row, zeros past its end.  kVector: rows start on 16 bytes and are whole vectors.
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
                if (c + i >= columns) continue;
                if (kF32) w[i % kWords] = ((const uint32_t *)row)[c + i];
                else w[i / 2u] |= (uint32_t)((const uint16_t *)row)[c + i] << (16u * (i & 1u));
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
                if (c + i >= columns) continue;
                if (kF32) ((uint32_t *)row)[c + i] = w[i % kWords];
                else ((uint16_t *)row)[c + i] = (uint16_t)(w[i / 2u] >> (16u * (i & 1u)));
            }
        }
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
    const char *x = (const char *)a.x + row * a.hidden * kSize;
    const char *residual = (const char *)a.residual + row * a.hidden * kSize;
    Eight<kF32> s[kVectors], r[kVectors];
    Eight<false> w[kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) s[v].template load<kVector>(x, (v * kTeam + t) * 8u, columns);
    if (a.residual != nullptr) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) r[v].template load<kVector>(residual, (v * kTeam + t) * 8u, columns);
    }
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) w[v].template load<kVector>(a.weight, (v * kTeam + t) * 8u, columns);
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
        for (uint32_t v = 0; v < kVectors; v++) s[v].template store<kVector>(sum, (v * kTeam + t) * 8u, columns);
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
    const uint32_t pitch = pitch_of(a.hidden), blocks = blocks_of(a.hidden), scale_pitch = scale_pitch_of(a.hidden);
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        const uint32_t c = (v * kTeam + t) * 8u;
        float y[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) y[i] = __fmul_rn(__fmul_rn(s[v].value(i), rstd), w[v].value(i));
        if (a.y != nullptr) {
            Eight<false> out;
            out.set(y);
            out.template store<kVector>(a.y + row * a.hidden, c, columns);
        }
        if (a.codes != nullptr) {
            uint32_t most = 0u;
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                // zeros past the row's end times an infinite rstd are NaN: they are no part of the block
                if (c + i < a.hidden) most = max(most, __float_as_uint(y[i]) & 0x7fffffffu);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float scale = scale_of(most), inverse = inverse_of(scale), lift = lift_of(scale), by = scale * lift;
            uint32_t h[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                h[i] = codes2(divided(y[2u * i] * lift, by, inverse), divided(y[2u * i + 1u] * lift, by, inverse));
                if (c + 2u * i + 1u >= a.hidden) h[i] = c + 2u * i < a.hidden ? h[i] & 0xffu : 0u;
            }
            if (live && c < pitch) {
                *reinterpret_cast<uint2 *>(a.codes + row * pitch + c) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
            }
            if (live && c < a.hidden && (c & 127u) == 0u) a.scales[row * scale_pitch + c / kBlock] = scale;
        }
    }
    if (live && a.codes != nullptr && t < scale_pitch - blocks) a.scales[row * scale_pitch + blocks + t] = 0.0f;
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

// Rows team, team + teams, ..; the weight's gradient stays in registers over all of them.
template <bool kF32, bool kVector, uint32_t kTeam, uint32_t kVectors>
__global__ void __launch_bounds__(threads_of(kTeam)) norm_backward_kernel(NormGradArgs a) {
    pdl_wait();
    constexpr uint32_t kThreads = threads_of(kTeam), kTeams = kThreads / kTeam, kSize = kF32 ? 4u : 2u;
    __shared__ float scratch[2][32];
    extern __shared__ float shared_dw[];                             // [kTeams][hidden], several teams only
    const uint32_t t = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
    Eight<false> w[kVectors];
    float dw[kVectors][8];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; v++) {
        w[v].template load<kVector>(a.weight, (v * kTeam + t) * 8u, a.hidden);
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) dw[v][i] = 0.0f;
    }
    uint32_t turn = 0u;
    for (uint64_t first = (uint64_t)blockIdx.x * kTeams; first < a.rows; first += (uint64_t)gridDim.x * kTeams, turn ^= 1u) {
        const bool live = first + team < a.rows;
        const uint64_t row = live ? first + team : 0u;
        const uint32_t columns = live ? a.hidden : 0u;
        Eight<false> dy[kVectors];
        Eight<kF32> s[kVectors], d[kVectors];
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            dy[v].template load<kVector>(a.dy + row * a.hidden, (v * kTeam + t) * 8u, columns);
            s[v].template load<kVector>((const char *)a.sum + row * a.hidden * kSize, (v * kTeam + t) * 8u, columns);
        }
        if (a.d_sum != nullptr) {
#pragma unroll
            for (uint32_t v = 0; v < kVectors; v++) {
                d[v].template load<kVector>((const char *)a.d_sum + row * a.hidden * kSize, (v * kTeam + t) * 8u, columns);
            }
        }
        const float rstd = live ? a.rstd[row] : 0.0f;
        float dot = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const float g = dy[v].value(i), h = s[v].value(i) * rstd;
                dot = fmaf(g * w[v].value(i), h, dot);
                if (live) dw[v][i] = fmaf(g, h, dw[v][i]);
            }
        }
        dot = team_sum<kTeam>(dot, scratch[turn]) / (float)a.hidden;
        char *dx = (char *)a.dx + row * a.hidden * kSize;
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
            float f[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const float h = s[v].value(i) * rstd;
                f[i] = rstd * fmaf(-h, dot, dy[v].value(i) * w[v].value(i));
                if (a.d_sum != nullptr) f[i] += d[v].value(i);
            }
            Eight<kF32> out;
            out.set(f);
            out.template store<kVector>(dx, (v * kTeam + t) * 8u, columns);
        }
    }
    if (a.partial == nullptr) return;
    float *to = a.partial + (uint64_t)blockIdx.x * a.hidden;
    if (kTeams == 1u) {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const uint32_t c = (v * kTeam + t) * 8u + i;
                if (c < a.hidden) to[c] = dw[v][i];
            }
        }
    } else {
#pragma unroll
        for (uint32_t v = 0; v < kVectors; v++) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const uint32_t c = (v * kTeam + t) * 8u + i;
                if (c < a.hidden) shared_dw[team * a.hidden + c] = dw[v][i];
            }
        }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < a.hidden; c += kThreads) {
            float sum = shared_dw[c];
            for (uint32_t i = 1; i < kTeams; i++) sum += shared_dw[i * a.hidden + c];
            to[c] = sum;
        }
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
    if (hidden <= 16384u) return K3_SIZE(1024u, 2u);
    if (hidden <= 32768u) return K3_SIZE(1024u, 4u);
    return K3_SIZE(1024u, 8u);
#undef K3_SIZE
}

template <bool kF32, bool kVector>
bool launch_norm(const NormArgs &a, cudaStream_t stream) {
    return by_size(a.hidden, [&](auto team, auto vectors) {
        constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
        return launch_chained(norm_kernel<kF32, kVector, kTeam, decltype(vectors)::value>, (a.rows + kTeams - 1u) / kTeams, kThreads, 0,
                              stream, a);
    });
}

// Blocks of the gradient: two per SM of a B200, so that the partial rows of the weight's gradient do not depend on
// the device.
constexpr uint32_t kGradBlocks = 296;
uint32_t grad_blocks(uint32_t rows, uint32_t hidden) {
    const uint32_t teams = hidden <= 1024u ? 8u : 1u;
    return std::min((rows + teams - 1u) / teams, kGradBlocks);
}

template <bool kF32, bool kVector>
bool launch_backward(const NormGradArgs &a, cudaStream_t stream) {
    return by_size(a.hidden, [&](auto team, auto vectors) {
        constexpr uint32_t kTeam = decltype(team)::value, kThreads = threads_of(kTeam), kTeams = kThreads / kTeam;
        return launch_chained(norm_backward_kernel<kF32, kVector, kTeam, decltype(vectors)::value>, grad_blocks(a.rows, a.hidden), kThreads,
                              kTeams > 1u ? kTeams * a.hidden * 4u : 0u, stream, a);
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
    const bool vector = hidden % 8u == 0u && aligned(sum, 16u) && aligned(x, 16u) && aligned(residual, 16u) && aligned(weight, 16u) &&
                        aligned(y, 16u);
    if (f32) return vector ? launch_norm<true, true>(a, (cudaStream_t)stream) : launch_norm<true, false>(a, (cudaStream_t)stream);
    return vector ? launch_norm<false, true>(a, (cudaStream_t)stream) : launch_norm<false, false>(a, (cudaStream_t)stream);
}

extern "C" size_t k3_moe_norm_workspace_bytes(uint32_t rows, uint32_t hidden) {
    if (rows == 0u || !sizes_ok(rows, hidden, K3_MOE_NORM_F32)) return 0;
    return ((size_t)grad_blocks(rows, hidden) * hidden * 4u + 15u) / 16u * 16u;
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
    const bool vector = hidden % 8u == 0u && aligned(dx, 16u) && aligned(dy, 16u) && aligned(sum, 16u) && aligned(d_sum, 16u) &&
                        aligned(weight, 16u);
    const bool ok = f32 ? (vector ? launch_backward<true, true>(a, (cudaStream_t)stream) : launch_backward<true, false>(a, (cudaStream_t)stream))
                        : (vector ? launch_backward<false, true>(a, (cudaStream_t)stream) : launch_backward<false, false>(a, (cudaStream_t)stream));
    if (!ok || !d_weight) return ok;
    return launch_chained(norm_weight_kernel, (hidden + 31u) / 32u, 256, 0, (cudaStream_t)stream, (float *)d_weight,
                          (const float *)workspace, grad_blocks(rows, hidden), hidden, accumulate);
}
