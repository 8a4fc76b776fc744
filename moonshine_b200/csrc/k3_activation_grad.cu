// Gradient of the gated activation between an expert's products, with the routing weights (k3_moe_ops.h).
//
//   act = left(gate) right(up):  SwiGLU  left = g s(g),                right = u
//                                SiTU    left = b tanh(g / b) s(g),    right = l tanh(u / l)
//   d_gate = w d left'(g) right,  d_up = w d left right',  scaled = w act,  d_weights[route] = sum of d act
// with s the sigmoid and, without cancellation where they are small,
//   left' = s + g s (1 - s)   or   s / cosh^2(g / b) + left (1 - s),     right' = 1   or   1 / cosh^2(u / l)
//   1 - s(|g|) = e / (1 + e), e = exp(-|g|);     1 / cosh^2 x = 4 e / (1 + e)^2, e = exp(-2 |x|)
//
// Bound by memory: 12 bytes per element, each read or written once.  A row belongs to a warp, or, where there are
// fewer rows than warps to fill the SMs, to a block; its sum for the routing weight is taken in a fixed order.  32768 x 2048:
// 127 us, 6.3 TB/s.
#include "k3_common.cuh"
#include "k3_fp8_ptx.cuh"
#include "k3_moe_ops.h"

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kThreads = 256;

struct ActivationGradArgs {
    uint16_t *d_gate, *d_up, *scaled;
    float *d_weights;
    const uint16_t *d_out, *gate, *up;
    const float *weights;
    const uint32_t *routes, *offsets;
    uint32_t groups, rows, columns, route_count;
    float beta, by_beta, linear_beta, by_linear_beta;
};

struct Derived {
    float d_gate, d_up, act;                     // of the activation itself
};

// tanh x and 1 / cosh^2 x of one exponential and one reciprocal (with two of each the exponential unit bound SiTU, 32768 x
// 2048 at 215 us).  tanh: its Taylor series up to x^11 below 0.4, where the next term is 6e-8 of the value.
struct Bounded {
    float tanh, slope;
};
K3_DEVINL Bounded bounded(float x) {
    const float e = __expf(-2.0f * fabsf(x)), r = __fdividef(1.0f, 1.0f + e), y = x * x;
    float p = fmaf(y, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(y, p, -17.0f / 315.0f);
    p = fmaf(y, p, 2.0f / 15.0f);
    p = fmaf(y, p, -1.0f / 3.0f);
    return {fabsf(x) < 0.4f ? fmaf(x * y, p, x) : copysignf((1.0f - e) * r, x), 4.0f * e * r * r};
}

template <bool kSitu>
K3_DEVINL Derived derive(const ActivationGradArgs &a, float g, float u) {
    const float e = __expf(-fabsf(g)), r = __fdividef(1.0f, 1.0f + e);
    const float sig = g >= 0.0f ? r : e * r, rest = g >= 0.0f ? e * r : r;
    if (!kSitu) {
        const float left = g * sig;
        return {fmaf(left, rest, sig) * u, left, left * u};
    }
    const Bounded x = bounded(g * a.by_beta), y = bounded(u * a.by_linear_beta);
    const float left = a.beta * x.tanh * sig, right = a.linear_beta * y.tanh;
    return {fmaf(x.slope, sig, left * rest) * right, left * y.slope, left * right};
}

template <bool kSitu, bool kVector, uint32_t kTeam>
__global__ void __launch_bounds__(kThreads) activation_grad_kernel(ActivationGradArgs a) {
    pdl_wait();
    __shared__ float scratch[kThreads / kWarp];
    const uint32_t t = threadIdx.x % kTeam;
    const uint64_t row = (uint64_t)blockIdx.x * (kThreads / kTeam) + threadIdx.x / kTeam;
    const bool live = row < a.rows && (a.offsets == nullptr || (row >= a.offsets[0] && row < a.offsets[a.groups]));
    float sum = 0.0f;
    uint32_t route = 0u;
    bool routed = false;
    if (live) {
        route = a.routes ? a.routes[row] : (uint32_t)row;
        routed = route < a.route_count;
        const float weight = !routed ? 0.0f : a.weights ? a.weights[route] : 1.0f;
        const uint64_t base = row * a.columns;
        // a thread's eight columns are neighbours, or (rows that are not whole vectors) kTeam apart
        constexpr uint32_t kStep = kVector ? 1u : kTeam;
        for (uint32_t c = kVector ? t * 8u : t; c < a.columns; c += kTeam * 8u) {
            uint32_t g[4] = {}, u[4] = {}, d[4] = {};
            if (kVector) {
                const uint4 vg = *reinterpret_cast<const uint4 *>(a.gate + base + c), vu = *reinterpret_cast<const uint4 *>(a.up + base + c);
                const uint4 vd = *reinterpret_cast<const uint4 *>(a.d_out + base + c);
                g[0] = vg.x; g[1] = vg.y; g[2] = vg.z; g[3] = vg.w;
                u[0] = vu.x; u[1] = vu.y; u[2] = vu.z; u[3] = vu.w;
                d[0] = vd.x; d[1] = vd.y; d[2] = vd.z; d[3] = vd.w;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    if (c + i * kStep >= a.columns) continue;
                    const uint64_t at = base + c + i * kStep;
                    g[i / 2u] |= (uint32_t)a.gate[at] << (16u * (i & 1u));
                    u[i / 2u] |= (uint32_t)a.up[at] << (16u * (i & 1u));
                    d[i / 2u] |= (uint32_t)a.d_out[at] << (16u * (i & 1u));
                }
            }
            uint32_t dg[4], du[4], sc[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const Derived lo = derive<kSitu>(a, bf16_lo(g[i]), bf16_lo(u[i])), hi = derive<kSitu>(a, bf16_hi(g[i]), bf16_hi(u[i]));
                const float d0 = bf16_lo(d[i]), d1 = bf16_hi(d[i]);
                sum = fmaf(d0, lo.act, sum);                          // + 0 past the row's end
                sum = fmaf(d1, hi.act, sum);
                const float w0 = weight * d0, w1 = weight * d1;
                dg[i] = bf16x2(w0 * lo.d_gate, w1 * hi.d_gate);
                du[i] = bf16x2(w0 * lo.d_up, w1 * hi.d_up);
                sc[i] = bf16x2(weight * lo.act, weight * hi.act);
            }
            if (kVector) {
                *reinterpret_cast<uint4 *>(a.d_gate + base + c) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
                *reinterpret_cast<uint4 *>(a.d_up + base + c) = make_uint4(du[0], du[1], du[2], du[3]);
                if (a.scaled) *reinterpret_cast<uint4 *>(a.scaled + base + c) = make_uint4(sc[0], sc[1], sc[2], sc[3]);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) {
                    if (c + i * kStep >= a.columns) continue;
                    const uint64_t at = base + c + i * kStep;
                    a.d_gate[at] = (uint16_t)(dg[i / 2u] >> (16u * (i & 1u)));
                    a.d_up[at] = (uint16_t)(du[i / 2u] >> (16u * (i & 1u)));
                    if (a.scaled) a.scaled[at] = (uint16_t)(sc[i / 2u] >> (16u * (i & 1u)));
                }
            }
        }
    }
    if (a.d_weights == nullptr) return;
    sum = warp_sum(sum);
    if (kTeam != kWarp) {
        if (threadIdx.x % kWarp == 0u) scratch[threadIdx.x / kWarp] = sum;
        __syncthreads();
        sum = warp_sum(threadIdx.x % kWarp < kThreads / kWarp ? scratch[threadIdx.x % kWarp] : 0.0f);
    }
    if (routed && t == 0u) a.d_weights[route] = sum;
}

template <bool kSitu, bool kVector>
bool launch(const ActivationGradArgs &a, cudaStream_t stream) {
    // a warp per row where it has few steps and there are warps enough (us, warp / block: 8192 x 2048 33 / 33, 2368 x 2048
    // 16 / 14, 4096 x 1024 12 / 16, 4096 x 512 8 / 14, 300 x 512 8 / 6)
    if (a.rows >= (uint32_t)sm_count() * 8u && a.rows >= 4u * (uint64_t)a.columns) {
        return launch_chained(activation_grad_kernel<kSitu, kVector, kWarp>, (a.rows + kThreads / kWarp - 1u) / (kThreads / kWarp), kThreads, 0,
                              stream, a);
    }
    return launch_chained(activation_grad_kernel<kSitu, kVector, kThreads>, a.rows, kThreads, 0, stream, a);
}

bool aligned(const void *p, uint32_t bytes) { return ((uintptr_t)p & (bytes - 1u)) == 0u; }

}  // namespace

extern "C" bool k3_moe_activation_backward(void *d_gate, void *d_up, void *scaled, void *d_weights, const void *d_out, const void *gate,
                                           const void *up, const void *weights, const void *routes, const void *offsets, uint32_t groups,
                                           uint32_t rows, uint32_t columns, uint32_t route_count, int activation, float beta,
                                           float linear_beta, void *stream) {
    if (!d_gate || !d_up || !d_out || !gate || !up || rows == 0u || rows > (1u << 30) || columns == 0u || columns > (1u << 30)) return false;
    if (activation != kActSitu && activation != kActSwiglu) return false;
    if (activation == kActSitu && !(beta > 0.0f && linear_beta > 0.0f)) return false;
    bool vector = columns % 8u == 0u;
    for (const void *p : {(const void *)d_gate, (const void *)d_up, (const void *)scaled, d_out, gate, up}) {
        if (!aligned(p, 2u)) return false;
        vector = vector && aligned(p, 16u);
    }
    if (!aligned(d_weights, 4u) || !aligned(weights, 4u) || !aligned(routes, 4u) || !aligned(offsets, 4u)) return false;
    const ActivationGradArgs a{(uint16_t *)d_gate, (uint16_t *)d_up, (uint16_t *)scaled, (float *)d_weights, (const uint16_t *)d_out,
                               (const uint16_t *)gate, (const uint16_t *)up, (const float *)weights, (const uint32_t *)routes, (const uint32_t *)offsets, groups,
                               rows, columns, route_count, beta, 1.0f / beta, linear_beta, 1.0f / linear_beta};
    if (activation == kActSitu) return vector ? launch<true, true>(a, (cudaStream_t)stream) : launch<true, false>(a, (cudaStream_t)stream);
    return vector ? launch<false, true>(a, (cudaStream_t)stream) : launch<false, false>(a, (cudaStream_t)stream);
}
