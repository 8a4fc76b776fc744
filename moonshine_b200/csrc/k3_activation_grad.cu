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
// SwiGLU 127 to 129 us, 6.3 TB/s, SiTU 135, with three exponentials and three reciprocals per element.  SiTU with a block per row
// spills 44 bytes of registers under the bound of five blocks per SM.
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

// Of the activation itself, for two elements.
struct Derived {
    uint64_t d_gate, d_up, act;
};

K3_DEVINL uint64_t pair_of(uint32_t v) { return pack2(bf16_lo(v), bf16_hi(v)); }
K3_DEVINL uint32_t bf16_of(uint64_t v) { return bf16x2(lo2(v), hi2(v)); }
// exp(-by x)
K3_DEVINL float exp_of(float by, float x) { return exp2_fast(-by * kLog2E * x); }
K3_DEVINL uint64_t reciprocal2(uint64_t d) { return pack2(reciprocal_fast(lo2(d)), reciprocal_fast(hi2(d))); }

// tanh x = (1 - e) / (1 + e) and 1 / (4 cosh^2 x), e = exp(-2 |x|).  Below 0.1, where 1 - e would lose the value's bits,
// tanh x = x - x^3 / 3 + 2 x^5 / 15, whose next term is 6e-8 of the value.
struct Bounded {
    uint64_t tanh, slope;
};
K3_DEVINL float tanh_of(float x, float near, float far) { return fabsf(x) < 0.1f ? near : copysignf(far, x); }
K3_DEVINL Bounded bounded(uint64_t x) {
    const uint64_t one = both2(1.0f), y = mul2(x, x);
    const uint64_t e = pack2(exp_of(2.0f, fabsf(lo2(x))), exp_of(2.0f, fabsf(hi2(x))));
    const uint64_t r = reciprocal2(add2(e, one)), far = mul2(fma2(e, both2(-1.0f), one), r);
    const uint64_t near = fma2(mul2(x, y), fma2(y, both2(2.0f / 15.0f), both2(-1.0f / 3.0f)), x);
    return {pack2(tanh_of(lo2(x), lo2(near), lo2(far)), tanh_of(hi2(x), hi2(near), hi2(far))), mul2(mul2(e, r), r)};
}

// Two elements at a time: element by element the arithmetic bounds SiTU (32768 x 2048, one array for all inputs: 180 us, 149 in
// pairs, 98 SwiGLU, which the memory bounds).
template <bool kSitu>
K3_DEVINL Derived derive(const ActivationGradArgs &a, uint64_t g, uint64_t u) {
    // s = 1 / (1 + e), 1 - s = e / (1 + e).  From 88 on both s and s g are 0, and e stays finite.
    const uint64_t e = pack2(exp_of(1.0f, fmaxf(lo2(g), -88.0f)), exp_of(1.0f, fmaxf(hi2(g), -88.0f)));
    const uint64_t sig = reciprocal2(add2(e, both2(1.0f))), rest = mul2(e, sig);
    if (!kSitu) {
        const uint64_t left = mul2(g, sig);
        return {mul2(fma2(left, rest, sig), u), left, mul2(left, u)};
    }
    const Bounded x = bounded(mul2(g, both2(a.by_beta))), y = bounded(mul2(u, both2(a.by_linear_beta)));
    const uint64_t left = mul2(mul2(x.tanh, both2(a.beta)), sig), right = mul2(y.tanh, both2(a.linear_beta)), four = both2(4.0f);
    return {mul2(fma2(mul2(x.slope, four), sig, mul2(left, rest)), right), mul2(left, mul2(y.slope, four)), mul2(left, right)};
}

template <bool kSitu, bool kVector, uint32_t kTeam>
__global__ void __launch_bounds__(kThreads, kSitu && kVector ? 5 : 0) activation_grad_kernel(ActivationGradArgs a) {
    pdl_wait();
    __shared__ float scratch[kThreads / kWarp];
    const uint32_t t = threadIdx.x % kTeam;
    const uint64_t row = (uint64_t)blockIdx.x * (kThreads / kTeam) + threadIdx.x / kTeam;
    const bool live = row < a.rows && (a.offsets == nullptr || (row >= a.offsets[0] && row < a.offsets[a.groups]));
    uint64_t sums = 0ull;
    uint32_t route = 0u;
    bool routed = false;
    if (live) {
        route = a.routes ? a.routes[row] : (uint32_t)row;
        routed = route < a.route_count;
        const float weight = !routed ? 0.0f : a.weights ? a.weights[route] : 1.0f;
        const uint64_t base = row * a.columns, weight2 = both2(weight);
        // a thread's eight columns are neighbours, or (rows that are not whole vectors) kTeam apart
        constexpr uint32_t kStep = kVector ? 1u : kTeam;
        // vectors are loaded a step ahead (SiTU 156 us -> 139, with five blocks per SM 135; SwiGLU 129 either way, 133 with five)
        uint4 ng{}, nu{}, nd{};
        auto load = [&](uint32_t c) {
            if (kVector && c < a.columns) {
                ng = *reinterpret_cast<const uint4 *>(a.gate + base + c);
                nu = *reinterpret_cast<const uint4 *>(a.up + base + c);
                nd = *reinterpret_cast<const uint4 *>(a.d_out + base + c);
            }
        };
        load(t * 8u);
        for (uint32_t c = kVector ? t * 8u : t; c < a.columns; c += kTeam * 8u) {
            uint32_t g[4] = {}, u[4] = {}, d[4] = {};
            if (kVector) {
                const uint4 vg = ng, vu = nu, vd = nd;
                load(c + kTeam * 8u);
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
                const Derived f = derive<kSitu>(a, pair_of(g[i]), pair_of(u[i]));
                const uint64_t out = pair_of(d[i]), weighted = mul2(out, weight2);
                sums = fma2(out, f.act, sums);                          // + 0 past the row's end
                dg[i] = bf16_of(mul2(weighted, f.d_gate));
                du[i] = bf16_of(mul2(weighted, f.d_up));
                sc[i] = bf16_of(mul2(weight2, f.act));
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
    float sum = warp_sum(lo2(sums) + hi2(sums));
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
