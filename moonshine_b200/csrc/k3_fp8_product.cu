// Products of E4M3 matrices with one f32 scale per block of 128:
//
//   out[m, n] = sum_kb sa[m, kb] sb[n or n / 128, kb] sum_{k in kb} a[m, k] b[n, k]
//
// One block of threads computes 64 x 128 of the result from codes turned to f32 in shared memory; a
// block's sum is scaled and added to a running f32 sum.
#include "k3_common.cuh"
#include "k3_fp8.h"
#include "k3_moe_layer.h"
#include "k3_moe_ops.h"

#include <cuda_fp8.h>

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kThreads = 256, BM = 64, BN = 128, BK = 32;

K3_DEVINL float code_value(uint8_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

struct Span {
    uint32_t begin, end, group;
};

// row tile t of the groups in order (a tile never crosses a group)
K3_DEVINL Span span_of(const Product &p, uint32_t t) {
    if (p.offsets == nullptr) return {t * BM, min(p.rows, t * BM + BM), 0u};
    for (uint32_t g = 0; g < p.groups; g++) {
        const uint32_t begin = p.offsets[g], n = p.offsets[g + 1u] - begin, tiles = (n + BM - 1u) / BM;
        if (t < tiles) return {begin + t * BM, min(begin + n, begin + t * BM + BM), g};
        t -= tiles;
    }
    return {0u, 0u, 0u};
}

// acc[i][j] += rows begin + 4 ty' .. of a times rows n0 + tx + 16 j of b
K3_DEVINL void multiply(float (&acc)[4][8], const Product &p, const Span &s, uint32_t n0, const uint8_t *b, const float *bs,
                        float (*as)[BK + 1], float (*bt)[BK + 1]) {
    const uint32_t pitch = pitch_of(p.k), a_sp = scale_pitch_of(p.k), kb_count = blocks_of(p.k);
    const uint32_t tx = threadIdx.x % 16u, ty = threadIdx.x / 16u;
    const uint32_t b_sp = p.b_scale_layout == K3_MOE_FP8_ROWS ? a_sp : kb_count;
    for (uint32_t kb = 0; kb < kb_count; kb++) {
        float t[4][8] = {};
        for (uint32_t k0 = kb * kBlock; k0 < min(p.k, (kb + 1u) * kBlock); k0 += BK) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < BM * BK; i += kThreads) {
                const uint32_t r = s.begin + i / BK, k = k0 + i % BK;
                as[i / BK][i % BK] = r < s.end && k < p.k ? code_value(((const uint8_t *)p.a)[(uint64_t)r * pitch + k]) : 0.f;
            }
            for (uint32_t i = threadIdx.x; i < BN * BK; i += kThreads) {
                const uint32_t n = n0 + i / BK, k = k0 + i % BK;
                bt[i / BK][i % BK] = n < p.n && k < p.k ? code_value(b[(uint64_t)n * pitch + k]) : 0.f;
            }
            __syncthreads();
            for (uint32_t k = 0; k < BK; k++) {
                for (int i = 0; i < 4; i++) {
                    for (int j = 0; j < 8; j++) t[i][j] = fmaf(as[ty * 4u + i][k], bt[tx + 16u * j][k], t[i][j]);
                }
            }
        }
        for (int i = 0; i < 4; i++) {
            const uint32_t r = s.begin + ty * 4u + i;
            if (r >= s.end) continue;
            const float sa = ((const float *)p.a_scales)[(uint64_t)r * a_sp + kb];
            for (int j = 0; j < 8; j++) {
                const uint32_t n = n0 + tx + 16u * j;
                if (n >= p.n) continue;
                const float sb = bs[(uint64_t)(p.b_scale_layout == K3_MOE_FP8_ROWS ? n : n / kBlock) * b_sp + kb];
                acc[i][j] = fmaf(t[i][j], sa * sb, acc[i][j]);
            }
        }
    }
}

__global__ void __launch_bounds__(kThreads) product_kernel(Product p) {
    __shared__ float as[BM][BK + 1], bt[BN][BK + 1];
    pdl_wait();
    const Span s = span_of(p, blockIdx.y);
    if (s.begin >= s.end) return;
    const uint32_t n0 = blockIdx.x * BN, tx = threadIdx.x % 16u, ty = threadIdx.x / 16u;
    const uint64_t table = (uint64_t)s.group * p.n * pitch_of(p.k), scales = (uint64_t)s.group * blocks_of(p.n) * blocks_of(p.k);
    float acc[4][8] = {};
    multiply(acc, p, s, n0, (const uint8_t *)p.b + table, (const float *)p.b_scales + scales, as, bt);
    if (p.epilogue != kOutActivated) {
        for (int i = 0; i < 4; i++) {
            for (int j = 0; j < 8; j++) {
                const uint32_t r = s.begin + ty * 4u + i, n = n0 + tx + 16u * j;
                if (r >= s.end || n >= p.n) continue;
                const uint64_t at = (uint64_t)r * p.n + n;
                if (p.epilogue == kOutF32) {
                    float *to = (float *)p.out + at;
                    *to = p.accumulate ? *to + acc[i][j] : acc[i][j];
                } else {
                    ((uint16_t *)p.out)[at] = float_to_bf16_bits(acc[i][j]);
                }
            }
        }
        return;
    }
    float up[4][8] = {};
    multiply(up, p, s, n0, (const uint8_t *)p.b2 + table, (const float *)p.b2_scales + scales, as, bt);
    const uint32_t pitch = pitch_of(p.n), sp = scale_pitch_of(p.n);
    for (int i = 0; i < 4; i++) {
        uint32_t m = 0u;
        for (int j = 0; j < 8; j++) {
            const uint32_t n = n0 + tx + 16u * j;
            acc[i][j] = n < p.n ? activation(acc[i][j], up[i][j], p.activation, p.beta, p.linear_beta) : 0.f;
            m = max(m, __float_as_uint(acc[i][j]) & 0x7fffffffu);
        }
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float scale = m >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : fmaxf(__fdiv_rn(__uint_as_float(m), 448.f), 0x1p-126f);
        const uint32_t r = s.begin + ty * 4u + i;
        if (r >= s.end) continue;
        if (tx == 0u) ((float *)p.out_scales)[(uint64_t)r * sp + blockIdx.x] = scale;
        for (int j = 0; j < 8; j++) {
            const uint32_t n = n0 + tx + 16u * j;
            if (n < p.n) ((uint8_t *)p.out)[(uint64_t)r * pitch + n] = __nv_cvt_float_to_fp8(__fdiv_rn(acc[i][j], scale), __NV_SATFINITE, __NV_E4M3);
        }
    }
}

}  // namespace

bool k3::fp8::product(const Product &p, cudaStream_t stream) {
    const uint32_t tiles = (p.rows + BM - 1u) / BM + (p.offsets ? p.groups : 0u);
    return tiles <= 65535u && launch_chained(product_kernel, dim3(blocks_of(p.n), tiles), kThreads, 0, stream, p);
}

extern "C" bool k3_moe_fp8_product(void *out, const void *a, const void *a_scales, const void *b, const void *b_scales,
                                   uint32_t m, uint32_t n, uint32_t k, int b_scale_layout, int out_type, int accumulate,
                                   void *stream) {
    if (!out || !a || !a_scales || !b || !b_scales || !extent_ok(m) || !extent_ok(n) || !extent_ok(k) || !aligned16(a) ||
        !aligned16(a_scales) || !aligned16(b) || ((uintptr_t)b_scales & (b_scale_layout == K3_MOE_FP8_ROWS ? 15u : 3u)) != 0u ||
        (b_scale_layout != K3_MOE_FP8_BLOCKS && b_scale_layout != K3_MOE_FP8_ROWS) ||
        (out_type != K3_MOE_FP8_BF16 && out_type != K3_MOE_FP8_F32) || (accumulate && out_type != K3_MOE_FP8_F32) ||
        ((uintptr_t)out & (out_type == K3_MOE_FP8_F32 ? 3u : 1u)) != 0u) {
        return false;
    }
    Product p{};
    p.out = out;
    p.a = a;
    p.a_scales = a_scales;
    p.b = b;
    p.b_scales = b_scales;
    p.groups = 1u;
    p.rows = m;
    p.n = n;
    p.k = k;
    p.b_scale_layout = b_scale_layout;
    p.epilogue = out_type == K3_MOE_FP8_F32 ? kOutF32 : kOutBf16;
    p.accumulate = accumulate;
    return product(p, (cudaStream_t)stream);
}
