// What the E4M3 product kernels add to k3_tc_ptx.cuh: the kind::f8f6f4 MMA, register shares of
// warpgroups, scales and codes, tensor maps of code matrices.
#pragma once

#include "k3_fp8.h"
#include "k3_tc_ptx.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

namespace k3::fp8 {

using namespace k3::tc;

// Instruction descriptor, kind::f8f6f4: D f32 (bits 4..5 = 1), A and B E4M3 (0), both K-major, N >> 3 at bit 17, M >> 4 at 24.
K3_DEVINL constexpr uint32_t make_idesc_e4m3(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

// D[tmem] (+)= A[smem] B[smem]^T over 32 E4M3 columns
K3_DEVINL void mma_e4m3_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

K3_DEVINL uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <uint32_t kRegisters>
K3_DEVINL void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters)); }
template <uint32_t kRegisters>
K3_DEVINL void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters)); }

// tcgen05.wait::ld that the loaded registers depend on: no use of them moves in front of it
K3_DEVINL void tmem_ld_wait_for(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

// A wait that does not stop for the abort flag: for copies in flight, on the way out.
K3_DEVINL void mbar_drain(uint64_t *bar, uint32_t parity) {
    const unsigned long long t0 = global_timer_ns();
    while (!mbar_try_wait(bar, parity) && global_timer_ns() - t0 < 100000000ull) {}
}

// The expert activation with the fast exponential and reciprocal, 4e-7 of the result and, of a negative gate, 1.4e-7 times
// its size (the exponent's rounding), where the result is small: it is quantised to 4 bits next.
// The kind is a template argument, so that many elements go side by side: with a branch in each of a thread's elements
// the warps waited for one element's chain after the other.
//
// tanh x: its Taylor series up to x^11 below 0.4, where the next term is 6e-8 of the value, and 1 - 2 / (1 + e^2x)
// above, which is off by 1e-7.
K3_DEVINL float tanh_fast(float x) {
    const float y = x * x;
    float p = fmaf(y, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    p = fmaf(y, p, -17.0f / 315.0f);
    p = fmaf(y, p, 2.0f / 15.0f);
    p = fmaf(y, p, -1.0f / 3.0f);
    const float small = fmaf(x * y, p, x), large = fmaf(-2.0f, __fdividef(1.0f, 1.0f + __expf(2.0f * x)), 1.0f);
    return fabsf(x) < 0.4f ? small : large;
}
template <bool kSitu>
struct ExpertActivation {
    float beta, by_beta, linear, by_linear;        // by_: the reciprocals
    K3_DEVINL float operator()(float g, float u) const {
        const float sig = __fdividef(1.0f, 1.0f + __expf(-g));
        if (kSitu) return beta * tanh_fast(g * by_beta) * sig * (linear * tanh_fast(u * by_linear));
        return g * sig * u;
    }
};

// The same for two elements at a time, with the sign turned around.
// 1 / (c + c e^(x s)), with s times log2 e
K3_DEVINL uint64_t logistic2(uint64_t x, float s, float c) {
    const uint64_t t = mul2(x, both2(s));
    const uint64_t d = fma2(pack2(exp2_fast(lo2(t)), exp2_fast(hi2(t))), both2(c), both2(c));
    return pack2(reciprocal_fast(lo2(d)), reciprocal_fast(hi2(d)));
}
K3_DEVINL uint64_t tanh2(uint64_t x) {
    const uint64_t y = mul2(x, x);
    uint64_t p = fma2(y, both2(-1382.0f / 155925.0f), both2(62.0f / 2835.0f));
    p = fma2(y, p, both2(-17.0f / 315.0f));
    p = fma2(y, p, both2(2.0f / 15.0f));
    p = fma2(y, p, both2(-1.0f / 3.0f));
    const uint64_t small = fma2(mul2(x, y), p, x), large = fma2(both2(-2.0f), logistic2(x, 2.0f * kLog2E, 1.0f), both2(1.0f));
    return pack2(fabsf(lo2(x)) < 0.4f ? lo2(small) : lo2(large), fabsf(hi2(x)) < 0.4f ? hi2(small) : hi2(large));
}
template <bool kSitu>
K3_DEVINL uint64_t negative_activation2(const ExpertActivation<kSitu> &a, uint64_t g, uint64_t u) {
    const uint64_t sig = logistic2(g, -kLog2E, -1.0f);
    if (kSitu) return mul2(mul2(mul2(tanh2(mul2(g, both2(a.by_beta))), both2(a.beta * a.linear)), sig), tanh2(mul2(u, both2(a.by_linear))));
    return mul2(mul2(g, sig), u);
}

// ------------------------------------------------------------------------------------------- codes
// x / by as an f32 division gives it: the product with the rounded reciprocal, corrected once by its
// remainder (Markstein 1990).  The remainder is taken from the product, and its negative added: the other way
// round -0 would become 0.
K3_DEVINL float divided(float x, float by, float inverse) {
    const float r = x * inverse;
    return fmaf(fmaf(r, by, -x), -inverse, r);
}
// scale of a block whose largest magnitude has these bits (without the sign): that over 448
K3_DEVINL float scale_of(uint32_t largest_bits) {
    if (largest_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
    return fmaxf(divided(__uint_as_float(largest_bits), 448.0f, 1.0f / 448.0f), 0x1p-126f);
}
// Below 2^-90 the remainders are subnormal and lose bits, so there x and the scale are both multiplied by 2^64.
K3_DEVINL float lift_of(float scale) { return scale < 0x1p-90f ? 0x1p64f : 1.0f; }
// 1 / (scale lift), rounded once: Newton's iteration from an estimate within two units of the last place, which ends
// beside the rounded value only where the mantissa is all ones (Markstein 1990).  No subroutine, as f32 division and
// the rounded reciprocal have for their rare cases: where the kernel of the wide products called one, its main loop
// moved the running sums between registers.
K3_DEVINL float inverse_of(float scale) {
    const float by = scale * lift_of(scale);
    float y = reciprocal_fast(by);
    y = fmaf(y, fmaf(-by, y, 1.0f), y);
    y = fmaf(y, fmaf(-by, y, 1.0f), y);
    return (__float_as_uint(by) & 0x7fffffu) == 0x7fffffu ? __uint_as_float(__float_as_uint(y) | 1u) : y;
}
// x / scale; inverse: inverse_of(scale)
K3_DEVINL float quotient(float x, float scale, float inverse) {
    const float lift = lift_of(scale);
    return divided(x * lift, scale * lift, inverse);
}
// divided() for two elements, given as -x; the divisor and the negative of its reciprocal, twice each
K3_DEVINL uint64_t divided2(uint64_t negative_x, uint64_t by, uint64_t negative_inverse) {
    const uint64_t r = mul2(negative_x, negative_inverse);
    return fma2(fma2(r, by, negative_x), negative_inverse, r);
}
// two codes, `lo` in the low byte
K3_DEVINL uint32_t codes2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// ------------------------------------------------------------------------------------- tensor maps
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess) {
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
        } else {
            (void)cudaGetLastError();
        }
    });
    return fn;
}

// Codes [rows, columns] with rows on 16 bytes; boxes of 128 columns x box_rows, 128-byte swizzle.  What lies past the
// columns reads as zero, whatever the padding holds.
inline bool map_codes(CUtensorMap *map, const void *codes, uint64_t rows, uint32_t columns, uint32_t box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {columns, rows};
    const cuuint64_t strides[1] = {pitch_of(columns)};
    const cuuint32_t box[2] = {kBlock, box_rows};
    const cuuint32_t steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace k3::fp8
