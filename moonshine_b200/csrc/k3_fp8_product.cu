// Products of E4M3 matrices with one f32 scale per block of 128: the entry point and the choice of kernel.
#include "k3_fp8.h"

using namespace k3::fp8;

// Lanes for b's rows or for a's.  One matrix, 7168 x 7168, us of b's rows as lanes / of a's: 1 row 11.7 / 13.6, 16 rows
// 12.0 / 14.0, 17 (64 columns instead of 16) 18.3 / 14.2, 128 31.5 / 17.1; 2048 x 7168 1 row 6.3 / 7.8, 17 rows 9.2 / 8.5.
// Groups of 7168 x 2048, a whole call through 16 of 64 experts chosen evenly: 16 rows a group on average 474 / 537, 32
// 503 / 539, 40 513 / 551, 48 526 / 564, 64 704 / 584; of 896: 5 rows 6351 / 8416, 37 6973 / 8710, 41 7128 / 9390, 73
// 12726 / 9631.  The average is what the host knows.  Where the choice is skewed the long groups decide: 896 experts, 37
// rows on average, by Zipf 5241 / 4514 and with one in 20 chosen 3439 / 2415; 2000 tokens through one expert 232 / 167.
bool k3::fp8::product(const Product &p, cudaStream_t stream) {
    const bool few = p.offsets ? grouped_few(p.rows, p.groups) : p.rows <= few_linear_rows;
    if (few && p.b_scale_layout == K3_MOE_FP8_BLOCKS) return few_product(p, stream);
    return wide_product(p, stream);
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
