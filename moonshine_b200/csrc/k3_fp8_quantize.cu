// Matrices to E4M3 codes with one f32 scale per block of 128: of a row, of a column (transposed), of a
// 128 x 128 tile; and a weight table's transposed layout.
//
//   scale = max(largest |x| of the block / 448, 2^-126),  code = e4m3(x / scale)
//
// Both quotients are those of f32 division.  One division per block gives the scale, one its
// reciprocal; an element's quotient is then the product with the reciprocal, corrected once by its
// remainder (Markstein 1990: with a correctly rounded reciprocal this is the rounded quotient), three
// operations in place of a division.  The distance matters: where the largest magnitude of bf16 data
// is a multiple of 7, one element in some hundred lies exactly between two codes.
//
// The largest magnitude is taken of the bit patterns without their signs, which order like the
// values and put infinities and NaN above all of them; a block with one gets the scale NaN.
#include "k3_common.cuh"
#include "k3_fp8_ptx.cuh"

using namespace k3;
using namespace k3::fp8;

namespace {

constexpr uint32_t kThreads = 256;

// Eight neighbouring elements as they lie in memory: bf16 stay packed until they are used, which leaves
// registers for more blocks of threads on an SM, and these for more bytes in flight.
template <bool kF32>
struct Eight {
    static constexpr uint32_t kWords = kF32 ? 8u : 4u;
    uint32_t w[kWords];

    // elements c .. c + 7 of a row, zeros past its end.  kVector: the row starts on 16 bytes and is a
    // multiple of 8 elements long.
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
    K3_DEVINL float value(uint32_t i) const {
        if (kF32) return __uint_as_float(w[i % kWords]);
        return i & 1u ? bf16_hi(w[i / 2u]) : bf16_lo(w[i / 2u]);
    }
    // largest magnitudes: one word for f32, both halves of a word for bf16
    K3_DEVINL uint32_t largest() const {
        uint32_t m = magnitude(w[0]);
#pragma unroll
        for (uint32_t i = 1; i < kWords; i++) m = larger(m, magnitude(w[i]));
        return m;
    }
    static K3_DEVINL uint32_t magnitude(uint32_t x) { return x & (kF32 ? 0x7fffffffu : 0x7fff7fffu); }
    static K3_DEVINL uint32_t larger(uint32_t a, uint32_t b) {
        if (kF32) return max(a, b);
        uint32_t r;
        asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    // of a word of larger(): the f32 bits
    static K3_DEVINL uint32_t bits(uint32_t m) { return kF32 ? m : max(m & 0xffff0000u, m << 16); }
    // quotient() with the rare lift in a branch: 8192 x 7168 in 29.6 us, 0.9 less without any lift
    K3_DEVINL uint2 codes(float scale, float inverse) {
        const float lift = lift_of(scale), by = scale * lift;
        if (lift != 1.0f) {
#pragma unroll
            for (uint32_t i = 0; i < kWords; i++) {                  // exact in bf16 as well
                w[i] = kF32 ? __float_as_uint(value(i) * lift) : bf16x2(value(2u * i) * lift, value(2u * i + 1u) * lift);
            }
        }
        uint32_t h[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            h[i] = codes2(divided(value(2u * i), by, inverse), divided(value(2u * i + 1u), by, inverse));
        }
        return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
    }
};

// Eight codes from column c on, zeros past the columns: there the quotient is one of 0, which a block's NaN scale makes NaN.
// kVector as in load().
template <bool kVector>
K3_DEVINL uint2 inside(uint2 codes, uint32_t c, uint32_t columns) {
    if (c + 8u <= columns) return codes;
    if (kVector || c >= columns) return make_uint2(0u, 0u);
    const uint32_t left = columns - c;
    return make_uint2(left < 4u ? codes.x & ((1u << (8u * left)) - 1u) : codes.x,
                      left > 4u ? codes.y & ((1u << (8u * (left - 4u))) - 1u) : 0u);
}

// ------------------------------------------------------------------------------------------- rows
// Half a warp takes four neighbouring blocks of a row: lane l holds elements 8 l .. 8 l + 7 of each.
struct RowsArgs {
    uint8_t *codes;
    float *scales;
    const void *x;
    uint32_t rows, columns, tasks_per_row;
    Placement at;
    uint4 *zero_row;                 // cleared on the way (zero_units 16-byte units), or null
    uint32_t zero_units;
};

template <bool kF32, bool kVector, bool kPlaced>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(RowsArgs a) {
    pdl_wait();
    if (kPlaced && blockIdx.x == 0u) {
        for (uint32_t i = threadIdx.x; i < a.zero_units; i += kThreads) a.zero_row[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    const uint32_t half = threadIdx.x / 16u, l = threadIdx.x % 16u;
    const uint64_t task = (uint64_t)blockIdx.x * (kThreads / 16u) + half;
    const uint32_t row = (uint32_t)task / a.tasks_per_row;
    const uint32_t group = (uint32_t)task - row * a.tasks_per_row;
    const bool live = task < (uint64_t)a.rows * a.tasks_per_row;     // the shuffles below want every lane
    const char *x = (const char *)a.x + (uint64_t)(live ? row : 0u) * a.columns * (kF32 ? 4u : 2u);
    // kPlaced: lane l has the places of the row's routes l and 16 + l
    constexpr uint32_t kNowhere = 0xffffffffu;
    uint32_t place[2] = {kNowhere, kNowhere};
#pragma unroll
    for (uint32_t h = 0; kPlaced && h < 2u; h++) {
        const uint32_t r = h * 16u + l, route = row * a.at.top_k + r;
        if (live && r < a.at.top_k) {
            if (a.at.ids[route] < a.at.experts) place[h] = a.at.place[route];
            else if (group == 0u) a.at.place[route] = a.at.spare;
        }
    }
    Eight<kF32> x8[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
        x8[b].template load<kVector>(x, (group * 4u + b) * kBlock + l * 8u, live ? a.columns : 0u);
    }
    pdl_trigger();                   // a product behind may fetch its table now (Product::b_ready)
    // lane l divides for block l % 4
    uint32_t most = 0u;
#pragma unroll
    for (int b = 0; b < 4; b++) {
        uint32_t m = x8[b].largest();
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = Eight<kF32>::larger(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (l % 4u == (uint32_t)b) most = m;
    }
    const float my_scale = scale_of(Eight<kF32>::bits(most)), my_inverse = inverse_of(my_scale);
    float scale[4];
    uint2 out[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
        scale[b] = __shfl_sync(0xffffffffu, my_scale, b, 16);
        out[b] = x8[b].codes(scale[b], __shfl_sync(0xffffffffu, my_inverse, b, 16));
        if ((group * 4u + b) * kBlock >= a.columns) scale[b] = 0.0f;  // padding of the scales' row
    }
    if ((group + 1u) * 4u * kBlock > a.columns) {                     // the row's last task: a test in each of all tasks took 2 of 33 us
#pragma unroll
        for (int b = 0; b < 4; b++) out[b] = inside<kVector>(out[b], (group * 4u + b) * kBlock + l * 8u, a.columns);
    }
    const uint32_t pitch = pitch_of(a.columns), scale_pitch = a.tasks_per_row * 4u;
    auto store = [&](uint32_t to) {
        if (l == 0u) {
            *reinterpret_cast<float4 *>(a.scales + (uint64_t)to * scale_pitch + group * 4u) =
                make_float4(scale[0], scale[1], scale[2], scale[3]);
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const uint32_t c = (group * 4u + b) * kBlock + l * 8u;
            if (c < pitch) *reinterpret_cast<uint2 *>(a.codes + (uint64_t)to * pitch + c) = out[b];
        }
    };
    if (!kPlaced) {
        if (live) store(row);
    } else {
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            for (uint32_t r = 0; r < 16u; r++) {
                const uint32_t to = __shfl_sync(0xffffffffu, place[h], r, 16);
                if (to != kNowhere) store(to);
                if (h * 16u + r + 1u >= a.at.top_k) break;
            }
            if (a.at.top_k <= 16u) break;
        }
    }
}

// ---------------------------------------------------------------------------------------- columns
// One block of threads takes 128 rows x 64 columns: thread (rt, ct) the rows 4 rt .. 4 rt + 3 of
// columns 8 ct .. 8 ct + 7.  Four codes of a column make one word of the transposed tile, which
// goes through shared memory and leaves as 128 contiguous bytes per column.
constexpr uint32_t kTileColumns = 64, kTileWords = 33;                // words per column, one to spare

template <bool kF32, bool kVector>
__global__ void __launch_bounds__(kThreads, kF32 ? 4 : 6)
quantize_columns_kernel(uint8_t *codes, float *scales, const void *x, uint32_t rows, uint32_t columns) {
    __shared__ uint32_t largest[8][kTileColumns];
    __shared__ uint32_t tile[kTileColumns * kTileWords];
    __shared__ float2 column_scale[kTileColumns];
    pdl_wait();
    const uint32_t r0 = blockIdx.y * kBlock, c0 = blockIdx.x * kTileColumns;
    const uint32_t ct = threadIdx.x % 8u, rt = threadIdx.x / 8u, warp = threadIdx.x / kWarp;
    Eight<kF32> x8[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t r = r0 + rt * 4u + i;
        const char *row = (const char *)x + (uint64_t)(r < rows ? r : 0u) * columns * (kF32 ? 4u : 2u);
        x8[i].template load<kVector>(row, c0 + ct * 8u, r < rows ? columns : 0u);
    }
    // of each column: this thread's four rows, the warp's four threads with the column, the eight warps
#pragma unroll
    for (uint32_t k = 0; k < Eight<kF32>::kWords; k++) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) m = Eight<kF32>::larger(m, Eight<kF32>::magnitude(x8[i].w[k]));
        m = Eight<kF32>::larger(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = Eight<kF32>::larger(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if (threadIdx.x % kWarp < 8u) {
            if (kF32) {
                largest[warp][ct * 8u + k] = m;
            } else {
                largest[warp][ct * 8u + 2u * k] = m << 16;
                largest[warp][ct * 8u + 2u * k + 1u] = m & 0xffff0000u;
            }
        }
    }
    __syncthreads();
    // a column's scale and reciprocal once, by one thread
    const uint32_t scale_pitch = scale_pitch_of(rows);
    if (threadIdx.x < kTileColumns) {
        uint32_t all = 0u;
#pragma unroll
        for (int w = 0; w < 8; w++) all = max(all, largest[w][threadIdx.x]);
        const float scale = scale_of(all);
        column_scale[threadIdx.x] = make_float2(scale, inverse_of(scale));
        if (c0 + threadIdx.x < columns) {
            float *to = scales + (uint64_t)(c0 + threadIdx.x) * scale_pitch + blockIdx.y;
            *to = scale;
            if (blockIdx.y + 1u == gridDim.y) {
                for (uint32_t p = 1u; blockIdx.y + p < scale_pitch; p++) to[p] = 0.0f;
            }
        }
    }
    __syncthreads();
    const uint32_t first = r0 + rt * 4u, mine = first < rows ? rows - first : 0u;          // this thread's rows that exist
    const uint32_t mask = mine >= 4u ? 0xffffffffu : (1u << (8u * mine)) - 1u;
#pragma unroll
    for (uint32_t j = 0; j < 8u; j++) {
        const float2 s = column_scale[ct * 8u + j];
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = quotient(x8[i].value(j), s.x, s.y);
        tile[(ct * 8u + j) * kTileWords + rt] = (codes2(q[0], q[1]) | (codes2(q[2], q[3]) << 16)) & mask;
    }
    __syncthreads();
    const uint32_t pitch = pitch_of(rows);
#pragma unroll
    for (uint32_t i = 0; i < 2u; i++) {
        const uint32_t unit = i * kThreads + threadIdx.x, c = unit / 8u, u = unit % 8u;
        const uint32_t r = r0 + u * 16u;
        if (c0 + c < columns && r < pitch) {
            const uint32_t *w = tile + c * kTileWords + u * 4u;
            *reinterpret_cast<uint4 *>(codes + (uint64_t)(c0 + c) * pitch + r) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ----------------------------------------------------------------------------------------- blocks
template <bool kF32, bool kVector>
__global__ void __launch_bounds__(kThreads)
quantize_blocks_kernel(uint8_t *codes, float *scales, const void *x, uint32_t rows, uint32_t columns) {
    __shared__ uint32_t largest[8];
    pdl_wait();
    const uint32_t r0 = blockIdx.y * kBlock, c = blockIdx.x * kBlock + (threadIdx.x % 16u) * 8u, rt = threadIdx.x / 16u;
    Eight<kF32> x8[8];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + i * 16u + rt;
        const char *row = (const char *)x + (uint64_t)(r < rows ? r : 0u) * columns * (kF32 ? 4u : 2u);
        x8[i].template load<kVector>(row, c, r < rows ? columns : 0u);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, Eight<kF32>::bits(x8[i].largest()));
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x % kWarp == 0u) largest[threadIdx.x / kWarp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) m = max(m, largest[w]);
    const float scale = scale_of(m), inverse = inverse_of(scale);
    if (threadIdx.x == 0u) scales[(uint64_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    const uint32_t pitch = pitch_of(columns);
    const bool last = (blockIdx.x + 1u) * kBlock > columns;           // of the columns, and partial
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + i * 16u + rt;
        if (r < rows && c < pitch) {
            *reinterpret_cast<uint2 *>(codes + (uint64_t)r * pitch + c) =
                last ? inside<kVector>(x8[i].codes(scale, inverse), c, columns) : x8[i].codes(scale, inverse);
        }
    }
}

// ------------------------------------------------------------------------------------- transposing
// 128 x 128 codes through shared memory; a table is laid out once, so this is plain.
__global__ void __launch_bounds__(kThreads)
transpose_blocks_kernel(uint8_t *to, float *to_scales, const uint8_t *from, const float *from_scales, uint32_t rows,
                        uint32_t columns) {
    __shared__ uint8_t tile[kBlock][kBlock + 4u];
    pdl_wait();
    const uint32_t r0 = blockIdx.y * kBlock, c0 = blockIdx.x * kBlock;
    const uint32_t from_pitch = pitch_of(columns), to_pitch = pitch_of(rows);
    for (uint32_t i = threadIdx.x; i < kBlock * kBlock; i += kThreads) {
        const uint32_t r = i / kBlock, c = i % kBlock;
        tile[r][c] = r0 + r < rows && c0 + c < columns ? from[(uint64_t)(r0 + r) * from_pitch + c0 + c] : 0u;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBlock * kBlock; i += kThreads) {
        const uint32_t c = i / kBlock, r = i % kBlock;
        if (c0 + c < columns && r0 + r < to_pitch) to[(uint64_t)(c0 + c) * to_pitch + r0 + r] = tile[r][c];
    }
    if (threadIdx.x == 0u) to_scales[(uint64_t)blockIdx.x * gridDim.y + blockIdx.y] = from_scales[(uint64_t)blockIdx.y * gridDim.x + blockIdx.x];
}

// Rows whose length and start allow 16-byte loads.
bool vector_rows(const void *x, uint32_t columns) { return aligned16(x) && columns % 8u == 0u; }

bool arguments_ok(const void *codes, const void *scales, const void *x, uint32_t rows, uint32_t columns, int type) {
    return codes && scales && x && aligned16(codes) && aligned16(scales) && extent_ok(rows) && extent_ok(columns) &&
           (type == K3_MOE_FP8_BF16 || type == K3_MOE_FP8_F32) &&
           ((uintptr_t)x & (type == K3_MOE_FP8_F32 ? 3u : 1u)) == 0u;
}

bool launch_rows(RowsArgs a, bool f32, bool placed, cudaStream_t stream) {
    a.tasks_per_row = scale_pitch_of(a.columns) / 4u;
    const uint64_t tasks = (uint64_t)a.rows * a.tasks_per_row;
    if (tasks > 0xffffffffull) return false;
    const dim3 grid((uint32_t)((tasks + kThreads / 16u - 1u) / (kThreads / 16u)));
    const bool v = vector_rows(a.x, a.columns);
    if (placed) {
        return launch_chained(v ? quantize_rows_kernel<false, true, true> : quantize_rows_kernel<false, false, true>, grid,
                              kThreads, 0, stream, a);
    }
    return launch_chained(f32 ? (v ? quantize_rows_kernel<true, true, false> : quantize_rows_kernel<true, false, false>)
                              : (v ? quantize_rows_kernel<false, true, false> : quantize_rows_kernel<false, false, false>),
                          grid, kThreads, 0, stream, a);
}

}  // namespace

bool k3::fp8::quantize_placed(void *codes, void *scales, const void *x, uint32_t rows, uint32_t columns,
                              const Placement &placement, void *zero_row, uint32_t zero_bytes, cudaStream_t stream) {
    RowsArgs a{};
    a.codes = (uint8_t *)codes;
    a.scales = (float *)scales;
    a.x = x;
    a.rows = rows;
    a.columns = columns;
    a.at = placement;
    a.zero_row = (uint4 *)zero_row;
    a.zero_units = zero_bytes / 16u;
    return launch_rows(a, false, true, stream);
}

extern "C" bool k3_moe_fp8_quantize_rows(void *codes, void *scales, const void *x, uint32_t rows, uint32_t columns,
                                         int x_type, void *stream) {
    if (!arguments_ok(codes, scales, x, rows, columns, x_type)) return false;
    RowsArgs a{};
    a.codes = (uint8_t *)codes;
    a.scales = (float *)scales;
    a.x = x;
    a.rows = rows;
    a.columns = columns;
    return launch_rows(a, x_type == K3_MOE_FP8_F32, false, (cudaStream_t)stream);
}

extern "C" bool k3_moe_fp8_quantize_columns(void *codes, void *scales, const void *x, uint32_t rows, uint32_t columns,
                                            int x_type, void *stream) {
    if (!arguments_ok(codes, scales, x, rows, columns, x_type) || blocks_of(rows) > 65535u) return false;
    const dim3 grid((columns + kTileColumns - 1u) / kTileColumns, blocks_of(rows));
    const bool f32 = x_type == K3_MOE_FP8_F32, v = vector_rows(x, columns);
    return launch_chained(f32 ? (v ? quantize_columns_kernel<true, true> : quantize_columns_kernel<true, false>)
                              : (v ? quantize_columns_kernel<false, true> : quantize_columns_kernel<false, false>),
                          grid, kThreads, 0, (cudaStream_t)stream, (uint8_t *)codes, (float *)scales, x, rows, columns);
}

extern "C" bool k3_moe_fp8_quantize_blocks(void *codes, void *scales, const void *x, uint32_t rows, uint32_t columns,
                                           int x_type, void *stream) {
    if (!arguments_ok(codes, scales, x, rows, columns, x_type) || blocks_of(rows) > 65535u) return false;
    const dim3 grid(blocks_of(columns), blocks_of(rows));
    const bool f32 = x_type == K3_MOE_FP8_F32, v = vector_rows(x, columns);
    return launch_chained(f32 ? (v ? quantize_blocks_kernel<true, true> : quantize_blocks_kernel<true, false>)
                              : (v ? quantize_blocks_kernel<false, true> : quantize_blocks_kernel<false, false>),
                          grid, kThreads, 0, (cudaStream_t)stream, (uint8_t *)codes, (float *)scales, x, rows, columns);
}

extern "C" bool k3_moe_fp8_transpose_blocks(void *codes_out, void *scales_out, const void *codes, const void *scales,
                                            uint32_t rows, uint32_t columns, void *stream) {
    if (!codes_out || !scales_out || !codes || !scales || codes_out == codes || !aligned16(codes_out) || !aligned16(codes) ||
        (((uintptr_t)scales_out | (uintptr_t)scales) & 3u) != 0u || !extent_ok(rows) || !extent_ok(columns) || blocks_of(rows) > 65535u) {
        return false;
    }
    return launch_chained(transpose_blocks_kernel, dim3(blocks_of(columns), blocks_of(rows)), kThreads, 0, (cudaStream_t)stream,
                          (uint8_t *)codes_out, (float *)scales_out, (const uint8_t *)codes, (const float *)scales, rows,
                          columns);
}
