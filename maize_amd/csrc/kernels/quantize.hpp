// maize_quantize_{bf16,f16,f32}_{rows,blocks}: the operands of block-scaled products.
//
// Every block of 1 x 128 (rows) or 128 x 128 (blocks) elements becomes E4M3 values and one fp32 scale:
//   m = max(largest |x|, 2^-100),   scale = m / 448,   q = RNE_e4m3(x * (448 / m))
// 448 is the format's largest value, so that nothing overflows; the floor keeps the reciprocal of an all-zero block finite (its
// values are zero, whatever the scale).  NaN elements become NaN and do not count for m; an infinite element makes the scale
// infinite, so that every product with its block is NaN.
//
// Bound by HBM: 3 bytes an element (16-bit input), some eight operations; 8192 x 4096 bf16 in 20.7 us, 4.9 TB/s (what a large copy reaches), fp32 in 29.9 us.  16 neighbouring lanes hold the 128 elements of a row of a
// block, eight each (one 16-byte load of 16-bit elements); their largest is found by exchanges between lanes.  An 1 x 128 block is
// held by 16 lanes and a workgroup takes 16 rows of one column of blocks, so that its scales lie in one run; a 128 x 128 block is
// held in the registers of one workgroup, eight rows a thread.  Nothing is read twice.
#pragma once
#include "common.hpp"

namespace maize {

struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    uint32_t rows, cols, ldx, ldq, ld_scale, batch;
    uint64_t stride_x, stride_q, stride_scale;
};
static_assert(sizeof(QuantArgs) == 72, "kernel parameter block layout");

namespace quant {

constexpr float TOP = 448.0f;
enum { BF16 = 0, F16 = 1, F32 = 2 };

template <int T>
__device__ __forceinline__ float one(const void* x, uint64_t at) {
    if constexpr (T == F32) return ((const float*)x)[at];
    else if constexpr (T == F16) return f16_bits_to_f32(((const uint16_t*)x)[at]);
    else return bf16_bits_to_f32(((const uint16_t*)x)[at]);
}
// Eight elements from `at` on, of which `count` exist (zeros behind); any alignment.
template <int T>
__device__ __forceinline__ void load8(const void* x, uint64_t at, uint32_t count, float (&v)[8]) {
    if (count >= 8u) {
        if constexpr (T == F32) {
            __builtin_memcpy(v, (const float*)x + at, 32);
        } else {
            uint32_t w[4];
            __builtin_memcpy(w, (const uint16_t*)x + at, 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                v[e] = T == F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
            }
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) v[e] = e < count ? one<T>(x, at + e) : 0.0f;
    }
}
__device__ __forceinline__ float largest8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = __builtin_fmaxf(m, __builtin_fabsf(v[e]));
    return m;
}
// The largest over 16 neighbouring lanes.
__device__ __forceinline__ float largest16(float m) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d, 64));
    return m;
}
__device__ __forceinline__ void store8(uint8_t* q, uint64_t at, uint32_t count, const float (&v)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, 0, false);
        w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, x, true);
    }
    if (count >= 8u) {
        __builtin_memcpy(q + at, w, 8);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e)
            if (e < count) q[at + e] = (uint8_t)(w[e >> 2] >> (8u * (e & 3u)));
    }
}
__device__ __forceinline__ uint32_t inside(uint32_t from, uint32_t end) { return from < end ? end - from : 0u; }

struct Place { uint32_t z, row, block; };       // batch member, first row, column block
template <uint32_t ROWS>
__device__ __forceinline__ Place place(const QuantArgs& p) {
    const uint32_t across = (p.cols + 127u) / 128u, down = (p.rows + ROWS - 1u) / ROWS, r = blockIdx.x / across;
    return Place{r / down, r % down * ROWS, blockIdx.x % across};
}

// grid: batch x ceil(rows / 16) x column blocks, the last one fastest (neighbouring workgroups read neighbouring columns)
template <int T>
__device__ __forceinline__ void rows_body(const QuantArgs& p) {
    const Place b = place<16>(p);
    const uint32_t tid = threadIdx.x, row = b.row + tid / 16u, col = b.block * 128u + tid % 16u * 8u;
    const uint32_t count = row < p.rows ? inside(col, p.cols) : 0u;
    const uint64_t z = b.z;
    float v[8];
    load8<T>(p.x, z * p.stride_x + (uint64_t)row * p.ldx + col, count, v);
    const float m = __builtin_fmaxf(largest16(largest8(v)), 0x1p-100f);
    if (row < p.rows && tid % 16u == 0u) p.scale[z * p.stride_scale + (uint64_t)b.block * p.ld_scale + row] = m / TOP;
    store8(p.q, z * p.stride_q + (uint64_t)row * p.ldq + col, count, v, TOP / m);
}

// grid: batch x row blocks x column blocks
template <int T>
__device__ __forceinline__ void blocks_body(const QuantArgs& p) {
    __shared__ float most[4];
    const Place b = place<128>(p);
    const uint32_t tid = threadIdx.x, row = b.row + tid / 16u, col = b.block * 128u + tid % 16u * 8u;
    const uint32_t count = inside(col, p.cols);
    const uint64_t z = b.z;
    float v[8][8], m = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) load8<T>(p.x, z * p.stride_x + (uint64_t)(row + 16u * i) * p.ldx + col, row + 16u * i < p.rows ? count : 0u, v[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __builtin_fmaxf(m, largest8(v[i]));
    m = largest16(m);
    m = __builtin_fmaxf(m, __shfl_xor(m, 16, 64));
    m = __builtin_fmaxf(m, __shfl_xor(m, 32, 64));
    if (tid % 64u == 0u) most[tid / 64u] = m;
    __syncthreads();
    m = __builtin_fmaxf(__builtin_fmaxf(most[0], most[1]), __builtin_fmaxf(most[2], most[3]));
    m = __builtin_fmaxf(m, 0x1p-100f);
    if (tid == 0u) p.scale[z * p.stride_scale + (uint64_t)(b.row / 128u) * p.ld_scale + b.block] = m / TOP;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) store8(p.q, z * p.stride_q + (uint64_t)(row + 16u * i) * p.ldq + col, row + 16u * i < p.rows ? count : 0u, v[i], TOP / m);
}

}  // namespace quant

#define MAIZE_QUANTIZE(tag, T) \
    extern "C" __global__ __launch_bounds__(256) void maize_quantize_##tag##_rows(QuantArgs p) { quant::rows_body<quant::T>(p); } \
    extern "C" __global__ __launch_bounds__(256) void maize_quantize_##tag##_blocks(QuantArgs p) { quant::blocks_body<quant::T>(p); }
MAIZE_QUANTIZE(bf16, BF16)
MAIZE_QUANTIZE(f16, F16)
MAIZE_QUANTIZE(f32, F32)
#undef MAIZE_QUANTIZE

}  // namespace maize
