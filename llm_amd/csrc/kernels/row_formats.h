// row_formats.h -- f32 values -> the formats a KV-cache row can have (f16, bf16, q8_0, q4_0): the one arithmetic behind CPY, SET_ROWS,
// the KV store and the normalised / rotated store (elementwise.hip, qk_norm_rope.hip), so every path writes the same bits.
#pragma once
#include "common.h"

template <class TS, class TD> static __device__ __forceinline__ TD cvt(TS v);
template <> __device__ __forceinline__ float  cvt<float, float>(float v) { return v; }
template <> __device__ __forceinline__ __half cvt<float, __half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __half cvt<__half, __half>(__half v) { return v; }
template <> __device__ __forceinline__ float  cvt<__half, float>(__half v) { return __half2float(v); }
// bf16 as the reference rounds it (ggml_compute_fp32_to_bf16, ggml-impl.h:453-466): nearest even on the bits, NaNs made quiet
struct bf16_bits { uint16_t bits; };
template <> __device__ __forceinline__ bf16_bits cvt<float, bf16_bits>(float v) {
    const uint32_t i = __float_as_uint(v);
    bf16_bits h;
    if ((i & 0x7fffffffu) > 0x7f800000u) h.bits = (uint16_t)((i >> 16) | 64);
    else                                 h.bits = (uint16_t)((i + (0x7fffu + ((i >> 16) & 1u))) >> 16);
    return h;
}

// 32 f32 -> one q8_0 block (quantize_row_q8_0_ref, ggml-quants.c:188-211): the one arithmetic behind CPY, SET_ROWS and the KV store
static __device__ __forceinline__ void quant_block_q8_0(const float * xs, uint8_t * blk) {
    float v[32], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; j++) { v[j] = xs[j]; amax = fmaxf(amax, fabsf(v[j])); }
    const float dd = __fdiv_rn(amax, 127.0f);
    const float id = dd != 0.0f ? __fdiv_rn(1.0f, dd) : 0.0f;
    *(uint16_t *)blk = __half_as_ushort(__float2half_rn(dd));
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const float r = roundf(__fmul_rn(v[j], id));
        ((int8_t *)blk)[2 + j] = fabsf(r) < 2147483648.0f ? (int8_t)(int)r : 0;
    }
}

// 32 f32 -> one q4_0 block (quantize_row_q4_0_ref, ggml-quants.c:25-60): d = (the value of largest magnitude) / -8, q = min(15, trunc(x / d
// + 8.5)), value j in the low nibble of byte j, value j + 16 in its high nibble
static __device__ __forceinline__ void quant_block_q4_0(const float * xs, uint8_t * blk) {
    float v[32], amax = 0.0f, mx = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; j++) { v[j] = xs[j]; if (amax < fabsf(v[j])) { amax = fabsf(v[j]); mx = v[j]; } }
    const float dd = __fmul_rn(mx, -0.125f);      // max / -8, exact; an all-zero block stores d = -0 as the reference does (0x8000)
    const float id = dd != 0.0f ? __fdiv_rn(1.0f, dd) : 0.0f;
    *(uint16_t *)blk = mx == 0.0f ? (uint16_t)0x8000 : __half_as_ushort(__float2half_rn(dd));   // (+0 / -8 = -0: spelt out, the product's sign did not survive the compiler)
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const float x0 = __fmul_rn(v[j], id), x1 = __fmul_rn(v[16 + j], id);
        // (int8_t)(x + 8.5f): the sum lies in [0.5, 16.5] for finite input; NaN / inf input converts to 0 here (undefined in C)
        const float s0 = __fadd_rn(x0, 8.5f), s1 = __fadd_rn(x1, 8.5f);
        const int q0 = fabsf(s0) < 2147483648.0f ? (int)(int8_t)(int)s0 : 0, q1 = fabsf(s1) < 2147483648.0f ? (int)(int8_t)(int)s1 : 0;
        const uint8_t u0 = (uint8_t)q0 < 15 ? (uint8_t)q0 : 15, u1 = (uint8_t)q1 < 15 ? (uint8_t)q1 : 15;
        blk[2 + j] = (uint8_t)(u0 | (u1 << 4));
    }
}
template <int TYPE> static __device__ __forceinline__ void quant_block(const float * xs, uint8_t * blk) {
    if (TYPE == MI355_TYPE_Q8_0) quant_block_q8_0(xs, blk); else quant_block_q4_0(xs, blk);
}
template <int TYPE> struct QBlk { static constexpr int bytes = TYPE == MI355_TYPE_Q8_0 ? 34 : 18; };
