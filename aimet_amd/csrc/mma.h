// Matrix-core helpers shared by the packed linear layer and the attention over an 8-bit cache: fragments of the
// 16 x 16 x 32 matrix instruction (wave64), with float32 operands written as sums of bfloat16 values.
//
// Fragment layout (lane = 16 * c + i): A holds row i, B holds column i, both at the eight contraction indexes 8 c + e;
// the result holds rows 4 c + r (r = 0..3) of column i.  Both operands count the contraction the same way, so any
// assignment of data to contraction indexes is right as long as A and B agree on it.
#pragma once

#include "ahq_device.h"

namespace ahq {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// High halves of two float32 bit patterns as one pair of bfloat16 (truncation; exact where the low halves are zero).
__device__ __forceinline__ uint32_t pack_high_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(f32_to_bits(hi), f32_to_bits(lo), 0x07060302u);
}

// Eight float32 values as a sum of N bfloat16 fragments: each part is the value with its low 16 bits cut off, the next
// one what is left (both steps exact), the last one rounded.  N = 2 keeps 16 bits of each value, N = 3 all 24.
template <int N>
__device__ __forceinline__ void split_bf16(const float* v, bf16x8* out) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
    for (int p = 0; p < N; ++p) {
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (p + 1 == N) {
                bf16x2 r = {(__bf16)rest[2 * e], (__bf16)rest[2 * e + 1]};
                w[e] = __builtin_bit_cast(uint32_t, r);
            } else {
                w[e] = pack_high_halves(rest[2 * e], rest[2 * e + 1]);
                rest[2 * e] -= bits_to_f32(f32_to_bits(rest[2 * e]) & 0xffff0000u);
                rest[2 * e + 1] -= bits_to_f32(f32_to_bits(rest[2 * e + 1]) & 0xffff0000u);
            }
        }
        out[p] = __builtin_bit_cast(bf16x8, w);
    }
}

}  // namespace ahq
