// 32x32x16 matrix products of 16-bit operands with fp32 accumulators, and packing of their results.
#pragma once

#include "common.hpp"

namespace peco {

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT> struct Mfma;
template <> struct Mfma<kBF16> {
    static __device__ __forceinline__ f32x16 run(u16x8 a, u16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    // Two fp32 -> packed pair with round-to-nearest-even (v_cvt_pk_bf16_f32).
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, b2));
    }
    // acc + lo(p) + hi(p) of a packed pair (v_dot2_f32_bf16 against (1, 1)).
    static __device__ __forceinline__ float sum2(uint32_t p, float acc) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, p), __builtin_bit_cast(b2, 0x3f803f80u), acc,
                                               false);
    }
};
template <> struct Mfma<kF16> {
    static __device__ __forceinline__ f32x16 run(u16x8 a, u16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, h2));
    }
    static __device__ __forceinline__ float sum2(uint32_t p, float acc) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, p), __builtin_bit_cast(h2, 0x3c003c00u), acc, false);
    }
};

}  // namespace peco
