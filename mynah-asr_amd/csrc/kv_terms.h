// kv_terms.h — f32 operands as sums of 16-bit terms, for the matrix products of
// the paged cache's attention on 16-bit caches (kv_attention.hip, kv_prompt.hip). K and
// V are exact in their type; q and the probabilities are f32, which N terms of that type
// carry: f16 two (22 bits), bf16 three (24 bits).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "product.h"

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

template <typename T> struct KvTerms;
template <> struct KvTerms<_Float16> {
    typedef half8 v8;
    static constexpr int N = 2;
    static constexpr uint32_t EXP = 0x7c00;   // the exponent bits: all set, not finite
    static __device__ __forceinline__ f16v mfma32(v8 a, v8 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 mfma16(v8 a, v8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split(const float (&x)[8], v8 (&t)[2]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            h[j] = __builtin_bit_cast(uint32_t, half2v{(_Float16)x[2 * j], (_Float16)x[2 * j + 1]});
            l[j] = lo_pair(h[j], x[2 * j], x[2 * j + 1]);
        }
        t[0] = __builtin_bit_cast(v8, uint4{h[0], h[1], h[2], h[3]});
        t[1] = __builtin_bit_cast(v8, uint4{l[0], l[1], l[2], l[3]});
    }
    // the exponent that brings a row's maximum to [2^13, 2^14), near the top of f16's
    // range: the second term of what matters is then no subnormal. At most 120, so that its
    // reciprocal is no subnormal either: smaller rows have scores of 0 all the same.
    static __device__ __forceinline__ int shift(float mx) {
        int e = 14;
        if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &e);
        return min(14 - e, 120);
    }
};
template <> struct KvTerms<__bf16> {
    typedef bf8 v8;
    static constexpr int N = 3;
    static constexpr uint32_t EXP = 0x7f80;
    static __device__ __forceinline__ f16v mfma32(v8 a, v8 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f4 mfma16(v8 a, v8 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // x0, x1 rounded to a pair of bf16, and what that leaves of them (the pair kept from the compiler's
    // sight: from conversions and their inverses it makes five instructions for each three)
    static __device__ __forceinline__ uint32_t pair(float &x0, float &x1) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        uint32_t h = __builtin_bit_cast(uint32_t, b2{(__bf16)x0, (__bf16)x1});
        asm("" : "+v"(h));
        x0 -= __uint_as_float(h << 16);
        x1 -= __uint_as_float(h & 0xffff0000u);
        return h;
    }
    static __device__ __forceinline__ void split(const float (&x)[8], v8 (&t)[3]) {
        uint32_t h[3][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x0 = x[2 * j], x1 = x[2 * j + 1];
#pragma unroll
            for (int k = 0; k < 3; k++) h[k][j] = pair(x0, x1);
        }
#pragma unroll
        for (int k = 0; k < 3; k++) t[k] = __builtin_bit_cast(v8, uint4{h[k][0], h[k][1], h[k][2], h[k][3]});
    }
    static __device__ __forceinline__ int shift(float) { return 0; }
};
// not finite, of two packed elements: which
template <typename T> __device__ __forceinline__ bool kv_odd_lo(uint32_t x) { return (x & KvTerms<T>::EXP) == KvTerms<T>::EXP; }
template <typename T> __device__ __forceinline__ bool kv_odd_hi(uint32_t x) { return kv_odd_lo<T>(x >> 16); }
