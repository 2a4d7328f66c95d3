// kv_terms.h — f32 operands as sums of 16-bit terms, for the matrix products of
// the paged cache's attention on 16-bit caches (kv_attention.hip, kv_prompt.hip). K and
// V are exact in their type; q and the probabilities are f32, which N terms of that type
// carry: f16 two (22 bits), bf16 three (24 bits).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "fmt.h"

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
#pragma unroll
        for (int j = 0; j < 8; j++) t[0][j] = (_Float16)x[j];
#pragma unroll
        for (int j = 0; j < 8; j++) t[1][j] = (_Float16)fmaf(-1.0f, (float)t[0][j], x[j]);
    }
    // the exponent that brings a row's maximum to [2^13, 2^14), near the top of f16's
    // range: the second term of what matters is then no subnormal
    static __device__ __forceinline__ int shift(float mx) {
        int e = 14;
        if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &e);
        return 14 - e;
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
    static __device__ __forceinline__ void split(const float (&x)[8], v8 (&t)[3]) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            t[0][j] = (__bf16)x[j];
            const float r = x[j] - (float)t[0][j];
            t[1][j] = (__bf16)r;
            t[2][j] = (__bf16)(r - (float)t[1][j]);
        }
    }
    static __device__ __forceinline__ int shift(float) { return 0; }
};
// not finite, of two packed elements: which
template <typename T> __device__ __forceinline__ bool kv_odd_lo(uint32_t x) { return (x & KvTerms<T>::EXP) == KvTerms<T>::EXP; }
template <typename T> __device__ __forceinline__ bool kv_odd_hi(uint32_t x) { return kv_odd_lo<T>(x >> 16); }
