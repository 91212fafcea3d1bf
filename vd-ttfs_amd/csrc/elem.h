// Element types of the 8-bit heads: loads, stores and activations.
#pragma once

#include <hip/hip_runtime.h>

#include "vdttfs.h"

namespace vdttfs {

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// Both round to nearest even; NaN stays NaN.
__device__ __forceinline__ uint16_t f32_to_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ float f16_to_f32(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ uint16_t f32_to_f16(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two values of a 16-bit type in one word.
__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
    if (bf16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

template <int ELEM>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
    if constexpr (ELEM == VDTTFS_ELEM_BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else if constexpr (ELEM == VDTTFS_ELEM_F16) return f16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void store_elem(void* p, int64_t i, float v, int elem) {
    if (elem == VDTTFS_ELEM_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = elem == VDTTFS_ELEM_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}

// v / (1 + exp(-v)).  The hardware's exp2 takes -v log2(e) in two pieces, so the
// result is right to a few roundings.  Below -60 the 1 is nothing beside the exp,
// and 2^-64 is split off it, so that neither it nor its reciprocal leaves the
// normal range, where the hardware's instructions flush; the last product rounds
// to a subnormal result, and to nothing below -126 (-inf: NaN, as the formula).
// The library's exp and an IEEE division are more instructions: the first product
// of 8192 rows through 8 of 64 gated experts, 2048 -> 1024, took 407 us with them
// and 372 with what serves above -60; values below that cost some 10 us of the
// layer's 745 more.
__device__ __forceinline__ float silu(float v) {
    const bool far = v < -60.0f;
    const float c = __builtin_amdgcn_fmed3f(v, -126.0f, 88.0f);
    constexpr float kHi = 1.44269504088896341f, kLo = 1.925963033500e-8f, kLn2 = 0.693147180559945f;
    const float t = c * -kHi;
    const float r = __builtin_fmaf(c, -kLo, __builtin_fmaf(c, -kHi, -t));
    const float e = __builtin_amdgcn_exp2f(far ? t - 64.0f : t);
    const float d = (far ? 0.0f : 1.0f) + __builtin_fmaf(e, r * kLn2, e);
    return v * __builtin_amdgcn_rcpf(d) * (v < -126.0f ? 0.0f : far ? 0x1p-64f : 1.0f);
}

// The same in every kernel: what is quantised again may not depend on which
// one made it.
__device__ __forceinline__ float apply_act(float v, int act) {
    if (act == VDTTFS_ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (act == VDTTFS_ACT_SILU) return silu(v);
    return v;
}

}  // namespace vdttfs
