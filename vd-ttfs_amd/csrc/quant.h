// Quantisation of values to 8-bit codes, shared by the kernels that do it.
#pragma once

#include "elem.h"
#include "wave.h"

namespace vdttfs {

// max of two values >= 0 or NaN; a NaN wins.
__device__ __forceinline__ float nan_max(float a, float b) { return (a >= b || a != a) ? a : b; }

__device__ __forceinline__ float scale_of(float amax) {
    return amax < __builtin_inff() ? amax / 127.0f : __builtin_nanf("");
}

__device__ __forceinline__ float wave_nan_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = nan_max(v, __shfl_xor(v, off, 64));
    return v;
}

// The code of x under scale s (s > 0): the IEEE quotient rounded half to even.
__device__ __forceinline__ int exact_code(float x, float s) {
    return (int)fminf(fmaxf(rintf(x / s), -127.0f), 127.0f);
}

// A row's scale, made ready for its codes.
struct Coder {
    float s, r;
    bool none, exact;  // codes are 0; the reciprocal does not serve
};
__device__ __forceinline__ Coder coder_of(float s) {
    // below 2^-125 the reciprocal or its products leave the normal range
    return Coder{s, 1.0f / s, !(s > 0.0f), s < 2.35e-38f};
}

// Eight codes by the reciprocal; true where one of them may be wrong.  x * r is
// within 127.1 * 2^-23 of the quotient and the 32-bit quotient within
// 127.1 * 2^-24, so both round alike unless the product lies within 2.3e-5 of
// a half.
__device__ __forceinline__ bool codes8_fast(const float (&x)[8], const Coder& c, int (&k)[8]) {
    bool close = c.exact;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = x[i] * c.r, q = rintf(t);
        close |= fabsf(t - q) > 0.5f - 3e-5f;
        k[i] = c.none ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);
    }
    return close && !c.none;
}
// ... by division: a wave that holds such a value.
__device__ __forceinline__ void codes8_exact(const float (&x)[8], const Coder& c, int (&k)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = c.none ? 0 : exact_code(x[i], c.s);
}
__device__ __forceinline__ void codes8(const float (&x)[8], const Coder& c, int (&k)[8]) {
    if (__any(codes8_fast(x, c, k))) codes8_exact(x, c, k);
}

// The code of a spike time (vdttfs_quant_rows); levels = min(T, 127).
__device__ __forceinline__ int time_code(float t, float tfs, int T, int levels) {
    const int b = arrival_bin(t, tfs, T);
    return b < 0 ? 0 : (int)rintf((float)((T - b) * levels) / (float)T);
}

// Eight neighbouring values of a row as they lie in memory.  Loading and
// unpacking are apart so that a thread's loads can all be in flight: inside one
// branch the compiler waits for each before the next.
template <int ELEM>
struct Raw8 {
    static constexpr bool kWide = ELEM == VDTTFS_ELEM_F32 || ELEM == VDTTFS_ELEM_TIMES;
    uint4 v[kWide ? 2 : 1];
};
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(1))) AnyUint4 {
    v4u v;
};
// What is not there: 0, or no spike.
template <int ELEM>
__device__ __forceinline__ Raw8<ELEM> nothing8() {
    const uint32_t w = ELEM == VDTTFS_ELEM_TIMES ? __float_as_uint(kInfTime) : 0;
    Raw8<ELEM> r;
#pragma unroll
    for (auto& v : r.v) v = make_uint4(w, w, w, w);
    return r;
}
// The eight values from element `at` of x on, all of them there; rows need no
// more than their type's alignment (gfx950 loads 16 bytes from any address).
template <int ELEM>
__device__ __forceinline__ Raw8<ELEM> raw8(const void* x, int64_t at) {
    Raw8<ELEM> r;
    const AnyUint4* p =
        reinterpret_cast<const AnyUint4*>(static_cast<const char*>(x) + at * (Raw8<ELEM>::kWide ? 4 : 2));
    const v4u a = p[0].v;
    r.v[0] = make_uint4(a[0], a[1], a[2], a[3]);
    if constexpr (Raw8<ELEM>::kWide) {
        const v4u b = p[1].v;
        r.v[1] = make_uint4(b[0], b[1], b[2], b[3]);
    }
    return r;
}
template <int ELEM>
__device__ __forceinline__ void unpack8(const Raw8<ELEM>& r, float (&f)[8]) {
    if constexpr (Raw8<ELEM>::kWide) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[4 * i] = __uint_as_float(r.v[i].x), f[4 * i + 1] = __uint_as_float(r.v[i].y);
            f[4 * i + 2] = __uint_as_float(r.v[i].z), f[4 * i + 3] = __uint_as_float(r.v[i].w);
        }
    } else {
        const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            f[i] = ELEM == VDTTFS_ELEM_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
        }
    }
}
// The run from column c of a row of `cols`, which ends inside it.  (Columns are
// compared by differences: c + 8 can pass 2^31.)
template <int ELEM>
__device__ __forceinline__ void tail8(const void* x, int64_t row, int c, int cols, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < cols - c) f[i] = load_elem<ELEM>(x, row + c + i);
}
template <int ELEM>
__device__ __forceinline__ void load8(const void* x, int64_t row, int c, int cols, float (&f)[8]) {
    unpack8<ELEM>(cols - c >= 8 ? raw8<ELEM>(x, row + c) : nothing8<ELEM>(), f);
    if (c < cols && cols - c < 8) tail8<ELEM>(x, row, c, cols, f);
}

__device__ __forceinline__ uint2 pack8(const int (&k)[8]) {
    uint2 w;
    w.x = (k[0] & 255) | (k[1] & 255) << 8 | (k[2] & 255) << 16 | (uint32_t)k[3] << 24;
    w.y = (k[4] & 255) | (k[5] & 255) << 8 | (k[6] & 255) << 16 | (uint32_t)k[7] << 24;
    return w;
}

}  // namespace vdttfs
