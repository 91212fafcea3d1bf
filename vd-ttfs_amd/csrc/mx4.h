// Microscaled rows in 4 bits: blocks of 32 neighbours with a power of two as
// their scale and elements of the type e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6).
#pragma once

#include "quant.h"

namespace vdttfs {

constexpr int kMxBlock = 32, kMxNan = 255;  // a scale that makes its block NaN

// The scale's byte, X + 127 with X = floor(log2 a) - 2 within [-127, 127], from
// the bits of a block's largest magnitude a: the largest element is then in
// [4, 8), of which what is past 6 becomes 6.  0 and subnormals have X = -127;
// an infinity or a NaN, whose bits are above all others, makes the block NaN.
__device__ __forceinline__ int mx4_scale(uint32_t a) {
    const int e = (int)(a >> 23);
    return e == 255 ? kMxNan : e > 2 ? e - 2 : 0;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest of the four lanes that share a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);  // lane ^ 1
    v = v > a ? v : a;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);  // lane ^ 2
    return v > b ? v : b;
}

// Eight elements' codes, the first in the lowest bits.  x * 2^-X is exact above
// the subnormals (below, it rounds to 0 as the element does), so the conversion's
// rounding, to nearest and half to even and no further than 6, is the only one.
__device__ __forceinline__ uint32_t mx4_codes8(const float (&x)[8], int scale) {
    const float r = __uint_as_float((uint32_t)(254 - scale) << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * r, x[1] * r, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * r, x[3] * r, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * r, x[5] * r, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * r, x[7] * r, 1.0f, 3);
    return scale == kMxNan ? 0 : w;
}

typedef v4u v4u_any __attribute__((aligned(1)));
// 16 bytes to any address, past the caches: what is written here is read by another
// launch, and large outputs push out what this one still reads (16384 x 4096 normed
// 99.5 us with ordinary stores, 96.3 so; 16384 x 8 rows of 2048 to their experts and
// back 240 and 218; each call by itself, not a chain whose rows the caches would hold).
__device__ __forceinline__ void put16(void* p, v4u v) { __builtin_nontemporal_store(v, static_cast<v4u_any*>(p)); }
// Eight neighbouring values to a row of a float type; all there.
__device__ __forceinline__ void put8(void* p, int64_t at, int elem, const float (&f)[8]) {
    if (elem == VDTTFS_ELEM_F32) {
        float* to = static_cast<float*>(p) + at;
        put16(to, v4u{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
        put16(to + 4, v4u{__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])});
        return;
    }
    uint16_t* to = static_cast<uint16_t*>(p) + at;
    if (elem == VDTTFS_ELEM_BF16)
        put16(to, v4u{pack2(f[0], f[1], true), pack2(f[2], f[3], true), pack2(f[4], f[5], true),
                      pack2(f[6], f[7], true)});
    else
        put16(to, v4u{pack2(f[0], f[1], false), pack2(f[2], f[3], false), pack2(f[4], f[5], false),
                      pack2(f[6], f[7], false)});
}

struct __attribute__((packed, aligned(1))) AnyUint {
    uint32_t v;
};
// Codes of columns c..c+7 of a row that ends at `cols` (its last byte's upper
// half is 0 where they are odd), by the lane that has them; the block's first
// lane stores its scale too.
__device__ __forceinline__ void mx4_store8(uint8_t* q, uint8_t* s, int c, int cols, uint32_t w, int scale) {
    if (c >= cols) return;
    if ((c & (kMxBlock - 1)) == 0) s[c / kMxBlock] = (uint8_t)scale;
    if (cols - c >= 8) {
        reinterpret_cast<AnyUint*>(q + c / 2)->v = w;
        return;
    }
    const int left = cols - c;  // elements past the end are 0: so are their codes, but for a sign
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (2 * i < left) q[c / 2 + i] = (uint8_t)(w >> (8 * i) & (2 * i + 1 < left ? 255 : 15));
}

}  // namespace vdttfs
