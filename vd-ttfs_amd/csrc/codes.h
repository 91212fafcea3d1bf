// Rows of 8-bit codes in memory.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vdttfs {

typedef int v4i __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(1))) Bytes16 {
    v4i v;
};

// Codes k..k+15 of a row of K, those past its end as 0.  The row may have any
// alignment (gfx950 loads 16 bytes from any address); where fewer than 16 are
// left, the row's last 16 are loaded and shifted.
__device__ __forceinline__ v4i load16(const int8_t* row, int k, int K) {
    const int valid = K - k;
    if (valid >= 16) return reinterpret_cast<const Bytes16*>(row + k)->v;
    uint64_t lo = 0, hi = 0;
    if (valid > 0 && K >= 16) {
        const v4i v = reinterpret_cast<const Bytes16*>(row + K - 16)->v;
        lo = (uint64_t)(uint32_t)v[1] << 32 | (uint32_t)v[0];
        hi = (uint64_t)(uint32_t)v[3] << 32 | (uint32_t)v[2];
        const int bits = 8 * (16 - valid);  // 8..120
        if (bits >= 64) {
            lo = hi >> (bits - 64);
            hi = 0;
        } else {
            lo = lo >> bits | hi << (64 - bits);
            hi >>= bits;
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < valid; ++i) {
            const uint64_t b = (uint64_t)(uint8_t)row[k + i] << (8 * (i & 7));
            if (i < 8) lo |= b;
            else hi |= b;
        }
    }
    return v4i{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}

}  // namespace vdttfs
