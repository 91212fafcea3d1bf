// What the products' large tiles share: their order, and loads from memory to LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vdttfs {

// XCD-aware tile order: workgroups are handed to the eight XCDs in turn, so
// every XCD gets a contiguous run of tiles; a run goes through bands of kBand
// row tiles, column by column, so that the tiles in flight on an XCD share
// their rows and channels in its L2.
constexpr int kXcds = 8, kBand = 8;
__device__ __forceinline__ bool tile_of(int b, int blocks, int tiles_m, int tiles_n, int* tm, int* tn) {
    const int per = blocks / kXcds, rest = blocks % kXcds, x = b % kXcds;
    if (b / kXcds >= per + (x < rest ? 1 : 0)) return false;  // past the last tile
    b = x * per + (x < rest ? x : rest) + b / kXcds;
    const int band = b / (kBand * tiles_n), in = b % (kBand * tiles_n);
    const int left = tiles_m - band * kBand;
    const int h = left < kBand ? left : kBand;
    *tm = band * kBand + in % h;
    *tn = in / h;
    return true;
}

typedef const __attribute__((address_space(1))) void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

// 16 (4) bytes a lane from p + lane_at + at to 1024 (256) bytes of LDS, in the order
// of the lanes; lane_at + at is below 2^31 - 16.
__device__ __forceinline__ void to_lds16(const void* p, unsigned lane_at, int at, void* lds) {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, 0x7fffffff, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)lds, 16, lane_at, at, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void* p, unsigned lane_at, int at, void* lds) {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, 0x7fffffff, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)lds, 4, lane_at, at, 0, 0);
}

// Waits until at most N of the wave's loads are outstanding (LDS writes: none).
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 0 << 8);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Workgroups of a launch: fewer than 2^32 threads.
constexpr int64_t max_blocks(int threads) { return ((int64_t)1 << 32) / threads - 1; }

}  // namespace vdttfs
