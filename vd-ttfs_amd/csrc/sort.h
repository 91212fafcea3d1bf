// The sort of few pairs by expert, by one workgroup of 1024 threads.
#pragma once
#include "common.h"
#include "wave.h"

namespace vdttfs {

constexpr int kMaxExperts = 1024;

// Sum of v over the threads before this one (1024 threads); total: over all.
__device__ __forceinline__ int block_excl_scan(int v, int* lds, int* total) {
    const int incl = wave_incl_scan(v);
    const int wave = threadIdx.x >> 6;
    if (lane_id() == 63) lds[wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 16; ++i) {
        const int s = lds[i];
        if (i < wave) before += s;
        all += s;
    }
    __syncthreads();
    *total = all;
    return before + incl - v;
}

struct SortOne {
    const int32_t* idx;
    int pairs, E, top_k, bm;
    int4* tiles;
    int* n_tiles;
    int* pair;
    int* row;
};
// All of the sort, for up to kSortOne pairs: some 5 us in place of three launches
// of 10.
constexpr int kSortOne = 8192;
__device__ __forceinline__ void sort_one(const SortOne& a) {
    __shared__ int lds[16];
    __shared__ int at[kMaxExperts];
    int e[kSortOne / 1024];
#pragma unroll
    for (int i = 0; i < kSortOne / 1024; ++i) {
        const int q = i * 1024 + threadIdx.x;
        e[i] = q < a.pairs ? a.idx[q] : -1;
    }
    at[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortOne / 1024; ++i)
        if (e[i] >= 0 && e[i] < a.E) atomicAdd(&at[e[i]], 1);
    __syncthreads();
    const int n = at[threadIdx.x], t = (n + a.bm - 1) / a.bm;
    int all, t_all;
    const int start = block_excl_scan(n, lds, &all);
    const int t0 = block_excl_scan(t, lds, &t_all);
    for (int i = 0; i < t; ++i) a.tiles[t0 + i] = make_int4(threadIdx.x, start + i * a.bm, start + n, 0);
    if (threadIdx.x == 0) *a.n_tiles = t_all;
    at[threadIdx.x] = start;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortOne / 1024; ++i)
        if (e[i] >= 0 && e[i] < a.E) {
            const int q = i * 1024 + threadIdx.x, to = atomicAdd(&at[e[i]], 1);
            a.pair[to] = q;
            a.row[to] = q / a.top_k;
        }
}

}  // namespace vdttfs
