// Rows to the order of their experts and back, and the gradients of both.
//
// A pair is (row m, slot j), number m * top_k + j; its place is its rank among
// the pairs with an expert, by expert and then by number.  Rows move as they are;
// sums over slots are in 32 bits, in the order of the slots.
#include "elem.h"
#include "head.h"
#include "quant.h"
#include "sort.h"
#include "wave.h"

namespace vdttfs {
namespace {

constexpr int kPairs = 2048;  // pairs of a workgroup of the sort
constexpr int kWaves = 16;    // of such a workgroup

__device__ __forceinline__ int expert_of(const PlaceArgs& a, int64_t q, int64_t pairs) {
    const int e = q < pairs ? a.idx[q] : -1;
    return e >= 0 && e < a.E ? e : -1;
}

// The lanes with this lane's value of 0 <= e < E (none where e is below 0).
__device__ __forceinline__ uint64_t lanes_like(int e, int bits) {
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
        const bool on = e >> b & 1;
        const uint64_t with = __ballot(on);
        same &= on ? with : ~with;
    }
    return e >= 0 ? same : 0;
}

// Pairs of each workgroup by expert: hist[block][expert].
__global__ __launch_bounds__(1024) void k_place_count(PlaceArgs a, int* __restrict__ hist) {
    __shared__ int h[kMaxExperts];
    const int64_t pairs = a.M * a.top_k, q0 = (int64_t)blockIdx.x * kPairs + threadIdx.x;
    const int e0 = expert_of(a, q0, pairs), e1 = expert_of(a, q0 + 1024, pairs);
    if ((int)threadIdx.x < a.E) h[threadIdx.x] = 0;
    __syncthreads();
    if (e0 >= 0) atomicAdd(&h[e0], 1);
    if (e1 >= 0) atomicAdd(&h[e1], 1);
    __syncthreads();
    if ((int)threadIdx.x < a.E) hist[(int64_t)blockIdx.x * a.E + threadIdx.x] = h[threadIdx.x];
}

// One workgroup: hist[block][expert] becomes the place of the block's first pair
// of the expert.  2^log threads go over the experts, and share the blocks in
// 1024 >> log runs.
__global__ __launch_bounds__(1024) void k_place_scan(PlaceArgs a, int* __restrict__ hist, int blocks, int log) {
    __shared__ int lds[16];
    __shared__ int sums[1024];
    __shared__ int starts[kMaxExperts];
    const int e = threadIdx.x & ((1 << log) - 1), run = threadIdx.x >> log, runs = 1024 >> log;
    const int per = (blocks + runs - 1) / runs;
    const int b0 = run * per < blocks ? run * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
    int n = 0;
    if (e < a.E)
#pragma unroll 4
        for (int b = b0; b < b1; ++b) n += hist[(int64_t)b * a.E + e];
    sums[threadIdx.x] = n;
    __syncthreads();
    int total = 0;
    if (run == 0)
        for (int r = 0; r < runs; ++r) total += sums[(r << log) + e];
    int all;
    const int first = block_excl_scan(total, lds, &all);
    if (run == 0) starts[e] = first;
    if (a.start && run == 0 && e < a.E) a.start[e] = first;
    if (a.start && threadIdx.x == 0) a.start[a.E] = all;
    __syncthreads();
    if (e >= a.E) return;
    int at = starts[e];
    for (int r = 0; r < run; ++r) at += sums[(r << log) + e];
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int64_t i = (int64_t)b * a.E + e;
        const int h = hist[i];
        hist[i] = at;
        at += h;
    }
}

// Each pair's place: a wave has 128 neighbouring pairs, counts them by expert,
// adds what the waves before it have, and ranks 64 at a time among themselves.
__global__ __launch_bounds__(1024) void k_place(PlaceArgs a, const int* __restrict__ hist, int bits) {
    extern __shared__ int at[];  // [kWaves][E]
    const int64_t pairs = a.M * a.top_k;
    const int wave = threadIdx.x >> 6, lane = lane_id();
    const int64_t q0 = (int64_t)blockIdx.x * kPairs + wave * (kPairs / kWaves) + lane;
    int e[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) e[i] = expert_of(a, q0 + 64 * i, pairs);
    for (int i = threadIdx.x; i < kWaves * a.E; i += 1024) at[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (e[i] >= 0) atomicAdd(&at[wave * a.E + e[i]], 1);
    __syncthreads();
    if ((int)threadIdx.x < a.E) {
        int sum = hist[(int64_t)blockIdx.x * a.E + threadIdx.x];
        for (int w = 0; w < kWaves; ++w) {
            const int n = at[w * a.E + threadIdx.x];
            at[w * a.E + threadIdx.x] = sum;
            sum += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t same = lanes_like(e[i], bits);
        const int rank = __popcll(same & lanemask_lt());
        int to = -1;
        if (e[i] >= 0) to = at[wave * a.E + e[i]] + rank;
        wave_sync();  // read by all before the first of them moves it on
        if (e[i] >= 0 && rank == 0) at[wave * a.E + e[i]] = to + __popcll(same);
        wave_sync();
        if (q0 + 64 * i < pairs) a.place[q0 + 64 * i] = to;
    }
}

// A row's bytes to another; both may start anywhere that their type allows.
constexpr int kCopy = 256;
__device__ __forceinline__ void copy_to_slots(void* z, int64_t ld_bytes, const void* x_row, int64_t bytes, int unit,
                                              const int* place, int n, int64_t rows) {
    const char* from = static_cast<const char*>(x_row);
    const int64_t whole = bytes / 16 * 16;
    for (int64_t b = (int64_t)threadIdx.x * 16; b < whole; b += kCopy * 16) {
        const v4u v = reinterpret_cast<const AnyUint4*>(from + b)->v;
        for (int j = 0; j < n; ++j) {
            const int p = place[j];
            if (p >= 0 && p < rows) reinterpret_cast<AnyUint4*>(static_cast<char*>(z) + p * ld_bytes + b)->v = v;
        }
    }
    for (int64_t b = whole + (int64_t)threadIdx.x * unit; b < bytes; b += kCopy * unit)
        for (int j = 0; j < n; ++j) {
            const int p = place[j];
            if (p < 0 || p >= rows) continue;
            char* to = static_cast<char*>(z) + p * ld_bytes + b;
            if (unit == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from + b);
            else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from + b);
        }
}
__global__ __launch_bounds__(kCopy) void k_dispatch_rows(PlaceArgs a, void* __restrict__ z, int64_t ldz,
                                                         const void* __restrict__ x, int64_t ldx, int cols, int unit) {
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x)
        copy_to_slots(z, ldz * unit, static_cast<const char*>(x) + m * ldx * unit, (int64_t)cols * unit, unit,
                      a.place + m * a.top_k, a.top_k, a.M * a.top_k);
}

// A row of floats with its slots.  T threads a row, eight neighbours a thread and
// turn.
__device__ __forceinline__ bool placed(int p, int64_t rows) { return p >= 0 && p < rows; }

template <int ZE>
__global__ __launch_bounds__(256) void k_gather_sum(void* __restrict__ out, int out_elem, int64_t ldo,
                                                    const void* __restrict__ z, int64_t ldz,
                                                    const int32_t* __restrict__ place, const float* __restrict__ wt,
                                                    int64_t M, int top_k, int cols, int log_t) {
    const int T = 1 << log_t, rows = 256 >> log_t, lane = threadIdx.x & (T - 1);
    const int64_t most = M * top_k;
    for (int64_t m = (int64_t)blockIdx.x * rows + (threadIdx.x >> log_t); m < M; m += (int64_t)gridDim.x * rows) {
        for (unsigned c = lane * 8; c < (unsigned)cols; c += T * 8) {
            float sum[8] = {};
            for (int j = 0; j < top_k; ++j) {
                const int p = place[m * top_k + j];
                if (!placed(p, most)) continue;
                const float w = wt ? wt[m * top_k + j] : 1.0f;
                float f[8];
                load8<ZE>(z, (int64_t)p * ldz, (int)c, cols, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += w * f[i];
            }
            const int64_t o = m * ldo + c;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < cols - (int)c) store_elem(out, o + i, sum[i], out_elem);
        }
    }
}

// A workgroup per row: dout is read for each group of slots, and every slot's z
// once.
template <int ZE, int OE>
__global__ __launch_bounds__(256) void k_combine_grad(void* __restrict__ dz, int64_t lddz, float* __restrict__ dw,
                                                      const void* __restrict__ z, int64_t ldz,
                                                      const void* __restrict__ dout, int64_t ldo,
                                                      const int32_t* __restrict__ place, const float* __restrict__ wt,
                                                      int64_t M, int top_k, int cols) {
    __shared__ float part[4];
    const int64_t most = M * top_k;
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        for (int j = 0; j < top_k; ++j) {
            const int64_t q = m * top_k + j;
            const int p = place[q];
            const bool on = placed(p, most);  // the same for the workgroup
            float dot = 0.0f;
            if (on) {
                const float w = wt ? wt[q] : 1.0f;
                for (unsigned c = threadIdx.x * 8; c < (unsigned)cols; c += 256 * 8) {
                    float d[8];
                    load8<OE>(dout, m * ldo, (int)c, cols, d);
                    if (dw) {
                        float f[8];
                        load8<ZE>(z, (int64_t)p * ldz, (int)c, cols, f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(d[i], f[i], dot);
                    }
                    if (dz) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < cols - (int)c) store_elem(dz, (int64_t)p * lddz + c + i, w * d[i], ZE);
                    }
                }
            }
            if (!dw) continue;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
            if (lane_id() == 0) part[threadIdx.x >> 6] = dot;
            __syncthreads();
            if (threadIdx.x == 0) dw[q] = part[0] + part[1] + part[2] + part[3];
            __syncthreads();
        }
    }
}

unsigned grid_of(int64_t blocks, unsigned most) { return (unsigned)(blocks < most ? blocks : most); }

}  // namespace

size_t dispatch_place_bytes(int64_t pairs, int n_experts) {
    return (size_t)((pairs + kPairs - 1) / kPairs) * n_experts * 4;
}

int launch_place(vdttfs_ctx* ctx, const PlaceArgs& a, int* hist) {
    const int64_t pairs = a.M * a.top_k;
    const int blocks = (int)((pairs + kPairs - 1) / kPairs);
    int log = 0;
    while ((1 << log) < a.E) ++log;
    if (blocks > 0) {
        k_place_count<<<dim3((unsigned)blocks), 1024, 0, ctx->stream>>>(a, hist);
        VD_HIP(hipGetLastError());
    }
    k_place_scan<<<dim3(1), 1024, 0, ctx->stream>>>(a, hist, blocks, log);
    VD_HIP(hipGetLastError());
    if (blocks > 0) {
        k_place<<<dim3((unsigned)blocks), 1024, (size_t)kWaves * a.E * 4, ctx->stream>>>(a, hist, log);
        VD_HIP(hipGetLastError());
    }
    return VDTTFS_OK;
}

int launch_dispatch_rows(vdttfs_ctx* ctx, const PlaceArgs& a, void* z, int64_t ldz, const void* x, int elem, int64_t ldx,
                         int cols) {
    if (a.M <= 0 || cols <= 0) return VDTTFS_OK;
    k_dispatch_rows<<<dim3(grid_of(a.M, 1 << 20)), kCopy, 0, ctx->stream>>>(a, z, ldz, x, ldx, cols,
                                                                            elem == VDTTFS_ELEM_F32 ? 4 : 2);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_gather_sum(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const void* z, int z_elem, int64_t ldz,
                      const int32_t* place, const float* wt, int64_t M, int top_k, int cols) {
    int log_t = 2;
    while (log_t < 8 && (8 << log_t) < cols) ++log_t;
    const int64_t rows = 256 >> log_t;
    const dim3 grid(grid_of((M + rows - 1) / rows, 1 << 20));
    if (z_elem == VDTTFS_ELEM_F32)
        k_gather_sum<VDTTFS_ELEM_F32><<<grid, 256, 0, ctx->stream>>>(out, out_elem, ldo, z, ldz, place, wt, M, top_k,
                                                                     cols, log_t);
    else if (z_elem == VDTTFS_ELEM_BF16)
        k_gather_sum<VDTTFS_ELEM_BF16><<<grid, 256, 0, ctx->stream>>>(out, out_elem, ldo, z, ldz, place, wt, M, top_k,
                                                                      cols, log_t);
    else
        k_gather_sum<VDTTFS_ELEM_F16><<<grid, 256, 0, ctx->stream>>>(out, out_elem, ldo, z, ldz, place, wt, M, top_k,
                                                                     cols, log_t);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

template <int ZE>
static void combine_grad_z(vdttfs_ctx* ctx, void* dz, int64_t lddz, float* dw, const void* z, int64_t ldz,
                           const void* dout, int out_elem, int64_t ldo, const int32_t* place, const float* wt, int64_t M,
                           int top_k, int cols) {
    const dim3 grid(grid_of(M, 1 << 20));
    if (out_elem == VDTTFS_ELEM_F32)
        k_combine_grad<ZE, VDTTFS_ELEM_F32><<<grid, 256, 0, ctx->stream>>>(dz, lddz, dw, z, ldz, dout, ldo, place, wt,
                                                                           M, top_k, cols);
    else if (out_elem == VDTTFS_ELEM_BF16)
        k_combine_grad<ZE, VDTTFS_ELEM_BF16><<<grid, 256, 0, ctx->stream>>>(dz, lddz, dw, z, ldz, dout, ldo, place, wt,
                                                                            M, top_k, cols);
    else
        k_combine_grad<ZE, VDTTFS_ELEM_F16><<<grid, 256, 0, ctx->stream>>>(dz, lddz, dw, z, ldz, dout, ldo, place, wt,
                                                                           M, top_k, cols);
}

int launch_combine_grad(vdttfs_ctx* ctx, void* dz, int64_t lddz, float* dw, const void* z, int z_elem, int64_t ldz,
                        const void* dout, int out_elem, int64_t ldo, const int32_t* place, const float* wt, int64_t M,
                        int top_k, int cols) {
    if (z_elem == VDTTFS_ELEM_F32)
        combine_grad_z<VDTTFS_ELEM_F32>(ctx, dz, lddz, dw, z, ldz, dout, out_elem, ldo, place, wt, M, top_k, cols);
    else if (z_elem == VDTTFS_ELEM_BF16)
        combine_grad_z<VDTTFS_ELEM_BF16>(ctx, dz, lddz, dw, z, ldz, dout, out_elem, ldo, place, wt, M, top_k, cols);
    else
        combine_grad_z<VDTTFS_ELEM_F16>(ctx, dz, lddz, dw, z, ldz, dout, out_elem, ldo, place, wt, M, top_k, cols);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
