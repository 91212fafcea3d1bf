// Routing of rows to experts, the sort of the chosen pairs by expert, and the
// weighted sum of the experts' outputs.
#include "elem.h"
#include "head.h"
#include "wave.h"

namespace vdttfs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxExperts = 1024;
constexpr int kSortPairs = 2048;  // pairs a workgroup of the sort takes

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

struct RouteArgs {
    int32_t* idx;
    float* wt;
    int32_t* count;
    const void* logits;
    int64_t ld;
    const float* bias;
    const uint8_t* row_mask;
    int64_t M;
    int E, k, score, groups, top_groups, group_top, renorm;
    float scale;
};

// A wave per row, NPL neighbouring experts a lane: the largest value of the
// wave is then first in index order at the first lane that holds it.
template <int ELEM, int NPL>
__global__ __launch_bounds__(kThreads) void k_route(RouteArgs a) {
    __shared__ int hist[kMaxExperts];
    __shared__ float group_c[kWaves][64 * NPL];
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    if (a.count) {
        for (int e = threadIdx.x; e < a.E; e += kThreads) hist[e] = 0;
        __syncthreads();
    }
    float bias[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int e = lane * NPL + i;
        bias[i] = a.bias && e < a.E ? a.bias[e] : 0.0f;
    }
    const int per = a.E / a.groups;
    for (int64_t m = (int64_t)blockIdx.x * kWaves + wave; m < a.M; m += (int64_t)gridDim.x * kWaves) {
        const bool row = !a.row_mask || a.row_mask[m] != 0;
        float p[NPL], c[NPL];
        float mx = neg_inf();
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int e = lane * NPL + i;
            const float l = row && e < a.E ? load_elem<ELEM>(a.logits, m * a.ld + e) : neg_inf();
            c[i] = l > neg_inf() ? l : neg_inf();  // NaN: not choosable
            mx = fmaxf(mx, c[i]);
        }
        if (a.score == VDTTFS_SCORE_SOFTMAX) {
            mx = wave_max(mx);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                p[i] = c[i] > neg_inf() ? (c[i] == mx ? 1.0f : expf(c[i] - mx)) : 0.0f;
                sum += p[i];
            }
            sum = wave_sum(sum);
#pragma unroll
            for (int i = 0; i < NPL; ++i) p[i] = p[i] / sum;  // a row without experts is never read
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) p[i] = 1.0f / (1.0f + expf(-c[i]));
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float v = p[i] + bias[i];
            c[i] = c[i] > neg_inf() && v > neg_inf() ? v : neg_inf();
        }
        if (a.groups > 1) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) group_c[wave][lane * NPL + i] = c[i];
            wave_sync();
            float t0 = neg_inf(), t1 = neg_inf();
            if (lane < a.groups)
                for (int i = 0; i < per; ++i) {
                    const float v = group_c[wave][lane * per + i];
                    t1 = fmaxf(t1, fminf(t0, v));
                    t0 = fmaxf(t0, v);
                }
            wave_sync();
            const float g = a.group_top == 2 && t1 > neg_inf() ? t0 + t1 : t0;
            int rank = 0;
            for (int o = 0; o < a.groups; ++o) {
                const float v = __shfl(g, o, 64);
                rank += v > g || (v == g && o < lane) ? 1 : 0;
            }
            const uint64_t keep = __ballot(lane < a.groups && rank < a.top_groups);
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const int e = lane * NPL + i;
                if (e < a.E && !((keep >> (e / per)) & 1)) c[i] = neg_inf();
            }
        }
        int my_idx = -1;
        float my_w = 0.0f;
        for (int j = 0; j < a.k; ++j) {
            float bv = neg_inf(), bp = 0.0f;
            int bi = -1;
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (c[i] > bv) {
                    bv = c[i];
                    bp = p[i];
                    bi = lane * NPL + i;
                }
            const float best = wave_max(bv);
            if (!(best > neg_inf())) break;
            const int src = __builtin_ctzll(__ballot(bv == best));
            const int e = __shfl(bi, src, 64);
            const float w = __shfl(bp, src, 64);
            if (lane == j) {
                my_idx = e;
                my_w = w;
            }
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                if (lane * NPL + i == e) c[i] = neg_inf();
        }
        if (a.renorm) {
            const float sum = wave_sum(my_w);
            my_w = sum > 0.0f ? my_w / sum : 0.0f;
        }
        if (lane < a.k) {
            a.idx[m * a.k + lane] = my_idx;
            a.wt[m * a.k + lane] = my_w * a.scale;
            if (a.count && my_idx >= 0) atomicAdd(&hist[my_idx], 1);
        }
    }
    if (a.count) {
        __syncthreads();
        for (int e = threadIdx.x; e < a.E; e += kThreads) {
            if (gridDim.x == 1)
                a.count[e] = hist[e];
            else if (hist[e])
                atomicAdd(&a.count[e], hist[e]);
        }
    }
}

__global__ void k_zero(int* p, int n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) p[i] = 0;
}

template <int ELEM>
void route_npl(vdttfs_ctx* ctx, const RouteArgs& a, dim3 grid) {
    if (a.E <= 64) k_route<ELEM, 1><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 128) k_route<ELEM, 2><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 256) k_route<ELEM, 4><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 512) k_route<ELEM, 8><<<grid, kThreads, 0, ctx->stream>>>(a);
    else k_route<ELEM, 16><<<grid, kThreads, 0, ctx->stream>>>(a);
}

// Experts of each workgroup's pairs: hist[block][expert].
__global__ __launch_bounds__(kThreads) void k_sort_count(const int32_t* __restrict__ idx, int64_t pairs, int E,
                                                         int* __restrict__ hist) {
    __shared__ int h[kMaxExperts];
    for (int e = threadIdx.x; e < E; e += kThreads) h[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kSortPairs; i += kThreads) {
        const int64_t q = (int64_t)blockIdx.x * kSortPairs + i;
        if (q >= pairs) break;
        const int e = idx[q];
        if (e >= 0 && e < E) atomicAdd(&h[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads) hist[(int64_t)blockIdx.x * E + e] = h[e];
}

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

// One workgroup: hist[block][expert] becomes the sorted position of the
// block's first pair of the expert; the row tiles of every expert follow.
__global__ __launch_bounds__(1024) void k_sort_plan(int* __restrict__ hist, int blocks, int E, int bm,
                                                    int4* __restrict__ tiles, int* __restrict__ n_tiles) {
    __shared__ int lds[16];
    const int e = threadIdx.x;
    int n = 0;
    if (e < E)
        for (int b = 0; b < blocks; ++b) n += hist[(int64_t)b * E + e];
    int all;
    const int start = block_excl_scan(n, lds, &all);
    if (e < E) {
        int at = start;
        for (int b = 0; b < blocks; ++b) {
            const int h = hist[(int64_t)b * E + e];
            hist[(int64_t)b * E + e] = at;
            at += h;
        }
    }
    const int t = (n + bm - 1) / bm;
    int t_all;
    const int t0 = block_excl_scan(t, lds, &t_all);
    for (int i = 0; i < t; ++i) tiles[t0 + i] = make_int4(e, start + i * bm, start + n, 0);
    if (threadIdx.x == 0) *n_tiles = t_all;
}

// Each pair to its place.  The order of an expert's pairs within a workgroup
// is that of its LDS atomics; nothing that is computed depends on it.
__global__ __launch_bounds__(kThreads) void k_sort_place(const int32_t* __restrict__ idx, int64_t pairs, int E,
                                                         int top_k, const int* __restrict__ hist,
                                                         int* __restrict__ pair, int* __restrict__ row) {
    __shared__ int at[kMaxExperts];
    for (int e = threadIdx.x; e < E; e += kThreads) at[e] = hist[(int64_t)blockIdx.x * E + e];
    __syncthreads();
    for (int i = threadIdx.x; i < kSortPairs; i += kThreads) {
        const int64_t q = (int64_t)blockIdx.x * kSortPairs + i;
        if (q >= pairs) break;
        const int e = idx[q];
        if (e < 0 || e >= E) continue;
        const int to = atomicAdd(&at[e], 1);
        pair[to] = (int)q;
        row[to] = (int)(q / top_k);
    }
}

// A workgroup per row: the slots' outputs summed in order.
__global__ __launch_bounds__(kThreads) void k_combine(void* __restrict__ out, int out_elem, int64_t ldo,
                                                      const float* __restrict__ z, const int32_t* __restrict__ idx,
                                                      const float* __restrict__ wt, int64_t M, int N, int top_k,
                                                      int E) {
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        for (int n = threadIdx.x; n < N; n += kThreads) {
            float sum = 0.0f;
            for (int j = 0; j < top_k; ++j) {
                const int64_t q = m * top_k + j;
                const int e = idx[q];
                if (e >= 0 && e < E) sum += wt[q] * z[q * N + n];
            }
            store_elem(out, m * ldo + n, sum, out_elem);
        }
    }
}

}  // namespace

int launch_route(vdttfs_ctx* ctx, int32_t* idx, float* wt, int32_t* count, const void* logits, int elem, int64_t ld,
                 const float* bias, const uint8_t* row_mask, int64_t M, const vdttfs_route_opts& o) {
    const int64_t blocks = (M + kWaves - 1) / kWaves;
    const dim3 grid((unsigned)(blocks < 2048 ? blocks : 2048));
    if (count && (M <= 0 || grid.x > 1)) {
        k_zero<<<dim3(1), kThreads, 0, ctx->stream>>>(count, o.n_experts);
        VD_HIP(hipGetLastError());
    }
    if (M <= 0) return VDTTFS_OK;
    const RouteArgs a{idx,           wt,      count,    logits,       ld,           bias,     row_mask, M,
                      o.n_experts,   o.top_k, o.score,  o.groups,     o.top_groups, o.group_top, o.renorm, o.scale};
    if (elem == VDTTFS_ELEM_F32) route_npl<VDTTFS_ELEM_F32>(ctx, a, grid);
    else if (elem == VDTTFS_ELEM_BF16) route_npl<VDTTFS_ELEM_BF16>(ctx, a, grid);
    else route_npl<VDTTFS_ELEM_F16>(ctx, a, grid);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int dispatch_blocks(int64_t pairs) { return (int)((pairs + kSortPairs - 1) / kSortPairs); }

int launch_dispatch(vdttfs_ctx* ctx, const int32_t* idx, int64_t pairs, int top_k, int n_experts, int bm,
                    const Dispatch& d) {
    const int blocks = dispatch_blocks(pairs);
    k_sort_count<<<dim3((unsigned)blocks), kThreads, 0, ctx->stream>>>(idx, pairs, n_experts, d.hist);
    VD_HIP(hipGetLastError());
    k_sort_plan<<<dim3(1), 1024, 0, ctx->stream>>>(d.hist, blocks, n_experts, bm, d.tiles, d.n_tiles);
    VD_HIP(hipGetLastError());
    k_sort_place<<<dim3((unsigned)blocks), kThreads, 0, ctx->stream>>>(idx, pairs, n_experts, top_k, d.hist, d.pair,
                                                                       d.row);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_combine(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const float* z, const int32_t* idx,
                   const float* wt, int64_t M, int N, int top_k, int n_experts) {
    const dim3 grid((unsigned)(M < (1 << 20) ? M : 1 << 20));
    k_combine<<<grid, kThreads, 0, ctx->stream>>>(out, out_elem, ldo, z, idx, wt, M, N, top_k, n_experts);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
