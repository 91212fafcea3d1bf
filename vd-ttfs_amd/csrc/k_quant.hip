// Rows of floats or spike times to 8-bit codes with a float scale each, and
// the weights blob's FC kernels to the products' layout.
#include "elem.h"
#include "head.h"
#include "quant.h"
#include "sort.h"

namespace vdttfs {
namespace {

constexpr int kThreads = 256;

// The largest magnitude over WAVES waves (all of the workgroup, or one).
template <int WAVES>
__device__ __forceinline__ float row_max(float v, float* lds) {
    v = wave_nan_max(v);
    if constexpr (WAVES > 1) {
        if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = nan_max(v, lds[i]);
        __syncthreads();
    }
    return v;
}

// Eight codes at column c; columns past `end` are not there.
__device__ __forceinline__ void store8(int8_t* q, int64_t row, int c, int end, bool vec, const int (&k)[8]) {
    if (vec && end - c >= 8) {
        *reinterpret_cast<uint2*>(q + row + c) = pack8(k);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < end - c) q[row + c + i] = (int8_t)k[i];
}

// The largest magnitude over LANES lanes that share a row: a part of a wave, a
// wave, or the workgroup.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v, float* lds) {
    if constexpr (LANES >= 64) return row_max<LANES / 64>(v, lds);
#pragma unroll
    for (int o = 1; o < LANES && o < 64; o *= 2) v = nan_max(v, __shfl_xor(v, o, 64));
    return v;
}

// LANES lanes hold a row in registers, eight values a lane and turn (NV turns),
// so it is read once: its largest magnitude, then its codes.  Bound by memory:
// 8192 x 4096 of BF16 in 27 us, 3.7 TB/s; 61000 x 1024 of F32 that a product has
// just left in 57, 5.4.
// THREADS a workgroup, this one `block` of `blocks`.
template <int ELEM, int NV, int LANES, int THREADS>
__device__ __forceinline__ void quant_rows(const void* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                                           int8_t* __restrict__ q, int64_t ldq, int cols_zero,
                                           float* __restrict__ scale, int vec_out, unsigned block, unsigned blocks) {
    static_assert(LANES <= 64 || LANES == THREADS, "a row has a part of a wave, a wave or the workgroup");
    __shared__ float lds[THREADS / 64];
    constexpr int kRows = THREADS / LANES, kLanes = LANES;
    const int lane = threadIdx.x % kLanes;
    for (int64_t m = (int64_t)block * kRows + threadIdx.x / kLanes; m < rows; m += (int64_t)blocks * kRows) {
        Raw8<ELEM> raw[NV];
        float f[NV][8], a = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * kLanes + lane) * 8;
            raw[v] = nothing8<ELEM>();
            if (c + 8 <= cols) raw[v] = raw8<ELEM>(x, m * ldx + c);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * kLanes + lane) * 8;
            unpack8<ELEM>(raw[v], f[v]);
            if (c < cols && c + 8 > cols) tail8<ELEM>(x, m * ldx, c, cols, f[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) a = nan_max(a, fabsf(f[v][i]));
        const float s = scale_of(lanes_max<LANES>(a, lds));
        if (lane == 0) scale[m] = s;
        const Coder coder = coder_of(s);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            int k[8];
            codes8(f[v], coder, k);
            store8(q, m * ldq, (v * kLanes + lane) * 8, cols_zero, vec_out, k);
        }
    }
}
template <int ELEM, int NV, int LANES>
__global__ __launch_bounds__(kThreads) void k_quant_rows(const void* __restrict__ x, int64_t ldx, int64_t rows,
                                                         int cols, int8_t* __restrict__ q, int64_t ldq,
                                                         int cols_zero, float* __restrict__ scale, int vec_out) {
    quant_rows<ELEM, NV, LANES, kThreads>(x, ldx, rows, cols, q, ldq, cols_zero, scale, vec_out, blockIdx.x, gridDim.x);
}

// Longer rows: a workgroup each, read twice (the second time from the caches).
template <int ELEM>
__global__ __launch_bounds__(kThreads) void k_quant_long(const void* __restrict__ x, int64_t ldx, int64_t rows,
                                                         int cols, int8_t* __restrict__ q, int64_t ldq,
                                                         int cols_zero, float* __restrict__ scale, int vec_out) {
    __shared__ float lds[kThreads / 64];
    for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
        float a = 0.0f;
        // unsigned: a thread's column goes past the row's end, and past 2^31
        for (unsigned c = threadIdx.x * 8; c < (unsigned)cols; c += kThreads * 8) {
            float f[8];
            load8<ELEM>(x, m * ldx, (int)c, cols, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) a = nan_max(a, fabsf(f[i]));
        }
        const float s = scale_of(row_max<kThreads / 64>(a, lds));
        if (threadIdx.x == 0) scale[m] = s;
        const Coder coder = coder_of(s);
        for (unsigned c = threadIdx.x * 8; c < (unsigned)cols_zero; c += kThreads * 8) {
            float f[8];
            int k[8];
            load8<ELEM>(x, m * ldx, (int)c, cols, f);
            codes8(f, coder, k);
            store8(q, m * ldq, (int)c, cols_zero, vec_out, k);
        }
    }
}

// Runs of eight in a row, at least one.
__host__ __device__ __forceinline__ int runs_of(int cols) { return cols > 0 ? (cols - 1) / 8 + 1 : 1; }

// Spike times: eight a thread; the scale is the same for every row.
__device__ __forceinline__ void quant_times(const float* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                                            int8_t* __restrict__ q, int64_t ldq, int cols_zero,
                                            float* __restrict__ scale, float tfs, int T, int vec_out, unsigned block,
                                            unsigned blocks) {
    const int levels = T < 127 ? T : 127, per = runs_of(cols_zero);
    for (int64_t at = (int64_t)block * blockDim.x + threadIdx.x; at < rows * per; at += (int64_t)blocks * blockDim.x) {
        const int64_t m = at / per;
        const int c = (int)(at - m * per) * 8;
        float f[8];
        int k[8];
        load8<VDTTFS_ELEM_TIMES>(x, m * ldx, c, cols, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = time_code(f[i], tfs, T, levels);
        store8(q, m * ldq, c, cols_zero, vec_out, k);
        if (c == 0) scale[m] = 1.0f / (float)levels;
    }
}
__global__ __launch_bounds__(kThreads) void k_quant_times(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                          int cols, int8_t* __restrict__ q, int64_t ldq,
                                                          int cols_zero, float* __restrict__ scale, float tfs, int T,
                                                          int vec_out) {
    quant_times(x, ldx, rows, cols, q, ldq, cols_zero, scale, tfs, T, vec_out, blockIdx.x, gridDim.x);
}

// Rows quantised and, by the first workgroup, the pairs of the experts that will
// take them sorted: neither needs the other, so one launch does both.
constexpr int kSortThreads = 1024;
template <int ELEM, int NV, int LANES>
__global__ __launch_bounds__(kSortThreads) void k_quant_sort(SortOne sort, const void* __restrict__ x, int64_t ldx,
                                                             int64_t rows, int cols, int8_t* __restrict__ q,
                                                             int64_t ldq, int cols_zero, float* __restrict__ scale,
                                                             float tfs, int T, int vec_out) {
    if (blockIdx.x == 0) {
        sort_one(sort);
    } else if constexpr (ELEM == VDTTFS_ELEM_TIMES) {
        quant_times(static_cast<const float*>(x), ldx, rows, cols, q, ldq, cols_zero, scale, tfs, T, vec_out,
                    blockIdx.x - 1, gridDim.x - 1);
    } else {
        quant_rows<ELEM, NV, LANES, kSortThreads>(x, ldx, rows, cols, q, ldq, cols_zero, scale, vec_out,
                                                  blockIdx.x - 1, gridDim.x - 1);
    }
}

// [C_in][C_out] floats to [C_out][ldw] codes: a lane per output channel reads
// down its column (64 neighbouring columns a wave, so rows come in whole
// lines), 16 threads of the workgroup sharing a column.  For a program's start:
// weights are laid out once.
__global__ __launch_bounds__(1024) void k_quant_kernel(const float* __restrict__ w, int c_in, int c_out,
                                                       int8_t* __restrict__ q, int64_t ldq,
                                                       float* __restrict__ scale) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane;
    float a = 0.0f;
    if (n < c_out)
        for (unsigned k = part; k < (unsigned)c_in; k += 16) a = nan_max(a, fabsf(w[(int64_t)k * c_out + n]));
    lds[part][lane] = a;
    __syncthreads();
    for (int i = 0; i < 16; ++i) a = nan_max(a, lds[i][lane]);
    if (n >= c_out) return;
    const float s = scale_of(a);
    if (part == 0) scale[n] = s;
    for (unsigned k = part; k < (unsigned)c_in; k += 16)
        q[(int64_t)n * ldq + k] = s > 0.0f ? (int8_t)exact_code(w[(int64_t)k * c_out + n], s) : (int8_t)0;
}

}  // namespace

namespace {

template <int ELEM, int NV, int LANES>
void quant_nv(vdttfs_ctx* ctx, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q, int64_t ldq,
              int cols_zero, float* scale, int vo) {
    constexpr int kRows = kThreads / LANES;
    const int64_t blocks = (rows + kRows - 1) / kRows;
    k_quant_rows<ELEM, NV, LANES><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), kThreads, 0, ctx->stream>>>(
        x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
}

// As many rows a wave as fit up to 256 columns (36477 x 60: 14.8 us with a wave
// per row, 6 so); a wave per row up to 2048 where there are rows for every SIMD;
// else four.
template <int ELEM>
void quant_elem(vdttfs_ctx* ctx, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q, int64_t ldq,
                int cols_zero, float* scale) {
    const int vo = (((uintptr_t)q | (uintptr_t)ldq) & 7) == 0;
    if (cols_zero <= 128) quant_nv<ELEM, 1, 16>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 256) quant_nv<ELEM, 1, 32>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 512) quant_nv<ELEM, 1, 64>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 1024 && rows >= 1024)
        quant_nv<ELEM, 2, 64>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 2048 && rows >= 1024)
        quant_nv<ELEM, 4, 64>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 2048) quant_nv<ELEM, 1, 256>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 4096) quant_nv<ELEM, 2, 256>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else if (cols_zero <= 8192) quant_nv<ELEM, 4, 256>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
    else
        k_quant_long<ELEM><<<dim3((unsigned)(rows < 65536 ? rows : 65536)), kThreads, 0, ctx->stream>>>(
            x, ldx, rows, cols, q, ldq, cols_zero, scale, vo);
}

template <int ELEM, int NV, int LANES>
void quant_sort(vdttfs_ctx* ctx, const SortOne& sort, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q,
                int64_t ldq, int cols_zero, float* scale) {
    // rows of a workgroup; of spike times, eight values a thread
    const int64_t blocks = ELEM == VDTTFS_ELEM_TIMES
                               ? (rows * runs_of(cols_zero) + kSortThreads - 1) / kSortThreads
                               : (rows + kSortThreads / LANES - 1) / (kSortThreads / LANES);
    const int vo = (((uintptr_t)q | (uintptr_t)ldq) & 7) == 0;
    k_quant_sort<ELEM, NV, LANES><<<dim3(1 + (unsigned)(blocks < 65536 ? blocks : 65536)), kSortThreads, 0, ctx->stream>>>(
        sort, x, ldx, rows, cols, q, ldq, cols_zero, scale, ctx->c.tfs, ctx->c.T, vo);
}

constexpr int kMaxSortCols = 2048;  // a wave holds a row
template <int ELEM>
void quant_sort_elem(vdttfs_ctx* ctx, const SortOne& sort, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q,
                     int64_t ldq, int cols_zero, float* scale) {
    if (cols_zero <= 128) quant_sort<ELEM, 1, 16>(ctx, sort, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (cols_zero <= 256) quant_sort<ELEM, 1, 32>(ctx, sort, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (cols_zero <= 512) quant_sort<ELEM, 1, 64>(ctx, sort, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (cols_zero <= 1024) quant_sort<ELEM, 2, 64>(ctx, sort, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else quant_sort<ELEM, 4, 64>(ctx, sort, x, ldx, rows, cols, q, ldq, cols_zero, scale);
}

}  // namespace

int launch_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                      int64_t ldq, int cols_zero, float* scale) {
    if (rows <= 0) return VDTTFS_OK;
    if (elem == VDTTFS_ELEM_F32) quant_elem<VDTTFS_ELEM_F32>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_BF16) quant_elem<VDTTFS_ELEM_BF16>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_F16) quant_elem<VDTTFS_ELEM_F16>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else {
        const int64_t blocks = (rows * runs_of(cols_zero) + kThreads - 1) / kThreads;
        k_quant_times<<<dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), kThreads, 0, ctx->stream>>>(
            static_cast<const float*>(x), ldx, rows, cols, q, ldq, cols_zero, scale, ctx->c.tfs, ctx->c.T,
            (((uintptr_t)q | (uintptr_t)ldq) & 7) == 0);
    }
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_quant_dispatch(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                          int64_t ldq, int cols_zero, float* scale, const int32_t* idx, int64_t pairs, int top_k,
                          int n_experts, int bm, const Dispatch& d) {
    if (pairs > kSortOne || cols_zero > kMaxSortCols) {
        VD_TRY(launch_quant_rows(ctx, x, elem, ldx, rows, cols, q, ldq, cols_zero, scale));
        return launch_dispatch(ctx, idx, pairs, top_k, n_experts, bm, d);
    }
    const SortOne s{idx, (int)pairs, n_experts, top_k, bm, d.tiles, d.n_tiles, d.pair, d.row};
    if (elem == VDTTFS_ELEM_F32)
        quant_sort_elem<VDTTFS_ELEM_F32>(ctx, s, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_BF16)
        quant_sort_elem<VDTTFS_ELEM_BF16>(ctx, s, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_F16)
        quant_sort_elem<VDTTFS_ELEM_F16>(ctx, s, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else quant_sort<VDTTFS_ELEM_TIMES, 1, 64>(ctx, s, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_quant_kernel(vdttfs_ctx* ctx, const float* kernel, int c_in, int c_out, int8_t* w, int64_t ldw,
                        float* scale) {
    if (c_out <= 0) return VDTTFS_OK;
    k_quant_kernel<<<dim3((unsigned)((c_out + 63) / 64)), 1024, 0, ctx->stream>>>(kernel, c_in, c_out, w, ldw, scale);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
