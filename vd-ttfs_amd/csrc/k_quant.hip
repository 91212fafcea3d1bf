// Rows of floats or spike times to 8-bit codes with a float scale each, and
// the weights blob's FC kernels to the products' layout.
#include "elem.h"
#include "head.h"
#include "wave.h"

namespace vdttfs {
namespace {

constexpr int kThreads = 256;

// The code of x under scale s (s finite): the IEEE quotient rounded half to
// even.  s == 0 is a row of zeros, or one whose largest value / 127 underflows.
__device__ __forceinline__ int code_of(float x, float s) {
    if (s == 0.0f) return 0;
    return (int)fminf(fmaxf(rintf(x / s), -127.0f), 127.0f);
}

// max over the workgroup of a value >= 0 or NaN; a NaN anywhere wins.
__device__ __forceinline__ float nan_max(float a, float b) { return (a >= b || a != a) ? a : b; }

__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = nan_max(v, __shfl_xor(v, off, 64));
    if (lane_id() == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) v = nan_max(v, lds[i]);
    __syncthreads();
    return v;
}

__device__ __forceinline__ float scale_of(float amax) {
    return amax < __builtin_inff() ? amax / 127.0f : __builtin_nanf("");
}

// One workgroup per row: the largest magnitude, then the codes (the second
// read of the row comes from the caches).
template <int ELEM>
__global__ __launch_bounds__(kThreads) void k_quant_rows(const void* __restrict__ x, int64_t ldx, int64_t rows,
                                                         int cols, int8_t* __restrict__ q, int64_t ldq,
                                                         int cols_zero, float* __restrict__ scale) {
    __shared__ float lds[kThreads / 64];
    for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
        float a = 0.0f;
        for (int i = threadIdx.x; i < cols; i += kThreads) a = nan_max(a, fabsf(load_elem<ELEM>(x, m * ldx + i)));
        const float s = scale_of(block_max(a, lds));
        if (threadIdx.x == 0) scale[m] = s;
        const bool ok = s == s;
        for (int i = threadIdx.x; i < cols_zero; i += kThreads)
            q[m * ldq + i] = i < cols && ok ? (int8_t)code_of(load_elem<ELEM>(x, m * ldx + i), s) : (int8_t)0;
    }
}

// Spike times: the scale is the same for every row.
__global__ __launch_bounds__(kThreads) void k_quant_times(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                          int cols, int8_t* __restrict__ q, int64_t ldq,
                                                          int cols_zero, float* __restrict__ scale, float tfs, int T) {
    const int L = T < 127 ? T : 127;
    for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
        if (threadIdx.x == 0) scale[m] = 1.0f / (float)L;
        for (int i = threadIdx.x; i < cols_zero; i += kThreads) {
            const int b = i < cols ? arrival_bin(x[m * ldx + i], tfs, T) : -1;
            q[m * ldq + i] = b < 0 ? (int8_t)0 : (int8_t)(int)rintf((float)((T - b) * L) / (float)T);
        }
    }
}

// [C_in][C_out] floats to [C_out][ldw] codes: a lane per output channel reads
// down its column (64 neighbouring columns a wave, so rows come in whole
// lines), 16 threads of the workgroup sharing a column.
__global__ __launch_bounds__(1024) void k_quant_kernel(const float* __restrict__ w, int c_in, int c_out,
                                                       int8_t* __restrict__ q, int64_t ldq,
                                                       float* __restrict__ scale) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + lane;
    float a = 0.0f;
    if (n < c_out)
        for (int k = part; k < c_in; k += 16) a = nan_max(a, fabsf(w[(int64_t)k * c_out + n]));
    lds[part][lane] = a;
    __syncthreads();
    for (int i = 0; i < 16; ++i) a = nan_max(a, lds[i][lane]);
    if (n >= c_out) return;
    const float s = scale_of(a);
    if (part == 0) scale[n] = s;
    for (int k = part; k < c_in; k += 16)
        q[(int64_t)n * ldq + k] = s == s ? (int8_t)code_of(w[(int64_t)k * c_out + n], s) : (int8_t)0;
}

}  // namespace

int launch_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                      int64_t ldq, int cols_zero, float* scale) {
    if (rows <= 0) return VDTTFS_OK;
    const dim3 grid((unsigned)(rows < (1 << 20) ? rows : 1 << 20));
    switch (elem) {
        case VDTTFS_ELEM_F32:
            k_quant_rows<VDTTFS_ELEM_F32><<<grid, kThreads, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, cols_zero,
                                                                             scale);
            break;
        case VDTTFS_ELEM_BF16:
            k_quant_rows<VDTTFS_ELEM_BF16><<<grid, kThreads, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, cols_zero,
                                                                              scale);
            break;
        case VDTTFS_ELEM_F16:
            k_quant_rows<VDTTFS_ELEM_F16><<<grid, kThreads, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, cols_zero,
                                                                             scale);
            break;
        default:
            k_quant_times<<<grid, kThreads, 0, ctx->stream>>>(static_cast<const float*>(x), ldx, rows, cols, q, ldq,
                                                              cols_zero, scale, ctx->c.tfs, ctx->c.T);
    }
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
