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

// max of two values >= 0 or NaN; a NaN wins.
__device__ __forceinline__ float nan_max(float a, float b) { return (a >= b || a != a) ? a : b; }

__device__ __forceinline__ float scale_of(float amax) {
    return amax < __builtin_inff() ? amax / 127.0f : __builtin_nanf("");
}

// The largest magnitude over WAVES waves (all of the workgroup, or one).
template <int WAVES>
__device__ __forceinline__ float row_max(float v, float* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = nan_max(v, __shfl_xor(v, off, 64));
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

// Eight neighbouring values from column c of a row, 0 past its end.  vec: rows
// start on 16 bytes.
template <int ELEM>
__device__ __forceinline__ void load8(const void* x, int64_t row, int c, int cols, bool vec, float (&f)[8]) {
    if (vec && c + 8 <= cols) {
        if constexpr (ELEM == VDTTFS_ELEM_F32) {
            const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + row + c);
            const float4 a = p[0], b = p[1];
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + row + c);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                f[i] = ELEM == VDTTFS_ELEM_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < cols ? load_elem<ELEM>(x, row + c + i) : 0.0f;
}

// Eight codes at column c; columns past `end` are not there.
__device__ __forceinline__ void store8(int8_t* q, int64_t row, int c, int end, bool vec, const int (&k)[8]) {
    if (vec && c + 8 <= end) {
        uint2 w;
        w.x = (k[0] & 255) | (k[1] & 255) << 8 | (k[2] & 255) << 16 | k[3] << 24;
        w.y = (k[4] & 255) | (k[5] & 255) << 8 | (k[6] & 255) << 16 | k[7] << 24;
        *reinterpret_cast<uint2*>(q + row + c) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < end) q[row + c + i] = (int8_t)k[i];
}

// WAVES waves hold a row in registers, eight values a lane and turn (NV turns),
// so it is read once: its largest magnitude, then its codes.  Bound by memory;
// the IEEE quotients overlap it.
template <int ELEM, int NV, int WAVES>
__global__ __launch_bounds__(kThreads) void k_quant_rows(const void* __restrict__ x, int64_t ldx, int64_t rows,
                                                         int cols, int8_t* __restrict__ q, int64_t ldq,
                                                         int cols_zero, float* __restrict__ scale, int vec_in,
                                                         int vec_out) {
    __shared__ float lds[kThreads / 64];
    constexpr int kRows = kThreads / 64 / WAVES, kLanes = WAVES * 64;
    const int lane = threadIdx.x % kLanes;
    for (int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes; m < rows; m += (int64_t)gridDim.x * kRows) {
        float f[NV][8];
        float a = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) load8<ELEM>(x, m * ldx, (v * kLanes + lane) * 8, cols, vec_in, f[v]);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) a = nan_max(a, fabsf(f[v][i]));
        const float s = scale_of(row_max<WAVES>(a, lds));
        if (lane == 0) scale[m] = s;
        const bool ok = s == s;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            int k[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = ok ? code_of(f[v][i], s) : 0;
            store8(q, m * ldq, (v * kLanes + lane) * 8, cols_zero, vec_out, k);
        }
    }
}

// Longer rows: a workgroup each, read twice (the second time from the caches).
template <int ELEM>
__global__ __launch_bounds__(kThreads) void k_quant_long(const void* __restrict__ x, int64_t ldx, int64_t rows,
                                                         int cols, int8_t* __restrict__ q, int64_t ldq,
                                                         int cols_zero, float* __restrict__ scale, int vec_in,
                                                         int vec_out) {
    __shared__ float lds[kThreads / 64];
    for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
        float a = 0.0f;
        for (int c = threadIdx.x * 8; c < cols; c += kThreads * 8) {
            float f[8];
            load8<ELEM>(x, m * ldx, c, cols, vec_in, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) a = nan_max(a, fabsf(f[i]));
        }
        const float s = scale_of(row_max<kThreads / 64>(a, lds));
        if (threadIdx.x == 0) scale[m] = s;
        const bool ok = s == s;
        for (int c = threadIdx.x * 8; c < cols_zero; c += kThreads * 8) {
            float f[8];
            int k[8];
            load8<ELEM>(x, m * ldx, c, cols, vec_in, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) k[i] = ok ? code_of(f[i], s) : 0;
            store8(q, m * ldq, c, cols_zero, vec_out, k);
        }
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

namespace {

template <int ELEM, int NV, int WAVES>
void quant_nv(vdttfs_ctx* ctx, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q, int64_t ldq,
              int cols_zero, float* scale, int vi, int vo) {
    constexpr int kRows = kThreads / 64 / WAVES;
    const int64_t blocks = (rows + kRows - 1) / kRows;
    k_quant_rows<ELEM, NV, WAVES><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), kThreads, 0, ctx->stream>>>(
        x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
}

// A wave per row up to 2048 columns where there are rows for every SIMD, else
// four.
template <int ELEM>
void quant_elem(vdttfs_ctx* ctx, const void* x, int64_t ldx, int64_t rows, int cols, int8_t* q, int64_t ldq,
                int cols_zero, float* scale) {
    const int size = ELEM == VDTTFS_ELEM_F32 ? 4 : 2;
    const int vi = (((uintptr_t)x | (uintptr_t)(ldx * size)) & 15) == 0;
    const int vo = (((uintptr_t)q | (uintptr_t)ldq) & 7) == 0;
    if (cols_zero <= 512) quant_nv<ELEM, 1, 1>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else if (cols_zero <= 1024 && rows >= 1024)
        quant_nv<ELEM, 2, 1>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else if (cols_zero <= 2048 && rows >= 1024)
        quant_nv<ELEM, 4, 1>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else if (cols_zero <= 2048) quant_nv<ELEM, 1, 4>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else if (cols_zero <= 4096) quant_nv<ELEM, 2, 4>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else if (cols_zero <= 8192) quant_nv<ELEM, 4, 4>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
    else
        k_quant_long<ELEM><<<dim3((unsigned)(rows < 65536 ? rows : 65536)), kThreads, 0, ctx->stream>>>(
            x, ldx, rows, cols, q, ldq, cols_zero, scale, vi, vo);
}

}  // namespace

int launch_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                      int64_t ldq, int cols_zero, float* scale) {
    if (rows <= 0) return VDTTFS_OK;
    if (elem == VDTTFS_ELEM_F32) quant_elem<VDTTFS_ELEM_F32>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_BF16) quant_elem<VDTTFS_ELEM_BF16>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else if (elem == VDTTFS_ELEM_F16) quant_elem<VDTTFS_ELEM_F16>(ctx, x, ldx, rows, cols, q, ldq, cols_zero, scale);
    else
        k_quant_times<<<dim3((unsigned)(rows < 65536 ? rows : 65536)), kThreads, 0, ctx->stream>>>(
            static_cast<const float*>(x), ldx, rows, cols, q, ldq, cols_zero, scale, ctx->c.tfs, ctx->c.T);
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
