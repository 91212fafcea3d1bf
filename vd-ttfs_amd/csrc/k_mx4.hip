// Microscaled rows in 4 bits: quantisation, and products on the matrix cores.
//
// out[m][n] = act(sum_k A[m][k] B[n][k] + bias[n]), A and B elements of e2m1 times
// their blocks' powers of two.  The matrix instruction of 4-bit operands
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes a block of 32 and its scale from each
// lane, so the scales cost no instruction of their own.  Products of two elements
// are multiples of a quarter up to 36, so a block's sum is exact; the sum over
// blocks is in 32-bit floats.
#include "codes.h"
#include "elem.h"
#include "head.h"
#include "mx4.h"
#include "wave.h"

namespace vdttfs {
namespace {

// ---- quantisation -----------------------------------------------------------------
// Eight values a thread, four neighbouring threads a block of 32.
template <int ELEM>
__global__ __launch_bounds__(256) void k_mx4_quant(const void* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                                                   uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ s,
                                                   int64_t lds, int cols_zero, float tfs, int T) {
    const int64_t per = ((int64_t)cols_zero + kMxBlock - 1) / kMxBlock * 4;  // runs of eight in a row
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < rows * per; at += (int64_t)gridDim.x * 256) {
        const int64_t m = at / per;
        const int c = (int)(at - m * per) * 8;
        float f[8];
        load8<ELEM>(x, m * ldx, c, cols, f);
        if constexpr (ELEM == VDTTFS_ELEM_TIMES) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int b = arrival_bin(f[i], tfs, T);
                f[i] = b < 0 ? 0.0f : (float)(T - b) / (float)T;
            }
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, magnitude(f[i]));
        const int scale = mx4_scale(quad_max(most));
        mx4_store8(q + m * ldq, s + m * lds, c, cols_zero, mx4_codes8(f, scale), scale);
    }
}

// [C_in][C_out] floats to [C_out][ldw] codes: a lane per output channel takes a
// block of 32 down its column, so rows come in whole lines.  For a program's
// start: weights are laid out once.
__global__ __launch_bounds__(256) void k_mx4_quant_kernel(const float* __restrict__ w, int c_in, int c_out,
                                                          uint8_t* __restrict__ q, int64_t ldq,
                                                          uint8_t* __restrict__ s, int64_t lds) {
    const int n = blockIdx.x * 64 + lane_id();
    const int blocks = c_in / kMxBlock + (c_in % kMxBlock != 0);
    for (int b = blockIdx.y * 4 + (threadIdx.x >> 6); b < blocks; b += gridDim.y * 4) {
        if (n >= c_out) continue;
        float f[kMxBlock];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kMxBlock; ++i) {
            f[i] = i < c_in - b * kMxBlock ? w[((int64_t)b * kMxBlock + i) * c_out + n] : 0.0f;
            most = max(most, magnitude(f[i]));
        }
        const int scale = mx4_scale(most);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float g[8] = {f[8 * r],     f[8 * r + 1], f[8 * r + 2], f[8 * r + 3],
                                f[8 * r + 4], f[8 * r + 5], f[8 * r + 6], f[8 * r + 7]};
            mx4_store8(q + n * ldq, s + n * lds, b * kMxBlock + 8 * r, c_in, mx4_codes8(g, scale), scale);
        }
    }
}

// ---- products -----------------------------------------------------------------------
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

// D[channel][row] += sum over 128 of weights x activations: lane l holds channel
// (row) l % 16, block l / 16 of the four, and receives channels (l / 16) * 4 + 0..3
// of row l % 16.  BYTE: which byte of a lane's scales.
template <int BYTE>
__device__ __forceinline__ v4f mfma4(const v4i& w, const v4i& x, const v4f& acc, int sw, int sx) {
    const v8i a = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, b = {x[0], x[1], x[2], x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, BYTE, sw, BYTE, sx);
}

constexpr int kOne = 127;  // the scale of what is not there: its codes are 0

// The scales of blocks b..b+3 of a row of `blocks`, at any alignment.
__device__ __forceinline__ uint32_t scales4(const uint8_t* row, int b, int blocks) {
    if (blocks - b >= 4) return reinterpret_cast<const AnyUint*>(row + b)->v;
    uint32_t v = kOne * 0x01010101u;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < blocks - b) v = (v & ~(255u << (8 * i))) | (uint32_t)row[b + i] << (8 * i);
    return v;
}

// 16 codes' bytes from byte k of a row of K elements, those past its end 0, also
// the upper half of a last byte.
__device__ __forceinline__ v4i codes16(const uint8_t* row, int k, int K) {
    const int bytes = K / 2 + (K & 1);
    v4i v = load16(reinterpret_cast<const int8_t*>(row), k, bytes);
    if ((K & 1) && bytes - 1 >= k && bytes - 1 < k + 16) {
        const int at = bytes - 1 - k;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at / 4 == i) v[i] &= ~(0xf0 << (8 * (at % 4)));
    }
    return v;
}

constexpr int kBK = 128;        // bytes of a row in one LDS tile: 256 elements, 8 blocks
constexpr int kBlocks = kBK / 16;

// A workgroup of WM x WN waves computes BM rows x BN channels.  Operands at any
// alignment pass through registers to LDS; chunk c (a block's 16 bytes) of row r
// lies at chunk c ^ (r & 7), so that the 16 rows of a fragment read at one chunk
// come from different banks.  A lane takes chunks 2 (l / 16) and the next one: its
// two scales are then neighbours too.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void k_mx4_tile(Mx4Args p, int tiles_n) {
    constexpr int kT = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int R = BM + BN, N16 = R * 8 / kT, NS = (R * 2 + kT - 1) / kT;
    static_assert(N16 * kT == R * 8, "chunks divide");
    __shared__ __align__(16) uint8_t lds[R * kBK];
    __shared__ __align__(16) uint8_t scales[R * kBlocks];
    const int tile_m = blockIdx.x / tiles_n, tile_n = blockIdx.x % tiles_n;
    const int64_t m0 = (int64_t)tile_m * BM;
    const int n0 = tile_n * BN;
    const int tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int blocks = p.K / kMxBlock + (p.K % kMxBlock != 0);
    const int bytes = p.K / 2 + (p.K & 1);
    // row r of the tile: an activation row, or a channel
    auto codes_of = [&](int r) -> const uint8_t* {
        if (r < BM) {
            const int64_t m = m0 + r < p.M ? m0 + r : p.M - 1;
            return p.A + m * p.lda;
        }
        const int n = n0 + r - BM < p.N ? n0 + r - BM : p.N - 1;
        return p.B + n * p.ldb;
    };
    auto scales_of = [&](int r) -> const uint8_t* {
        if (r < BM) {
            const int64_t m = m0 + r < p.M ? m0 + r : p.M - 1;
            return p.sa + m * p.ldsa;
        }
        const int n = n0 + r - BM < p.N ? n0 + r - BM : p.N - 1;
        return p.sb + n * p.ldsb;
    };
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    for (int k0 = 0; k0 < bytes; k0 += kBK) {
        v4i raw[N16];
        uint32_t sc[NS];
#pragma unroll
        for (int i = 0; i < N16; ++i) {
            const int at = tid + i * kT;
            raw[i] = codes16(codes_of(at / 8), k0 + at % 8 * 16, p.K);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int at = tid + i * kT;
            sc[i] = at < R * 2 ? scales4(scales_of(at / 2), k0 / 16 + at % 2 * 4, blocks) : 0;
        }
        __syncthreads();  // the previous tile is read
#pragma unroll
        for (int i = 0; i < N16; ++i) {
            const int at = tid + i * kT, r = at / 8;
            *reinterpret_cast<v4i*>(lds + r * kBK + (at % 8 ^ (r & 7)) * 16) = raw[i];
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int at = tid + i * kT;
            if (at < R * 2) *reinterpret_cast<uint32_t*>(scales + at * 4) = sc[i];
        }
        __syncthreads();
        const int r16 = lane & 15, g = lane >> 4;
        int sa[FM], sb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
            sa[i] = *reinterpret_cast<const uint16_t*>(scales + (wm + i * 16 + r16) * kBlocks + g * 2);
#pragma unroll
        for (int j = 0; j < FN; ++j)
            sb[j] = *reinterpret_cast<const uint16_t*>(scales + (BM + wn + j * 16 + r16) * kBlocks + g * 2);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c = ((g * 2 + kk) ^ (r16 & 7)) * 16;
            v4i fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const v4i*>(lds + (wm + i * 16 + r16) * kBK + c);
#pragma unroll
            for (int j = 0; j < FN; ++j)
                fb[j] = *reinterpret_cast<const v4i*>(lds + (BM + wn + j * 16 + r16) * kBK + c);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = kk == 0 ? mfma4<0>(fb[j], fa[i], acc[i][j], sb[j], sa[i])
                                        : mfma4<1>(fb[j], fa[i], acc[i][j], sb[j], sa[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t m = m0 + wm + i * 16 + (lane & 15);
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = n0 + wn + j * 16 + (lane >> 4) * 4 + e;
                if (n >= p.N) continue;
                float v = acc[i][j][e];
                if (p.bias) v += p.bias[n];
                store_elem(p.out, m * p.ldo + n, apply_act(v, p.act), p.out_elem);
            }
    }
}

constexpr int64_t max_blocks(int threads) { return ((int64_t)1 << 32) / threads - 1; }

template <int BM, int BN>
int run_tile(vdttfs_ctx* ctx, const Mx4Args& a) {
    const int64_t tn = (a.N + BN - 1) / BN, blocks = (a.M + BM - 1) / BM * tn;
    k_mx4_tile<BM, BN, 2, 2><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace

int launch_mx4(vdttfs_ctx* ctx, const Mx4Args& a) {
    if (a.M <= 0 || a.N <= 0) return VDTTFS_OK;
    const bool large = (a.M + 63) / 64 * ((a.N + 63) / 64) >= 192;
    const int t = large ? 64 : 32;
    const int64_t rows = max_blocks(256) / ((a.N + t - 1) / t) * t;  // as many a launch as its tiles allow
    for (int64_t m = 0; m < a.M; m += rows) {
        Mx4Args part = a;
        part.A += m * a.lda;
        part.sa += m * a.ldsa;
        part.out = static_cast<char*>(a.out) + m * a.ldo * (a.out_elem == VDTTFS_ELEM_F32 ? 4 : 2);
        part.M = a.M - m < rows ? a.M - m : rows;
        const int rc = large ? run_tile<64, 64>(ctx, part) : run_tile<32, 32>(ctx, part);
        if (rc != VDTTFS_OK) return rc;
    }
    return VDTTFS_OK;
}

int launch_mx4_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, uint8_t* q,
                          int64_t ldq, uint8_t* s, int64_t lds, int cols_zero) {
    if (rows <= 0 || cols_zero <= 0) return VDTTFS_OK;
    const int64_t per = ((int64_t)cols_zero + kMxBlock - 1) / kMxBlock * 4, blocks = (rows * per + 255) / 256;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
    const float tfs = ctx->c.tfs;
    const int T = ctx->c.T;
    if (elem == VDTTFS_ELEM_F32)
        k_mx4_quant<VDTTFS_ELEM_F32><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, cols_zero, tfs, T);
    else if (elem == VDTTFS_ELEM_BF16)
        k_mx4_quant<VDTTFS_ELEM_BF16><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, cols_zero, tfs, T);
    else if (elem == VDTTFS_ELEM_F16)
        k_mx4_quant<VDTTFS_ELEM_F16><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, cols_zero, tfs, T);
    else
        k_mx4_quant<VDTTFS_ELEM_TIMES><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, cols_zero, tfs, T);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_mx4_quant_kernel(vdttfs_ctx* ctx, const float* kernel, int c_in, int c_out, uint8_t* w, int64_t ldw,
                            uint8_t* s, int64_t lds) {
    if (c_out <= 0 || c_in <= 0) return VDTTFS_OK;
    const int blocks = c_in / kMxBlock + (c_in % kMxBlock != 0);
    k_mx4_quant_kernel<<<dim3((unsigned)((c_out + 63) / 64), (unsigned)(blocks < 256 ? (blocks + 3) / 4 : 64)), 256, 0,
                         ctx->stream>>>(kernel, c_in, c_out, w, ldw, s, lds);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
