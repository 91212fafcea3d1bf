// Microscaled rows in 4 bits: quantisation, and products on the matrix cores.
//
// out[m][n] = act(sum_k A[m][k] B[n][k] + bias[n]), A and B elements of e2m1 times
// their blocks' powers of two.  The matrix instruction of 4-bit operands
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes a block of 32 and its scale from each
// lane, so the scales cost no instruction of their own.  Products of two elements
// are multiples of a quarter up to 36, so a block's sum is exact; the sum over
// blocks is in 32-bit floats.
#include <type_traits>

#include "codes.h"
#include "elem.h"
#include "head.h"
#include "mx4.h"
#include "tiles.h"
#include "wave.h"

#ifndef MX4_EARLY
#define MX4_EARLY 0
#define MX4_PER 2
#endif
namespace vdttfs {
namespace {

// ---- quantisation -----------------------------------------------------------------
// The value of a spike time: its linear encoding's pixel.
__device__ __forceinline__ float time_value(float t, float tfs, int T) {
    const int b = arrival_bin(t, tfs, T);
    return b < 0 ? 0.0f : (float)(T - b) / (float)T;
}

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
            for (int i = 0; i < 8; ++i) f[i] = time_value(f[i], tfs, T);
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

// Chunk c (a block's 16 bytes) of row r lies at chunk c ^ swizzle(r) of the row.  A
// lane takes chunks 2 (l / 16) and the next one, so its two scales are neighbours.
// 16-byte reads are served in groups of 16 lanes, {0-3, 12-15, 20-23, 24-27} and so
// on, over 256 bytes of banks: with these two bits of the row all 16 come from
// different banks (with r & 7 in their place every other one collided: 26 M cycles
// of conflicts in 8192 x 8192 x 8192, and 300 us).
__device__ __forceinline__ int swizzle(int r) { return (r >> 1 & 1) | (r & 4); }

// A workgroup of WM x WN waves computes BM rows x BN channels.  Operands at any
// alignment pass through registers to LDS.
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
            *reinterpret_cast<v4i*>(lds + r * kBK + (at % 8 ^ swizzle(r)) * 16) = raw[i];
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
            const int c = ((g * 2 + kk) ^ swizzle(r16)) * 16;
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

// A wave's sums to its outputs.  A lane has four neighbouring channels of a row;
// stored from there, a wave would write 32 bytes of each of 16 rows at a time.  So
// two fragments of rows at a time pass through the wave's own part of LDS (16-byte
// chunk c of row r at chunk c ^ r), and leave eight neighbours a lane, a row's
// outputs together.  The loop over rows is one piece of code for all types, ends and
// activations: unrolled for each, a tile's end took 9.5 us, most of it instructions
// on their way.  nw: the wave's first channel.
template <int FM, int FN>
struct Stage {
    static constexpr int kFrags = FM > 1 ? 2 : 1, kRows = kFrags * 16, kCols = FN * 16;
    static constexpr int kBytes = kRows * kCols * 4;
};
template <int FM, int FN>
__device__ __forceinline__ void epilogue(const Mx4Args& p, const v4f (&acc)[FM][FN], int64_t m0, int nw, float* stage) {
    typedef Stage<FM, FN> S;
    constexpr int kChunks = S::kCols / 4, kLanes = S::kCols / 8, kPass = 64 / kLanes;  // lanes of a row, rows of a pass
    const int lane = lane_id(), c = lane % kLanes * 8, left = p.N - nw - c;
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = p.bias && e < left ? p.bias[nw + c + e] : 0.0f;
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += S::kFrags) {
        const int64_t mi = m0 + i0 * 16;
        if (mi >= p.M) return;
#pragma unroll
        for (int i = 0; i < S::kFrags; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int r = i * 16 + (lane & 15), at = (j * 4 + (lane >> 4)) ^ (r & (kChunks - 1));
                *reinterpret_cast<v4f*>(stage + r * S::kCols + at * 4) = acc[i0 + i][j];
            }
        wave_sync();
#pragma unroll 1
        for (int r = lane / kLanes; r < S::kRows; r += kPass) {
            if (mi + r >= p.M || left <= 0) break;
            const int x = r & (kChunks - 1);
            const v4f lo = *reinterpret_cast<const v4f*>(stage + r * S::kCols + ((c / 4) ^ x) * 4);
            const v4f hi = *reinterpret_cast<const v4f*>(stage + r * S::kCols + ((c / 4 + 1) ^ x) * 4);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            if (p.act == VDTTFS_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = apply_act(v[e], VDTTFS_ACT_RELU);
            } else if (p.act == VDTTFS_ACT_SILU) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = apply_act(v[e], VDTTFS_ACT_SILU);
            }
            const int64_t o = (mi + r) * p.ldo + nw + c;
            if (left >= 8) {
                put8(p.out, o, p.out_elem, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < left) store_elem(p.out, o + e, v[e], p.out_elem);
            }
        }
        wave_sync();
    }
}

// The large product: tiles of 128 bytes a row and the 8 scales of their blocks go
// from memory to LDS directly (16 and 4 bytes a lane, no registers between).  Rows
// of codes on 16 bytes, of scales on 4.  The last K % 256 elements come through
// registers with zeros behind them.
template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(WM* WN * 64, WM* WN == 4 && BM == 256 ? 1 : 2) void k_mx4_big(Mx4Args p, int tiles_m,
                                                                                          int tiles_n) {
    constexpr int kW = WM * WN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int NA = BM / 8 / kW, NB = BN / 8 / kW;  // loads of codes of a wave and tile, 8 rows each
    constexpr int kScaleLoads = (BM + BN) / 32, NS = (kScaleLoads + kW - 1) / kW;
    constexpr int NL = NA + NB + (S > 2 ? NS : 0);
    constexpr int kCodes = (BM + BN) * kBK, kTile = kCodes + (S > 2 ? (BM + BN) * kBlocks : 0);
    // two stages: the scales of four tiles at a time, 32 bytes a row, two deep
    constexpr int kSpan = 4, kRowScales = S > 2 ? kBlocks : kSpan * kBlocks, kScales = (BM + BN) * kRowScales;
    static_assert(NA * kW * 8 == BM && NB * kW * 8 == BN && BM % 32 == 0 && BN % 32 == 0, "loads divide");
    static_assert(S >= 2 && S <= 4 && (S - 2) * NL < 64, "stages");
    constexpr int kStage = kW * Stage<FM, FN>::kBytes;
    // an array for each stage: only then does the compiler see that reads of
    // one need not wait for loads into another
    __shared__ __align__(16) uint8_t s0[kTile > kStage ? kTile : kStage];
    __shared__ __align__(16) uint8_t s1[kTile];
    __shared__ __align__(16) uint8_t s2[S > 2 ? kTile : 16];
    __shared__ __align__(16) uint8_t s3[S > 3 ? kTile : 16];
    __shared__ __align__(16) uint8_t spans[S > 2 ? 16 : 2 * kScales];

    int tile_m, tile_n;
    if (!tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, &tile_m, &tile_n)) return;
    const int64_t m0 = (int64_t)tile_m * BM;
    const int n0 = tile_n * BN;
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6);
    const int lrow = lane / 8, chunk = (lane % 8 ^ swizzle(lrow)) * 16;
    // A lane's loads by their offsets from the tile's first row (below 2^31:
    // kMaxLd), so that their addresses take a register each and scalar steps in K.
    const uint8_t *A = p.A + m0 * p.lda, *B = p.B + n0 * p.ldb, *SA = p.sa + m0 * p.ldsa, *SB = p.sb + n0 * p.ldsb;
    const unsigned lda = (unsigned)p.lda, ldb = (unsigned)p.ldb;
    const int last_a = p.M - m0 < BM ? (int)(p.M - m0) - 1 : BM - 1, last_b = p.N - n0 < BN ? p.N - n0 - 1 : BN - 1;
    unsigned from[NA + NB], sfrom[NS];  // of codes, of scales (two lanes a row)
#pragma unroll
    for (int i = 0; i < NA; ++i) from[i] = min((wave * NA + i) * 8 + lrow, last_a) * lda + chunk;
#pragma unroll
    for (int i = 0; i < NB; ++i) from[NA + i] = min((wave * NB + i) * 8 + lrow, last_b) * ldb + chunk;
    // a wave's load of scales is of A's rows or of B's; past the last: again the
    // first ones, the same bytes
    auto s_load = [&](int i) __attribute__((always_inline)) { return (wave * NS + i) % kScaleLoads; };
    auto of_a = [&](int i) __attribute__((always_inline)) { return s_load(i) * 32 < BM; };
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int r = s_load(i) * 32 + lane / 2;
        sfrom[i] = of_a(i) ? min(r, last_a) * (unsigned)p.ldsa : min(r - BM, last_b) * (unsigned)p.ldsb;
    }
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int r16 = lane & 15, g4 = lane >> 4;
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0, 0, 0, 0};

    const int tiles = p.K / 256;
    // one of a wave's NL loads of tile t; past the end the last tile's, not used
    auto fetch_one = [&](uint8_t* s, int t, int l) __attribute__((always_inline)) {
        t = t < tiles ? t : tiles - 1;
        if (l < NA + NB) {
            const int at = l < NA ? wave * NA + l : BM / 8 + wave * NB + l - NA;
            to_lds16(l < NA ? A : B, from[l < NA + NB ? l : 0], t * kBK, s + at * 1024);
        } else {
            const int i = l < NA + NB ? 0 : l - NA - NB;
            to_lds4(of_a(i) ? SA : SB, sfrom[i] + (lane & 1) * 4, t * kBlocks, s + kCodes + s_load(i) * 256);
        }
    };
    auto fetch = [&](uint8_t* s, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int l = 0; l < NL; ++l) fetch_one(s, t, l);
    };
    // The scales of tiles 4 n .. 4 n + 3: 16 bytes a lane; where there are fewer
    // tiles, 4 bytes a lane, those past them the row's first again, not used.  (Of 8
    // bytes of a row in every tile, a wave's load touched 32 lines for 256 bytes:
    // 8192 x 8192 x 8192 took 276 us.)
    auto fetch_span = [&](int n) __attribute__((always_inline)) {
        uint8_t* to = spans + (n & 1) * kScales;
        if ((n + 1) * kSpan <= tiles) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                to_lds16(of_a(i) ? SA : SB, sfrom[i] + (lane & 1) * 16, n * kSpan * kBlocks, to + s_load(i) * 1024);
        } else {
            const int there = (tiles - n * kSpan) * 2, d = lane % 8 < there ? lane % 8 : 0;
            for (int i = wave; i < (BM + BN) / 8; i += kW) {
                const int r = i * 8 + lane / 8;
                const bool a = i * 8 < BM;
                to_lds4(a ? SA : SB, (a ? min(r, last_a) * (unsigned)p.ldsa : min(r - BM, last_b) * (unsigned)p.ldsb) + d * 4,
                        n * kSpan * kBlocks, to + i * 256);
            }
        }
    };
    // Each group is one row fragment against all channel fragments; fragments are
    // read two groups (channels: one k step) ahead.
    constexpr int G = 2 * FM;
    // Where a lane's fragments and scales start in a stage.  Opaque, so that every
    // read is one of these registers and an immediate: the compiler else makes
    // addresses of all of them, more than there are registers.
    auto place = [&](int kk) __attribute__((always_inline)) { return ((g4 * 2 + kk) ^ swizzle(r16)) * 16; };
    int oa[2] = {(wm + r16) * kBK + place(0), (wm + r16) * kBK + place(1)};
    int ob[2] = {(BM + wn + r16) * kBK + place(0), (BM + wn + r16) * kBK + place(1)};
    int osa = (wm + r16) * kRowScales + g4 * 2, osb = (BM + wn + r16) * kRowScales + g4 * 2;
    asm volatile("" : "+v"(oa[0]), "+v"(oa[1]), "+v"(ob[0]), "+v"(ob[1]), "+v"(osa), "+v"(osb));
    auto code_a = [&](const uint8_t* s, int g) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4i*>(s + oa[g / FM] + g % FM * 16 * kBK);
    };
    auto code_b = [&](const uint8_t* s, int kk, int j) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4i*>(s + ob[kk] + j * 16 * kBK);
    };
    auto scale_a = [&](const uint8_t* s, int i) __attribute__((always_inline)) {
        return (int)*reinterpret_cast<const uint16_t*>(s + osa + i * 16 * kRowScales);
    };
    auto scale_b = [&](const uint8_t* s, int j) __attribute__((always_inline)) {
        return (int)*reinterpret_cast<const uint16_t*>(s + osb + j * 16 * kRowScales);
    };
    // One tile multiplied, with the loads of tile t (to `next`) spread between: a
    // wave that issues its loads in one go waits for the address unit, and its
    // matrix instructions with it.
    auto multiply = [&](auto with_loads, const uint8_t* s, const uint8_t* sc, uint8_t* next, int t)
                        __attribute__((always_inline)) {
        v4i fa[3], fb[2][FN];
        int sa[FM], sb[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = scale_b(sc, j);
        sa[0] = scale_a(sc, 0);
        fa[0] = code_a(s, 0);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[0][j] = code_b(s, 0, j);
        if (FM > 1) sa[FM > 1 ? 1 : 0] = scale_a(sc, 1);
        fa[1] = code_a(s, 1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int kk = g / FM, i = g % FM;
            if (g + 2 < G) fa[(g + 2) % 3] = code_a(s, g + 2);
            if (g + 2 < FM) sa[g + 2 < FM ? g + 2 : 0] = scale_a(sc, g + 2);
            if (kk == 0) {
#pragma unroll
                for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) fb[1][j] = code_b(s, 1, j);
            }
            if constexpr (with_loads.value) {
#pragma unroll
                for (int l = 0; l < NL; ++l)
                    if (l * G / NL == g) fetch_one(next, t, l);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = kk == 0 ? mfma4<0>(fb[0][j], fa[g % 3], acc[i][j], sb[j], sa[i])
                                    : mfma4<1>(fb[1][j], fa[g % 3], acc[i][j], sb[j], sa[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Tile t is in s; the loads of tile t + S - 1 go to `next`, whose tile every
    // wave has read before the barrier.  No branch between loads and waits, so the
    // number in flight is known everywhere.
    auto step = [&](const uint8_t* s, uint8_t* next, int t) __attribute__((always_inline)) {
        wait_loads<(S - 2) * NL>();
        barrier();
        multiply(std::true_type{}, s, s + kCodes, next, t + S - 1);
    };
    if constexpr (S == 2) {
        // Two stages, the barrier before a tile's last two groups: by then all its
        // fragments are in registers, so the next tile's first ones are read, and
        // the loads of the one after that are issued into its LDS, while the matrix
        // instructions go on.
        static_assert(G % 4 == 0 && FM >= 4, "the ring of fragments comes round with the tile");
        v4i fa[4], fb[2][FN];
        int sa[2][FM], sb[2][FN];
        // Tile t's first fragments and all its scales, where no load is in flight (as
        // one into `spans` may be later, the compiler would wait for it)
        auto first = [&](auto turn, const uint8_t* s, int t) __attribute__((always_inline)) {
            const uint8_t* sc = spans + (t / kSpan & 1) * kScales + t % kSpan * kBlocks;
            fa[0] = code_a(s, 0);
            sa[turn.value][0] = scale_a(sc, 0);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                fb[0][j] = code_b(s, 0, j);
                sb[turn.value][j] = scale_b(sc, j);
            }
            fa[1] = code_a(s, 1);
#pragma unroll
            for (int i = 1; i < FM; ++i) sa[turn.value][i] = scale_a(sc, i);
        };
        // A tile's first kEarly loads go out behind the barrier that frees its LDS,
        // the others between the first groups of the next tile: all at once they
        // hold up the fragment reads.
        constexpr int kEarly = MX4_EARLY, kPer = MX4_PER;
        static_assert(kEarly + kPer * (G - 2) >= NL, "all loads go out");
        auto run = [&](auto turn, uint8_t* s, uint8_t* next, int t) __attribute__((always_inline)) {
            constexpr int kTurn = turn.value;
            if (kTurn == 0 && t % kSpan == 0 && t + kSpan < tiles) fetch_span(t / kSpan + 1);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int kk = g / FM, i = g % FM;
                if (g + 2 < G) fa[(g + 2) % 4] = code_a(s, g + 2);
                if (kk == 0) {
#pragma unroll
                    for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) fb[1][j] = code_b(s, 1, j);
                }
                if (g == G - 2) {
                    wait_loads<0>();
                    barrier();
                    first(std::integral_constant<int, 1 - kTurn>{}, next, t + 1);
                }
                if (kEarly > 0 && g >= G - 2) fetch_one(s, t + 2, g - (G - 2));
                else
#pragma unroll
                    for (int l = kEarly + g * kPer; l < kEarly + (g + 1) * kPer && l < NL; ++l)
                        fetch_one(next, t + 1, l);
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = kk == 0 ? mfma4<0>(fb[0][j], fa[g % 4], acc[i][j], sb[kTurn][j], sa[kTurn][i])
                                        : mfma4<1>(fb[1][j], fa[g % 4], acc[i][j], sb[kTurn][j], sa[kTurn][i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // at least two tiles (deep_ok)
        fetch_span(0);
        fetch(s0, 0);
        wait_loads<0>();
        barrier();
        first(std::integral_constant<int, 0>{}, s0, 0);
#pragma unroll
        for (int l = 0; l < kEarly; ++l) fetch_one(s1, 1, l);
        int t = 0;
        for (; t + 2 <= tiles; t += 2) {
            run(std::integral_constant<int, 0>{}, s0, s1, t);
            run(std::integral_constant<int, 1>{}, s1, s0, t + 1);
        }
        if (t < tiles) run(std::integral_constant<int, 0>{}, s0, s1, t);
    } else if (tiles == 1) {  // nothing to load ahead
        fetch(s0, 0);
        wait_loads<0>();
        barrier();
        multiply(std::false_type{}, s0, s0 + kCodes, s0, 0);
    } else if (tiles > 1) {
        fetch(s0, 0);
        fetch(s1, 1);
        if (S > 3) fetch(s2, 2);
        int t = 0;
        for (; t + S <= tiles; t += S) {
            step(s0, S == 3 ? s2 : s3, t);
            step(s1, s0, t + 1);
            step(s2, s1, t + 2);
            if (S > 3) step(s3, s2, t + 3);
        }
        // the last tiles % S are in flight
        wait_loads<0>();
        barrier();
        if (t < tiles) multiply(std::false_type{}, s0, s0 + kCodes, s0, 0);
        if (t + 1 < tiles) multiply(std::false_type{}, s1, s1 + kCodes, s1, 0);
        if (S > 3 && t + 2 < tiles) multiply(std::false_type{}, s2, s2 + kCodes, s2, 0);
    }
    wait_loads<0>();  // also those past the end
    if (p.K % 256) {
        const int k0 = tiles * kBK, blocks = p.K / kMxBlock + (p.K % kMxBlock != 0);
        uint8_t* sc = S > 2 ? s0 + kCodes : spans;
        v4i end[NA + NB];
        uint32_t ends[NS];
#pragma unroll
        for (int l = 0; l < NA + NB; ++l) end[l] = codes16((l < NA ? A : B) + (from[l] - chunk), k0 + chunk, p.K);
#pragma unroll
        for (int l = 0; l < NS; ++l)
            ends[l] = scales4((of_a(l) ? SA : SB) + sfrom[l], k0 / 16 + (lane & 1) * 4, blocks);
        __syncthreads();
#pragma unroll
        for (int l = 0; l < NA + NB; ++l)
            *reinterpret_cast<v4i*>(s0 + (l < NA ? wave * NA + l : BM / 8 + wave * NB + l - NA) * 1024 + lane * 16) = end[l];
#pragma unroll
        for (int l = 0; l < NS; ++l)
            *reinterpret_cast<uint32_t*>(sc + (s_load(l) * 32 + lane / 2) * kRowScales + (lane & 1) * 4) = ends[l];
        __syncthreads();
        multiply(std::false_type{}, s0, sc, s0, 0);
    }
    barrier();  // the stage takes the tiles' place
    epilogue<FM, FN>(p, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(s0) + wave * (Stage<FM, FN>::kBytes / 4));
}

// ---- few rows -------------------------------------------------------------------------
// A workgroup has 16 channels, its eight waves share K in spans of 512 elements, and
// the sums meet in LDS: bound by the weights, which are read once, straight to
// registers.  Of a span a lane takes 64 neighbouring bytes of a channel (blocks 4 g ..
// 4 g + 3, g = lane / 16) and their four scales.  Activations: up to 16 rows of codes
// in memory (ELEM kElemCodes), read alike (of 17 rows the smallest tiles take as long,
// of 64 x 8192 x 8192 16 us for 28); or of floats or spike times, quantised by every
// workgroup into LDS while its weights are on their way, where that is no more than
// eight runs of eight a thread (4 x 4096 x 4096 from BF16 5.5 us, 8.0 with a launch of
// its own for that; 8 x 4096 x 4096 7.4 and 7.9).
constexpr int kSpanBlocks = 16, kSmallWaves = 8, kSmallRows = 16, kSmallRuns = 8;
struct Span {
    v4i c[4];
    int s;
};
__device__ __forceinline__ Span load_span(const uint8_t* codes, const uint8_t* scales, int span, int g, int K) {
    Span r;
    const int b = span * kSpanBlocks + g * 4;
    if (K - span * 512 >= 512) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.c[i] = reinterpret_cast<const Bytes16*>(codes + (b + i) * 16)->v;
        r.s = (int)reinterpret_cast<const AnyUint*>(scales + b)->v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.c[i] = codes16(codes, (b + i) * 16, K);
        r.s = (int)scales4(scales, b, K / kMxBlock + (K % kMxBlock != 0));
    }
    return r;
}
template <int ELEM>
__global__ __launch_bounds__(kSmallWaves * 64) void k_mx4_small(Mx4Args p, const void* __restrict__ x, int64_t ldx,
                                                                float tfs, int T) {
    constexpr bool kCodesIn = ELEM == kElemCodes;
    constexpr int kQuant = kCodesIn ? 16 : kSmallRuns * kSmallWaves * 64 * 4;  // bytes of codes
    __shared__ float part[kSmallWaves][kSmallRows][16 + 1];
    __shared__ __align__(16) uint8_t q[kQuant];
    __shared__ __align__(4) uint8_t qs[kCodesIn ? 16 : kQuant / 16];
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;
    const uint8_t *wc = p.B + (int64_t)n * p.ldb, *ws = p.sb + (int64_t)n * p.ldsb;
    const int spans = p.K / 512 + (p.K % 512 != 0), M = (int)p.M;
    Span w{};
    if (wave < spans) w = load_span(wc, ws, wave, g, p.K);
    if constexpr (!kCodesIn) {
        // runs of eight to codes; blocks past the row's end to codes of 0
        const int per = spans * kSpanBlocks * 4;
        for (int at = threadIdx.x; at < M * per; at += kSmallWaves * 64) {
            const int m = at / per, c = (at - m * per) * 8, b = c / kMxBlock;
            float f[8];
            load8<ELEM>(x, m * ldx, c, p.K, f);
            if constexpr (ELEM == VDTTFS_ELEM_TIMES) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = time_value(f[i], tfs, T);
            }
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max(most, magnitude(f[i]));
            const int scale = mx4_scale(quad_max(most));
            // a span's 16 chunks at 16 places by the row, for the fragments' reads
            const int to = m * spans * kSpanBlocks + (b ^ m);
            *reinterpret_cast<uint32_t*>(q + to * 16 + c % kMxBlock / 2) = mx4_codes8(f, scale);
            if (c % kMxBlock == 0) qs[m * spans * kSpanBlocks + b] = (uint8_t)scale;
        }
        __syncthreads();
    }
    v4f acc = {0, 0, 0, 0};
    const int row = r16 < M ? r16 : M - 1;
    for (int span = wave; span < spans; span += kSmallWaves) {
        Span a;
        if constexpr (kCodesIn) {
            a = load_span(p.A + row * p.lda, p.sa + row * p.ldsa, span, g, p.K);
        } else {
            const int b = row * spans * kSpanBlocks;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a.c[i] = *reinterpret_cast<const v4i*>(q + (b + ((span * kSpanBlocks + g * 4 + i) ^ row)) * 16);
            a.s = *reinterpret_cast<const int*>(qs + b + span * kSpanBlocks + g * 4);
        }
        Span next{};
        if (span + kSmallWaves < spans) next = load_span(wc, ws, span + kSmallWaves, g, p.K);
        acc = mfma4<0>(w.c[0], a.c[0], acc, w.s, a.s);
        acc = mfma4<1>(w.c[1], a.c[1], acc, w.s, a.s);
        acc = mfma4<2>(w.c[2], a.c[2], acc, w.s, a.s);
        acc = mfma4<3>(w.c[3], a.c[3], acc, w.s, a.s);
        w = next;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][r16][g * 4 + e] = acc[e];
    __syncthreads();
    const int m = threadIdx.x / 16, c = threadIdx.x % 16;
    if (m >= M || n0 + c >= p.N) return;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kSmallWaves; ++i) v += part[i][m][c];
    if (p.bias) v += p.bias[n0 + c];
    store_elem(p.out, (int64_t)m * p.ldo + n0 + c, apply_act(v, p.act), p.out_elem);
}

template <int ELEM>
int run_small(vdttfs_ctx* ctx, const Mx4Args& a, const void* x, int64_t ldx) {
    k_mx4_small<ELEM><<<dim3((unsigned)((a.N + 15) / 16)), kSmallWaves * 64, 0, ctx->stream>>>(a, x, ldx, ctx->c.tfs,
                                                                                               ctx->c.T);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

template <int BM, int BN>
int run_tile(vdttfs_ctx* ctx, const Mx4Args& a) {
    const int64_t tn = (a.N + BN - 1) / BN, blocks = (a.M + BM - 1) / BM * tn;
    k_mx4_tile<BM, BN, 2, 2><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace

// Rows that loads to LDS can take.
constexpr int64_t kMaxLd = 1 << 22;  // 256 rows of them below 2^31 bytes
static bool aligned(const Mx4Args& a) {
    return a.lda <= kMaxLd && a.ldb <= kMaxLd && a.ldsa <= kMaxLd && a.ldsb <= kMaxLd && (((uintptr_t)a.A | (uintptr_t)a.B | (uintptr_t)a.lda | (uintptr_t)a.ldb) & 15) == 0 &&
           (((uintptr_t)a.sa | (uintptr_t)a.sb | (uintptr_t)a.ldsa | (uintptr_t)a.ldsb) & 3) == 0;
}

template <int BM, int BN, int WM, int WN, int S>
static int run_big(vdttfs_ctx* ctx, const Mx4Args& a) {
    const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    k_mx4_big<BM, BN, WM, WN, S><<<dim3((unsigned)(tm * tn)), WM * WN * 64, 0, ctx->stream>>>(a, (int)tm, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

struct Mx4Tile {
    int bm, bn;
};
static Mx4Tile tile_for(int64_t M, int N, int K, bool is_aligned) {
    auto tiles = [&](int bm, int bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); };
    if (!is_aligned) return tiles(64, 64) >= 192 ? Mx4Tile{64, 64} : Mx4Tile{32, 32};
    const int64_t big = tiles(256, 256), rounds = (big + 255) / 256;
    const bool deep = K >= 512;
    if (deep && (rounds == 1 ? big >= 160 : big * 10 >= rounds * 256 * 7)) return Mx4Tile{256, 256};
    if (deep && tiles(128, 128) >= 384) return Mx4Tile{128, 128};
    return tiles(64, 64) >= 192 ? Mx4Tile{64, 64} : Mx4Tile{32, 32};
}

#ifndef MX4_BIG
#define MX4_BIG 2, 4
#endif
// Whether rows of floats or spike times are quantised by their product.
bool mx4_small_linear_ok(int64_t M, int K) {
    const int64_t per = ((int64_t)K + 511) / 512 * 64;  // runs of eight of a row, whole spans
    return M <= kSmallRows && K > 0 && M * per <= kSmallRuns * kSmallWaves * 64;
}
int launch_mx4_small_linear(vdttfs_ctx* ctx, const Mx4Args& a, const void* x, int elem, int64_t ldx) {
    if (elem == VDTTFS_ELEM_F32) return run_small<VDTTFS_ELEM_F32>(ctx, a, x, ldx);
    if (elem == VDTTFS_ELEM_BF16) return run_small<VDTTFS_ELEM_BF16>(ctx, a, x, ldx);
    if (elem == VDTTFS_ELEM_F16) return run_small<VDTTFS_ELEM_F16>(ctx, a, x, ldx);
    return run_small<VDTTFS_ELEM_TIMES>(ctx, a, x, ldx);
}

int launch_mx4(vdttfs_ctx* ctx, const Mx4Args& a) {
    if (a.M <= 0 || a.N <= 0) return VDTTFS_OK;
    if (a.M <= kSmallRows) return run_small<kElemCodes>(ctx, a, nullptr, 0);
    const bool fast = aligned(a);
    const Mx4Tile t = tile_for(a.M, a.N, a.K, fast);
    const int64_t rows = max_blocks(512) / ((a.N + t.bn - 1) / t.bn) * t.bm;  // as many a launch as its tiles allow
    for (int64_t m = 0; m < a.M; m += rows) {
        Mx4Args part = a;
        part.A += m * a.lda;
        part.sa += m * a.ldsa;
        part.out = static_cast<char*>(a.out) + m * a.ldo * (a.out_elem == VDTTFS_ELEM_F32 ? 4 : 2);
        part.M = a.M - m < rows ? a.M - m : rows;
        int rc;
        if (!fast) rc = t.bm == 64 ? run_tile<64, 64>(ctx, part) : run_tile<32, 32>(ctx, part);
        else if (t.bm == 256) rc = run_big<256, 256, MX4_BIG, 2>(ctx, part);
        else if (t.bm == 128) rc = run_big<128, 128, 2, 2, 2>(ctx, part);
        else rc = t.bm == 64 ? run_big<64, 64, 2, 2, 4>(ctx, part) : run_big<32, 32, 2, 2, 4>(ctx, part);
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
