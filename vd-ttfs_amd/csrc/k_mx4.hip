// Microscaled rows in 4 bits: quantisation, and products on the matrix cores.
//
// out[m][n] = act(sum_k A[m][k] B[n][k] + bias[n]), A and B elements of e2m1 times
// their blocks' powers of two.  The matrix instruction of 4-bit operands
// (v_mfma_scale_f32_16x16x128_f8f6f4) takes a block of 32 and its scale from each
// lane, so the scales cost no instruction of their own.  Products of two elements
// are multiples of a quarter up to 36, so a block's sum is exact; the sum over
// blocks is in 32-bit floats.
#include <algorithm>
#include <type_traits>

#include "codes.h"
#include "elem.h"
#include "head.h"
#include "mx4.h"
#include "tiles.h"
#include "wave.h"

namespace vdttfs {
namespace {

// ---- quantisation -----------------------------------------------------------------
// The value of a spike time: its linear encoding's pixel.
__device__ __forceinline__ float time_value(float t, float tfs, int T) {
    const int b = arrival_bin(t, tfs, T);
    return b < 0 ? 0.0f : (float)(T - b) / (float)T;
}

// Eight values a thread, four neighbouring threads a block of 32.  Bound by memory: 8192
// x 4096 BF16 17 us, 85 MB at 5.0 TB/s.
template <int ELEM>
__global__ __launch_bounds__(256) void k_mx4_quant(const void* __restrict__ x, int64_t ldx, int64_t rows, int cols,
                                                   uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ s,
                                                   int64_t lds, float tfs, int T) {
    const int64_t per = ((int64_t)cols + kMxBlock - 1) / kMxBlock * 4;  // runs of eight in a row
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
        mx4_store8(q + m * ldq, s + m * lds, c, cols, mx4_codes8(f, scale), scale);
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

// The scales of blocks b and b + 1.
struct __attribute__((packed, aligned(1))) AnyShort {
    uint16_t v;
};
__device__ __forceinline__ int scales2(const uint8_t* row, int b, int blocks) {
    if (blocks - b >= 2) return reinterpret_cast<const AnyShort*>(row + b)->v;
    return b < blocks ? row[b] | kOne << 8 : kOne * 0x101;
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

// A workgroup of WM x WN waves computes BM rows x BN channels, operands at any
// alignment: codes pass through registers to LDS, the next tile's on their way while
// one is multiplied; a lane loads its fragments' scales itself.  Two barriers a step, so
// for what is not worth a copy or has few steps: 333 x 1111 x 1003 6.4 us, of which a
// launch is 4.5 (mx4_plan has what it takes beside the others).
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64) void k_mx4_tile(Mx4Args p, int tiles_n) {
    constexpr int kT = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int R = BM + BN, NL = R * 8 / kT;
    static_assert(NL * kT == R * 8, "chunks divide");
    constexpr int kStage = WM * WN * Stage<FM, FN>::kBytes;
    __shared__ __align__(16) uint8_t lds[R * kBK > kStage ? R * kBK : kStage];
    const int tile_m = blockIdx.x / tiles_n, tile_n = blockIdx.x % tiles_n;
    const int64_t m0 = (int64_t)tile_m * BM;
    const int n0 = tile_n * BN;
    const int tid = threadIdx.x, lane = lane_id(), wave = uniform(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int blocks = p.K / kMxBlock + (p.K % kMxBlock != 0);
    const int bytes = p.K / 2 + (p.K & 1);
    auto a_row = [&](int r) { return m0 + r < p.M ? m0 + r : p.M - 1; };
    auto b_row = [&](int r) { return (int64_t)(n0 + r < p.N ? n0 + r : p.N - 1); };
    const uint8_t* from[NL];  // row r of the tile: an activation row, or a channel
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int r = (tid + i * kT) / 8;
        from[i] = r < BM ? p.A + a_row(r) * p.lda : p.B + b_row(r - BM) * p.ldb;
    }
    const uint8_t *sfa[FM], *sfb[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) sfa[i] = p.sa + a_row(wm + i * 16 + r16) * p.ldsa;
#pragma unroll
    for (int j = 0; j < FN; ++j) sfb[j] = p.sb + b_row(wn + j * 16 + r16) * p.ldsb;
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
    v4i raw[NL];
    int na[FM], nb[FN];
    auto fetch = [&](int k0) {
        if (p.K - k0 * 2 >= 2 * kBK) {
#pragma unroll
            for (int i = 0; i < NL; ++i) raw[i] = reinterpret_cast<const Bytes16*>(from[i] + k0 + (tid & 7) * 16)->v;
        } else {
#pragma unroll
            for (int i = 0; i < NL; ++i) raw[i] = codes16(from[i], k0 + (tid & 7) * 16, p.K);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) na[i] = scales2(sfa[i], k0 / 16 + g * 2, blocks);
#pragma unroll
        for (int j = 0; j < FN; ++j) nb[j] = scales2(sfb[j], k0 / 16 + g * 2, blocks);
    };
    if (bytes > 0) fetch(0);
    for (int k0 = 0; k0 < bytes; k0 += kBK) {
        __syncthreads();  // the previous tile is read
        int sa[FM], sb[FN];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int r = (tid + i * kT) / 8;
            *reinterpret_cast<v4i*>(lds + r * kBK + ((tid & 7) ^ swizzle(r)) * 16) = raw[i];
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = na[i];
#pragma unroll
        for (int j = 0; j < FN; ++j) sb[j] = nb[j];
        __syncthreads();
        if (k0 + kBK < bytes) fetch(k0 + kBK);
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
    __syncthreads();
    epilogue<FM, FN>(p, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(lds) + wave * (Stage<FM, FN>::kBytes / 4));
}

// The large product: tiles of 128 bytes a row go from memory to LDS directly (16
// bytes a lane, no registers between), S deep.  Rows of codes on 16 bytes.  Of two
// stages the scales go to LDS too, those of four tiles at a time, of rows on 4 bytes;
// of more a lane loads those of its fragments, of any alignment, and holds them until
// their tile.  The last K % 256 elements come through registers with zeros behind them.
//
// 8192 x 4096 x 4096 from BF16's codes 71 to 77 us by the card (3.6 to 3.9 POP/s), 8192 x
// 8192 x 8192 249 to 262.  A tile of 256 x 256 takes 2 us to its first step, 1.75 a step
// of 256, and 6 to its outputs.  A step's matrix instructions alone take 1.24 us on random
// codes and 1.0 on zeros, as their power takes the clock from 2.37 GHz to 1.74; a step's
// 192 KB of reads and 64 KB of writes of LDS take it as many cycles, not all beside them.
// Halves of the waves in turn, one multiplying while the other loads: 80 and 267 us.
template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_mx4_big(Mx4Args p, int tiles_m, int tiles_n) {
    constexpr int kW = WM * WN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int NA = BM / 8 / kW, NB = BN / 8 / kW;  // loads of codes of a wave and tile, 8 rows each
    constexpr int kScaleLoads = (BM + BN) / 32, NS = (kScaleLoads + kW - 1) / kW;
    constexpr int NL = NA + NB + (S > 2 ? FM + FN : 0);  // loads of a wave and tile
    constexpr int kCodes = (BM + BN) * kBK, kTile = kCodes;
    constexpr int kSpan = 4, kRowScales = kSpan * kBlocks, kScales = (BM + BN) * kRowScales;
    static_assert(NA * kW * 8 == BM && NB * kW * 8 == BN && BM % 32 == 0 && BN % 32 == 0, "loads divide");
    static_assert((S == 2 || S == 4) && (S - 2) * NL < 64, "stages");
    constexpr int kStage = kW * Stage<FM, FN>::kBytes;
    // an array for each stage: only then does the compiler see that reads of
    // one need not wait for loads into another
    __shared__ __align__(16) uint8_t s0[kTile > kStage ? kTile : kStage];
    __shared__ __align__(16) uint8_t s1[kTile];
    __shared__ __align__(16) uint8_t s2[S > 2 ? kTile : 16];
    __shared__ __align__(16) uint8_t s3[S > 2 ? kTile : 16];
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
    unsigned from[NA + NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) from[i] = min((wave * NA + i) * 8 + lrow, last_a) * lda + chunk;
#pragma unroll
    for (int i = 0; i < NB; ++i) from[NA + i] = min((wave * NB + i) * 8 + lrow, last_b) * ldb + chunk;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int r16 = lane & 15, g4 = lane >> 4;
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0, 0, 0, 0};

    const int tiles = p.K / 256;  // at least two: from 512 elements on (mx4_plan)
    // The scales of a lane's fragments: two bytes of each row and channel.
    struct Scales {
        int a[FM], b[FN];
    };
    unsigned sfa[FM], sfb[FN];  // where they start
#pragma unroll
    for (int i = 0; i < FM; ++i) sfa[i] = min(wm + i * 16 + r16, last_a) * (unsigned)p.ldsa + g4 * 2;
#pragma unroll
    for (int j = 0; j < FN; ++j) sfb[j] = min(wn + j * 16 + r16, last_b) * (unsigned)p.ldsb + g4 * 2;
    // one of a wave's NL loads of tile t, of scales to sc; past the end the last
    // tile's, not used
    auto fetch_one = [&](uint8_t* s, Scales& sc, int t, int l) __attribute__((always_inline)) {
        t = t < tiles ? t : tiles - 1;
        if (l < NA + NB) {
            const int at = l < NA ? wave * NA + l : BM / 8 + wave * NB + l - NA;
            to_lds16(l < NA ? A : B, from[l < NA + NB ? l : 0], t * kBK, s + at * 1024);
        } else {
            const int i = l < NA + NB ? 0 : l - NA - NB;
            if (i < FM) sc.a[i < FM ? i : 0] = reinterpret_cast<const AnyShort*>(SA + t * kBlocks + sfa[i < FM ? i : 0])->v;
            else sc.b[i < FM ? 0 : i - FM] = reinterpret_cast<const AnyShort*>(SB + t * kBlocks + sfb[i < FM ? 0 : i - FM])->v;
        }
    };
    auto fetch = [&](uint8_t* s, Scales& sc, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int l = 0; l < NL; ++l) fetch_one(s, sc, t, l);
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
    asm volatile("" : "+v"(oa[0]), "+v"(oa[1]), "+v"(ob[0]), "+v"(ob[1]));
    auto code_a = [&](const uint8_t* s, int g) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4i*>(s + oa[g / FM] + g % FM * 16 * kBK);
    };
    auto code_b = [&](const uint8_t* s, int kk, int j) __attribute__((always_inline)) {
        return *reinterpret_cast<const v4i*>(s + ob[kk] + j * 16 * kBK);
    };
    // One tile multiplied, with the loads of tile t (to `next`) spread between: a
    // wave that issues its loads in one go waits for the address unit, and its
    // matrix instructions with it.
    auto multiply = [&](auto with_loads, const uint8_t* s, const Scales& sc, uint8_t* next, Scales& next_sc, int t)
                        __attribute__((always_inline)) {
        v4i fa[3], fb[2][FN];
        fa[0] = code_a(s, 0);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[0][j] = code_b(s, 0, j);
        fa[1] = code_a(s, 1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int kk = g / FM, i = g % FM;
            if (g + 2 < G) fa[(g + 2) % 3] = code_a(s, g + 2);
            if (kk == 0) {
#pragma unroll
                for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) fb[1][j] = code_b(s, 1, j);
            }
            if constexpr (with_loads.value) {
#pragma unroll
                for (int l = 0; l < NL; ++l)
                    if (l * G / NL == g) fetch_one(next, next_sc, t, l);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = kk == 0 ? mfma4<0>(fb[0][j], fa[g % 3], acc[i][j], sc.b[j], sc.a[i])
                                    : mfma4<1>(fb[1][j], fa[g % 3], acc[i][j], sc.b[j], sc.a[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Tile t is in s; the loads of tile t + S - 1 go to `next`, whose tile every
    // wave has read before the barrier.  No branch between loads and waits, so the
    // number in flight is known everywhere.
    Scales sc[S];
    auto step = [&](const uint8_t* s, const Scales& from_sc, uint8_t* next, Scales& next_sc, int t)
                    __attribute__((always_inline)) {
        wait_loads<(S - 2) * NL>();
        barrier();
        multiply(std::true_type{}, s, from_sc, next, next_sc, t + S - 1);
    };
    if constexpr (S == 2) {
        // The scales of tiles 4 n .. 4 n + 3, 32 bytes a row: 16 bytes a lane; where
        // there are fewer tiles, 4 bytes a lane, those past them the row's first again,
        // not used.  (Of 8 bytes of a row in every tile, a wave's load touched 32 lines
        // for 256 bytes: 8192 x 8192 x 8192 took 276 us in place of 259.)
        static_assert(kScaleLoads % kW == 0, "each wave has as many");
        // a wave's load of scales is of A's rows or of B's
        auto s_load = [&](int i) __attribute__((always_inline)) { return wave * NS + i; };
        auto row_at = [&](int r) __attribute__((always_inline)) {
            return r < BM ? min(r, last_a) * (unsigned)p.ldsa : min(r - BM, last_b) * (unsigned)p.ldsb;
        };
        unsigned sfrom[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) sfrom[i] = row_at(s_load(i) * 32 + lane / 2);
        auto fetch_span = [&](int n) __attribute__((always_inline)) {
            uint8_t* to = spans + (n & 1) * kScales;
            if ((n + 1) * kSpan <= tiles) {
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    to_lds16(s_load(i) * 32 < BM ? SA : SB, sfrom[i] + (lane & 1) * 16, n * kSpan * kBlocks,
                             to + s_load(i) * 1024);
            } else {
                const int there = (tiles - n * kSpan) * 2, d = lane % 8 < there ? lane % 8 : 0;
                for (int i = wave; i < (BM + BN) / 8; i += kW)
                    to_lds4(i * 8 < BM ? SA : SB, row_at(i * 8 + lane / 8) + d * 4, n * kSpan * kBlocks, to + i * 256);
            }
        };
        int osa = (wm + r16) * kRowScales + g4 * 2, osb = (BM + wn + r16) * kRowScales + g4 * 2;
        asm volatile("" : "+v"(osa), "+v"(osb));
        // Two stages, the barrier before a tile's last two groups: by then all its
        // fragments are in registers, so the next tile's first ones are read, and
        // the loads of the one after that are issued into its LDS, while the matrix
        // instructions go on.
        static_assert(G % 4 == 0 && FM >= 4, "the ring of fragments comes round with the tile");
        v4i fa[4], fb[2][FN];
        // Tile t's first fragments and all its scales, where no load is in flight (as
        // one into `spans` may be later, the compiler would wait for it)
        auto first = [&](auto turn, const uint8_t* s, int t) __attribute__((always_inline)) {
            const uint8_t* at = spans + (t / kSpan & 1) * kScales + t % kSpan * kBlocks;
            auto scale = [&](int o) __attribute__((always_inline)) {
                return (int)*reinterpret_cast<const uint16_t*>(at + o);
            };
            Scales& x = sc[turn.value];
            fa[0] = code_a(s, 0);
            x.a[0] = scale(osa);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                fb[0][j] = code_b(s, 0, j);
                x.b[j] = scale(osb + j * 16 * kRowScales);
            }
            fa[1] = code_a(s, 1);
#pragma unroll
            for (int i = 1; i < FM; ++i) x.a[i] = scale(osa + i * 16 * kRowScales);
        };
        // The next tile's loads go out between the first groups: all at once they
        // hold up the fragment reads.
        constexpr int kPer = 2;
        static_assert(kPer * (G - 2) >= NL, "all loads go out");
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
#pragma unroll
                for (int l = g * kPer; l < (g + 1) * kPer && l < NL; ++l) fetch_one(next, sc[0], t + 1, l);
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = kk == 0 ? mfma4<0>(fb[0][j], fa[g % 4], acc[i][j], sc[kTurn].b[j], sc[kTurn].a[i])
                                        : mfma4<1>(fb[1][j], fa[g % 4], acc[i][j], sc[kTurn].b[j], sc[kTurn].a[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        fetch_span(0);
        fetch(s0, sc[0], 0);
        wait_loads<0>();
        barrier();
        first(std::integral_constant<int, 0>{}, s0, 0);
        int t = 0;
        for (; t + 2 <= tiles; t += 2) {
            run(std::integral_constant<int, 0>{}, s0, s1, t);
            run(std::integral_constant<int, 1>{}, s1, s0, t + 1);
        }
        if (t < tiles) run(std::integral_constant<int, 0>{}, s0, s1, t);
    } else {
        // (in this order: else the compiler waits, in every turn of the loop, for scales
        // that it has put behind later loads here)
        fetch(s0, sc[0], 0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(s1, sc[1], 1);
        __builtin_amdgcn_sched_barrier(0);
        fetch(s2, sc[2], 2);
        __builtin_amdgcn_sched_barrier(0);
        int t = 0;
        for (; t + S <= tiles; t += S) {
            step(s0, sc[0], s3, sc[3], t);
            step(s1, sc[1], s0, sc[0], t + 1);
            step(s2, sc[2], s1, sc[1], t + 2);
            step(s3, sc[3], s2, sc[2], t + 3);
        }
        // the last tiles % S are in flight
        wait_loads<0>();
        barrier();
        if (t < tiles) multiply(std::false_type{}, s0, sc[0], s0, sc[0], 0);
        if (t + 1 < tiles) multiply(std::false_type{}, s1, sc[1], s1, sc[1], 0);
        if (t + 2 < tiles) multiply(std::false_type{}, s2, sc[2], s2, sc[2], 0);
    }
    wait_loads<0>();  // also those past the end
    if (p.K % 256) {
        const int k0 = tiles * kBK, blocks = p.K / kMxBlock + (p.K % kMxBlock != 0);
        v4i end[NA + NB];
#pragma unroll
        for (int l = 0; l < NA + NB; ++l) end[l] = codes16((l < NA ? A : B) + (from[l] - chunk), k0 + chunk, p.K);
        Scales ends;
#pragma unroll
        for (int i = 0; i < FM; ++i) ends.a[i] = scales2(SA + (sfa[i] - g4 * 2), k0 / 16 + g4 * 2, blocks);
#pragma unroll
        for (int j = 0; j < FN; ++j) ends.b[j] = scales2(SB + (sfb[j] - g4 * 2), k0 / 16 + g4 * 2, blocks);
        __syncthreads();
#pragma unroll
        for (int l = 0; l < NA + NB; ++l)
            *reinterpret_cast<v4i*>(s0 + (l < NA ? wave * NA + l : BM / 8 + wave * NB + l - NA) * 1024 + lane * 16) = end[l];
        __syncthreads();
        multiply(std::false_type{}, s0, ends, s0, ends, 0);
    }
    barrier();  // the stage takes the tiles' place
    epilogue<FM, FN>(p, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(s0) + wave * (Stage<FM, FN>::kBytes / 4));
}

// ---- few rows -------------------------------------------------------------------------
// A workgroup has 16 rows and 16 channels, its eight waves share K in spans of 512
// elements, and the sums meet in LDS: operands straight to registers, at any
// alignment.  For a row or a few the weights' bytes bound it, for few tiles of long
// rows it has eight times the waves.  Of a span a lane takes 64 neighbouring bytes of a
// channel (blocks 4 g .. 4 g + 3, g = lane / 16) and their four scales.  Activations:
// codes in memory (ELEM kElemCodes), read alike; or up to 16 rows of floats or spike
// times, quantised by every workgroup into LDS while its weights are on their way, where
// that is no more than eight runs of eight a thread (4 x 4096 x 4096 from BF16 5.5 us,
// 8.0 with a launch of its own for that; 8 x 4096 x 4096 7.4 and 7.9).
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
    const int tiles_n = (p.N + 15) / 16;
    const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * kSmallRows;
    const int n0 = blockIdx.x % tiles_n * 16, n = n0 + r16 < p.N ? n0 + r16 : p.N - 1;
    const uint8_t *wc = p.B + (int64_t)n * p.ldb, *ws = p.sb + (int64_t)n * p.ldsb;
    const int spans = p.K / 512 + (p.K % 512 != 0), M = p.M - m0 < kSmallRows ? (int)(p.M - m0) : kSmallRows;
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
            a = load_span(p.A + (m0 + row) * p.lda, p.sa + (m0 + row) * p.ldsa, span, g, p.K);
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
    store_elem(p.out, (m0 + m) * p.ldo + n0 + c, apply_act(v, p.act), p.out_elem);
}

// Rows at any alignment to rows on `ld_to` bytes, a multiple of 16, `fill` behind
// them: codes (K elements; the upper half of an odd row's last byte is cleared) or
// scales (K bytes), 16 bytes a thread.
template <bool CODES>
__device__ __forceinline__ void realign(const uint8_t* __restrict__ from, int64_t ld, int64_t rows, int K,
                                        uint8_t* __restrict__ to, int64_t ld_to) {
    const int64_t per = ld_to / 16, n = rows * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
        const int64_t r = n < (int64_t(1) << 32) ? (uint32_t)at / (uint32_t)per : at / per;
        const int k = (int)(at - r * per) * 16;
        v4i v;
        if constexpr (CODES) {
            v = codes16(from + r * ld, k, K);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (int)scales4(from + r * ld, k + 4 * i, K);
        }
        *reinterpret_cast<v4i*>(to + r * ld_to + k) = v;
    }
}
__global__ __launch_bounds__(256) void k_mx4_realign(Mx4Copies c, int K, int64_t ldq_to, int64_t lds_to) {
    const auto& o = c.of[blockIdx.y];
    if (o.to_q) realign<true>(o.q, o.ldq, o.rows, K, o.to_q, ldq_to);
    if (o.to_s) realign<false>(o.s, o.lds, o.rows, K / kMxBlock + (K % kMxBlock != 0), o.to_s, lds_to);
}

template <int ELEM>
int run_small(vdttfs_ctx* ctx, const Mx4Args& a, const void* x, int64_t ldx) {
    const int64_t blocks = (a.M + kSmallRows - 1) / kSmallRows * ((a.N + 15) / 16);
    k_mx4_small<ELEM><<<dim3((unsigned)blocks), kSmallWaves * 64, 0, ctx->stream>>>(a, x, ldx, ctx->c.tfs, ctx->c.T);
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

// Rows that loads to LDS can take: of codes on 16 bytes, and where scales go that way
// too (large tiles), of scales on 4.
constexpr int64_t kMaxLd = 1 << 22;  // 256 rows of them below 2^31 bytes
static bool off(const uint8_t* p, int64_t ld, int to) { return (((uintptr_t)p | (uintptr_t)ld) & (to - 1)) != 0 || ld > kMaxLd; }
template <int BM, int BN, int WM, int WN, int S>
static int run_big(vdttfs_ctx* ctx, const Mx4Args& a) {
    const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    k_mx4_big<BM, BN, WM, WN, S><<<dim3((unsigned)(tm * tn)), WM * WN * 64, 0, ctx->stream>>>(a, (int)tm, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

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

// The kernel of a product and what it wants copied first.  Measured (us; K last,
// "odd": rows off 16 bytes, LDS tiles with their copies):
//   few tiles, long rows: 256x256x8192 16x16 7.2, LDS 32 12.4, 64 22; 235x34x3873 odd
//   8.4, through registers 32 11.6; 128x1024x1024 5.0 and 4.8; 64x4096x4096 (256 tiles
//   of 32) 11.7 and 8.2
//   short rows: 7150x2496x128 through registers 64 20.5, LDS 64 28; 2000x2000x512 8.7,
//   LDS 64 9.6, LDS 128 8.2
//   8192x4096x4096 LDS 256 75; 3000x3000x3000 (144 tiles of 256) 45, 128 51;
//   2560x8192x2048 (320, so a second round a quarter full) 41.5 and 37
//   2048x2048x2048 (256 tiles of 128) LDS 128 11, 64 28; 512x4096x4096 (128) 18, 25;
//   256x4096x4096 (64) 14.3, 13.7; 4225x192x4864 (68) 21, 11.3, through registers 20
//   odd: 3000x3000x3000 copied 47, through registers 83; 2048x2048x2048 19 and 25;
//   4225x192x4864 24 and 24, one operand alone some 16; 2000x2000x512 14 and 9.7
Mx4Plan mx4_plan(const Mx4Args& a) {
    Mx4Plan p{};
    auto tiles = [&](int t) { return (a.M + t - 1) / t * ((a.N + t - 1) / t); };
    const bool many = tiles(64) >= 192;
    const Mx4Path registers = many ? kMx4Tile64 : kMx4Tile32;
    if (a.M <= kSmallRows || (a.K >= 1024 && tiles(32) <= 128)) return p.path = kMx4Few, p;
    if (a.K < 512 || a.K / 2 > kMaxLd - 128) return p.path = registers, p;  // or rows too long for copies too
    const int64_t big = tiles(256), rounds = (big + 255) / 256;
    const double work = (double)a.M * a.N * a.K;
    p.path = many ? kMx4Lds64 : kMx4Lds32;
    if (rounds == 1 ? big >= 160 : big * 10 >= rounds * 256 * 7) p.path = kMx4Lds256;
    else if (tiles(128) >= 110) p.path = kMx4Lds128;
    p.a = off(a.A, a.lda, 16);
    p.b = off(a.B, a.ldb, 16);
    p.sa = a.ldsa > kMaxLd;
    p.sb = a.ldsb > kMaxLd;
    if (p.a || p.b || p.sa || p.sb) {
        const bool both = (p.a || p.sa) && (p.b || p.sb);
        if (work < (both ? 6e9 : 3e9)) return Mx4Plan{registers, false, false, false, false};
    }
    if (p.path == kMx4Lds256 || p.path == kMx4Lds128) {  // whose scales go to LDS in fours
        const bool sa = off(a.sa, a.ldsa, 4), sb = off(a.sb, a.ldsb, 4);
        if (work < 2e9 && ((sa && !p.a) || (sb && !p.b))) {
            p.path = many ? kMx4Lds64 : kMx4Lds32;
        } else {
            p.sa |= sa;
            p.sb |= sb;
        }
    }
    return p;
}

int launch_mx4_realign(vdttfs_ctx* ctx, const Mx4Copies& c, int K, int64_t ldq_to, int64_t lds_to) {
    int64_t blocks = 0;
    for (const auto& o : c.of) {
        const int64_t n = o.rows * (o.to_q ? ldq_to : o.to_s ? lds_to : 0) / 16;
        blocks = std::max(blocks, (n + 255) / 256);
    }
    if (!blocks) return VDTTFS_OK;
    k_mx4_realign<<<dim3((unsigned)std::min(blocks, int64_t(1) << 20), 2), 256, 0, ctx->stream>>>(c, K, ldq_to, lds_to);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_mx4(vdttfs_ctx* ctx, const Mx4Args& a, Mx4Path path) {
    if (a.M <= 0 || a.N <= 0) return VDTTFS_OK;
    static constexpr struct {
        int bm, bn;
    } kTiles[] = {{16, 16}, {32, 32}, {64, 64}, {32, 32}, {64, 64}, {128, 128}, {256, 256}};
    const int bm = kTiles[path].bm, bn = kTiles[path].bn;
    const int64_t rows = max_blocks(512) / ((a.N + bn - 1) / bn) * bm;  // as many a launch as its tiles allow
    for (int64_t m = 0; m < a.M; m += rows) {
        Mx4Args part = a;
        part.A += m * a.lda;
        part.sa += m * a.ldsa;
        part.out = static_cast<char*>(a.out) + m * a.ldo * (a.out_elem == VDTTFS_ELEM_F32 ? 4 : 2);
        part.M = a.M - m < rows ? a.M - m : rows;
        int rc = VDTTFS_OK;
        switch (path) {
            case kMx4Few: rc = run_small<kElemCodes>(ctx, part, nullptr, 0); break;
            case kMx4Tile32: rc = run_tile<32, 32>(ctx, part); break;
            case kMx4Tile64: rc = run_tile<64, 64>(ctx, part); break;
            case kMx4Lds32: rc = run_big<32, 32, 2, 2, 4>(ctx, part); break;
            case kMx4Lds64: rc = run_big<64, 64, 2, 2, 4>(ctx, part); break;
            case kMx4Lds128: rc = run_big<128, 128, 2, 2, 2>(ctx, part); break;
            case kMx4Lds256: rc = run_big<256, 256, 2, 4, 2>(ctx, part); break;
        }
        if (rc != VDTTFS_OK) return rc;
    }
    return VDTTFS_OK;
}

int launch_mx4_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, uint8_t* q,
                          int64_t ldq, uint8_t* s, int64_t lds) {
    if (rows <= 0 || cols <= 0) return VDTTFS_OK;
    const int64_t per = ((int64_t)cols + kMxBlock - 1) / kMxBlock * 4, blocks = (rows * per + 255) / 256;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
    const float tfs = ctx->c.tfs;
    const int T = ctx->c.T;
    if (elem == VDTTFS_ELEM_F32)
        k_mx4_quant<VDTTFS_ELEM_F32><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, tfs, T);
    else if (elem == VDTTFS_ELEM_BF16)
        k_mx4_quant<VDTTFS_ELEM_BF16><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, tfs, T);
    else if (elem == VDTTFS_ELEM_F16)
        k_mx4_quant<VDTTFS_ELEM_F16><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, tfs, T);
    else
        k_mx4_quant<VDTTFS_ELEM_TIMES><<<grid, 256, 0, ctx->stream>>>(x, ldx, rows, cols, q, ldq, s, lds, tfs, T);
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
