// Products of 8-bit codes on the matrix cores, dense and by expert.
//
// out[m][n] = act(float(sum_k A[m][k] B[n][k]) * sa[m] * sb[n] + bias[n]), the
// sum in 32-bit integers (v_mfma_i32_16x16x64_i8), so no order of k matters.
#include <type_traits>

#include "codes.h"
#include "elem.h"
#include "head.h"
#include "tiles.h"
#include "wave.h"

namespace vdttfs {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

struct __attribute__((packed, aligned(4))) Floats4 {
    v4f v;
};
// p[0..3], the last of the first n_ok again past them (n_ok <= 0: p[0] .. is
// not there, and p[n_ok - 1] is).
__device__ __forceinline__ v4f take4(const float* p, int n_ok, bool whole) {
    if (whole) return reinterpret_cast<const Floats4*>(p)->v;
    v4f r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = p[e < n_ok ? e : n_ok - 1];
    return r;
}

// A wave's sums to its outputs.  A lane's four sums of a fragment are row
// m = lane & 15, channels (lane >> 4) * 4 + 0..3; stored from there, a wave
// would write 32 bytes of each of 16 rows at a time, and whole-chip stores
// then ran at 1 TB/s (64 of the 170 us of 8192 x 4096 x 4096).  So 16 rows at
// a time pass through the wave's own part of LDS (stage) and leave as 16
// bytes a lane, a row's outputs together.  m0: the wave's first row; wn: its
// first channel in the tile.
template <int FM, int FN, bool GATED>
struct Stage {
    static constexpr int kCols = GATED ? FN * 8 : FN * 16;  // outputs of a row
    static constexpr int kRow = kCols + 4;                  // floats from row to row
    static constexpr int kBytes = 16 * kRow * 4;
};
// A lane's rows (m0 + 16 i + lane % 16): their scales and output rows.  Loaded
// before the products, whose end would wait for them.
template <int FM>
struct Rows {
    float sa[FM];
    int o_row[FM];
};
template <int FM, bool GROUPED>
__device__ __forceinline__ Rows<FM> rows_of(const I8Args& p, int64_t m0, int64_t m_end) {
    Rows<FM> r;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        int64_t m = m0 + i * 16 + (lane_id() & 15);
        if (m >= m_end) m = m_end - 1;
        r.sa[i] = p.sa[GROUPED && p.a_rows ? p.a_rows[m] : m];
        r.o_row[i] = GROUPED && p.o_rows ? p.o_rows[m] : (int)m;
    }
    return r;
}
template <int FM, int FN, bool GATED>
__device__ __forceinline__ void epilogue(const I8Args& p, const v4i (&acc)[FM][FN], const Rows<FM>& rows, int64_t m0,
                                         int64_t m_end, int n0, int wn, const float* sb, const float* bias,
                                         float* stage) {
    typedef Stage<FM, FN, GATED> S;
    const int lane = lane_id();
    const int nw = n0 + (GATED ? wn / 2 : wn);  // the wave's first output column
    const int size = p.out_elem == VDTTFS_ELEM_F32 ? 4 : 2;
    const bool bf16 = p.out_elem == VDTTFS_ELEM_BF16;
    const bool whole = nw + S::kCols <= p.N;
    const bool vec = ((p.ldo * size) & 15) == 0 && (((uintptr_t)p.out + (size_t)nw * size) & 15) == 0;
    // everything that comes from memory first: the stores below may alias it,
    // so a load between them would wait in line
    constexpr int kFrags = GATED ? FN / 2 : FN, kStep = GATED ? 2 : 1;
    v4f s[kFrags], b[kFrags], s2[kFrags], b2[kFrags];
#pragma unroll
    for (int j = 0; j < kFrags; ++j) {
        const int n = nw + j * 16 + (lane >> 4) * 4;
        s[j] = take4(sb + n, p.N - n, whole);
        if (bias) b[j] = take4(bias + n, p.N - n, whole);
        if constexpr (GATED) {
            s2[j] = take4(sb + p.N + n, p.N - n, whole);
            if (bias) b2[j] = take4(bias + p.N + n, p.N - n, whole);
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t mi = m0 + i * 16;
        if (mi >= m_end) break;
        // the vectors that a lane stores where all 16 rows and all columns are
        // there: their places are known before the sums are
        constexpr int kPut2 = S::kCols < 32 ? 1 : S::kCols / 32, kPut4 = S::kCols / 16;  // of 2 bytes, of 4
        int64_t to[kPut4];
        const bool full = whole && vec && mi + 16 <= m_end && (S::kCols >= 32 || size == 4);
        if (full) {
            const int per = size == 2 ? S::kCols / 8 : S::kCols / 4;  // lanes of a row
#pragma unroll
            for (int r = 0; r < kPut4; ++r)
                if (r < kPut2 || size == 4)
                    to[r] = __shfl(rows.o_row[i], (r * (64 / per) + lane / per) & 15, 64) * p.ldo + nw + lane % per * (16 / size);
        }
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const int c = j * 16 + (lane >> 4) * 4;  // column of the wave's outputs
            v4f v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j * kStep][e] * rows.sa[i] * s[j][e];
            if (bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += b[j][e];
            }
            if (p.act == VDTTFS_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], VDTTFS_ACT_RELU);
            } else if (p.act == VDTTFS_ACT_SILU) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], VDTTFS_ACT_SILU);
            }
            if constexpr (GATED) {
                v4f u;
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = (float)acc[i][j * 2 + 1][e] * rows.sa[i] * s2[j][e];
                if (bias) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] += b2[j][e];
                }
                v *= u;
            }
            *reinterpret_cast<v4f*>(stage + (lane & 15) * S::kRow + c) = v;
        }
        wave_sync();
        if (full && size == 2) {
            constexpr int kLanes = S::kCols / 8;
            v4f x[kPut2], y[kPut2];
#pragma unroll
            for (int r = 0; r < kPut2; ++r) {
                const float* f = stage + (r * (64 / kLanes) + lane / kLanes) * S::kRow + lane % kLanes * 8;
                x[r] = *reinterpret_cast<const v4f*>(f);
                y[r] = *reinterpret_cast<const v4f*>(f + 4);
            }
#pragma unroll
            for (int r = 0; r < kPut2; ++r) {
                v4i w;
                if (bf16) w = v4i{(int)pack2(x[r][0], x[r][1], true), (int)pack2(x[r][2], x[r][3], true),
                                  (int)pack2(y[r][0], y[r][1], true), (int)pack2(y[r][2], y[r][3], true)};
                else w = v4i{(int)pack2(x[r][0], x[r][1], false), (int)pack2(x[r][2], x[r][3], false),
                             (int)pack2(y[r][0], y[r][1], false), (int)pack2(y[r][2], y[r][3], false)};
                __builtin_nontemporal_store(w, reinterpret_cast<v4i*>(static_cast<uint16_t*>(p.out) + to[r]));
            }
        } else if (full) {
            constexpr int kLanes = S::kCols / 4;
            v4f x[kPut4];
#pragma unroll
            for (int r = 0; r < kPut4; ++r)
                x[r] = *reinterpret_cast<const v4f*>(stage + (r * (64 / kLanes) + lane / kLanes) * S::kRow +
                                                     lane % kLanes * 4);
#pragma unroll
            for (int r = 0; r < kPut4; ++r)
                __builtin_nontemporal_store(x[r], reinterpret_cast<v4f*>(static_cast<float*>(p.out) + to[r]));
        } else if (vec && size == 2) {
            constexpr int kLanes = S::kCols / 8;  // lanes of a row
#pragma unroll
            for (int r = 0; r < 16; r += 64 / kLanes) {
                const int row = r + lane / kLanes, c = lane % kLanes * 8;
                const int64_t o = __shfl(rows.o_row[i], row & 15, 64) * p.ldo + nw + c;
                if (row >= 16 || mi + row >= m_end) continue;
                const float* f = stage + row * S::kRow + c;
                if (nw + c + 8 > p.N) {
#pragma unroll 1
                    for (int e = 0; e < p.N - nw - c; ++e) store_elem(p.out, o + e, f[e], p.out_elem);
                    continue;
                }
                const v4f x = *reinterpret_cast<const v4f*>(f), y = *reinterpret_cast<const v4f*>(f + 4);
                const v4i w = {(int)pack2(x[0], x[1], bf16), (int)pack2(x[2], x[3], bf16),
                               (int)pack2(y[0], y[1], bf16), (int)pack2(y[2], y[3], bf16)};
                __builtin_nontemporal_store(w, reinterpret_cast<v4i*>(static_cast<uint16_t*>(p.out) + o));
            }
        } else if (vec) {
            constexpr int kLanes = S::kCols / 4;
#pragma unroll
            for (int r = 0; r < 16; r += 64 / kLanes) {
                const int row = r + lane / kLanes, c = lane % kLanes * 4;
                const int64_t o = __shfl(rows.o_row[i], row & 15, 64) * p.ldo + nw + c;
                if (row >= 16 || mi + row >= m_end) continue;
                if (nw + c + 4 > p.N) {
#pragma unroll 1
                    for (int e = 0; e < p.N - nw - c; ++e) store_elem(p.out, o + e, stage[row * S::kRow + c + e], p.out_elem);
                    continue;
                }
                __builtin_nontemporal_store(*reinterpret_cast<const v4f*>(stage + row * S::kRow + c),
                                            reinterpret_cast<v4f*>(static_cast<float*>(p.out) + o));
            }
        } else {
#pragma unroll 1
            for (int at = lane; at < 16 * S::kCols; at += 64) {
                const int row = at / S::kCols, c = at % S::kCols;
                const int64_t o = __shfl(rows.o_row[i], row, 64) * p.ldo + nw + c;
                if (mi + row >= m_end || nw + c >= p.N) continue;
                store_elem(p.out, o, stage[row * S::kRow + c], p.out_elem);
            }
        }
        wave_sync();
    }
}

constexpr int kBK = 128;  // codes of a row in one LDS tile

// A workgroup of WM x WN waves computes BM rows x BN channels.  Both operands
// pass through LDS in tiles of 128 codes a row; the 16-byte chunk c of row r
// lies at chunk c ^ (r & 7), so that the 16 rows of a fragment read at one
// chunk come from different banks.  The weights are the matrix instruction's
// first operand: a lane then holds four neighbouring channels of one row.
// Gated: the tile's channels alternate in runs of 16 between gate and up, so a
// wave holds both halves of each of its outputs.
template <int BM, int BN, int WM, int WN, bool GATED, bool GROUPED>
__global__ __launch_bounds__(WM* WN * 64) void k_i8_tile(I8Args p, int tiles_n) {
    constexpr int kT = WM * WN * 64;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int NA = BM * 8 / kT, NB = BN * 8 / kT;  // 16-byte chunks a thread loads
    constexpr int OUT_N = GATED ? BN / 2 : BN;         // output columns of a tile
    static_assert(NA * kT == BM * 8 && NB * kT == BN * 8, "chunks divide");
    static_assert(!GATED || FN % 2 == 0, "a wave holds gate and up");
    __shared__ __align__(16) int8_t lds[(BM + BN) * kBK];
    int8_t* sA = lds;
    int8_t* sB = lds + BM * kBK;
    static_assert(WM * WN * Stage<FM, FN, GATED>::kBytes <= (BM + BN) * kBK, "the outputs' stage fits");

    const int tile_m = blockIdx.x / tiles_n, tile_n = blockIdx.x % tiles_n;
    int64_t m0 = (int64_t)tile_m * BM, m_end = p.M;
    const int8_t* B = p.B;
    const float* sb = p.sb;
    const float* bias = p.bias;
    if constexpr (GROUPED) {
        if (tile_m >= *p.n_tiles) return;
        const int4 t = p.tiles[tile_m];
        m0 = t.y;
        m_end = t.z;
        B += (int64_t)t.x * p.b_stride;
        sb += (int64_t)t.x * p.s_stride;
        if (bias) bias += (int64_t)t.x * p.s_stride;
    }
    const int n0 = tile_n * OUT_N;

    const int tid = threadIdx.x, lane = lane_id();
    const int8_t* pa[NA];
    const int8_t* pb[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        int64_t m = m0 + (tid + i * kT) / 8;
        if (m >= m_end) m = m_end - 1;  // a valid row, its products are not stored
        if (GROUPED && p.a_rows) m = p.a_rows[m];
        pa[i] = p.A + m * p.lda;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int c = (tid + i * kT) / 8;
        int n = GATED ? n0 + (c >> 5) * 16 + (c & 15) : n0 + c;
        if (n >= p.N) n = p.N - 1;
        if (GATED && (c & 16)) n += p.N;
        pb[i] = B + (int64_t)n * p.ldb;
    }
    const int chunk = (tid & 7) * 16;
    const int put = (tid >> 3) * kBK + (((tid & 7) ^ ((tid >> 3) & 7)) * 16);  // + i * kT * 16

    const int wave = uniform(tid >> 6);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const Rows<FM> rows = rows_of<FM, GROUPED>(p, m0 + wm, m_end);
    v4i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};

    v4i ra[NA], rb[NB];
    auto fetch = [&](int k0) {
        if (k0 + kBK <= p.K) {
#pragma unroll
            for (int i = 0; i < NA; ++i) ra[i] = reinterpret_cast<const Bytes16*>(pa[i] + k0 + chunk)->v;
#pragma unroll
            for (int i = 0; i < NB; ++i) rb[i] = reinterpret_cast<const Bytes16*>(pb[i] + k0 + chunk)->v;
            return;
        }
#pragma unroll
        for (int i = 0; i < NA; ++i) ra[i] = load16(pa[i], k0 + chunk, p.K);
#pragma unroll
        for (int i = 0; i < NB; ++i) rb[i] = load16(pb[i], k0 + chunk, p.K);
    };
    fetch(0);
    for (int k0 = 0; k0 < p.K; k0 += kBK) {
        __syncthreads();  // the previous tile is read
#pragma unroll
        for (int i = 0; i < NA; ++i) *reinterpret_cast<v4i*>(sA + put + i * kT * 16) = ra[i];
#pragma unroll
        for (int i = 0; i < NB; ++i) *reinterpret_cast<v4i*>(sB + put + i * kT * 16) = rb[i];
        __syncthreads();
        if (k0 + kBK < p.K) fetch(k0 + kBK);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c = kk * 4 + (lane >> 4);
            v4i fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int r = wm + i * 16 + (lane & 15);
                fa[i] = *reinterpret_cast<const v4i*>(sA + r * kBK + ((c ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int r = wn + j * 16 + (lane & 15);
                fb[j] = *reinterpret_cast<const v4i*>(sB + r * kBK + ((c ^ (r & 7)) * 16));
            }
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }

    __syncthreads();
    epilogue<FM, FN, GATED>(p, acc, rows, m0 + wm, m_end, n0, wn, sb, bias,
                            reinterpret_cast<float*>(lds) + wave * (Stage<FM, FN, GATED>::kBytes / 4));
}

// The large product: tiles of BK codes a row go from memory to LDS directly
// (16 bytes a lane, no registers between), S tiles deep: while one is
// multiplied, the loads of the next S - 1 are in flight.  A wave-wide load
// fills 1 KiB of LDS; the chunk that lies at place c of row r is chunk
// c ^ swizzle(r), so that the 16 rows of a fragment come from all banks.
// Needs 16-byte aligned rows; the last K % 16 codes go through registers with
// zeros behind them (S > 2; the two-stage tiles take whole chunks only).
// 8192x4096x4096 with the 256x256 tile takes 110 to 125 us, 2.2 to 2.5 POP/s of
// the 5 there are, as the codes' own bits let the clock be.  A step of 128 codes
// in K is 0.85 us of matrix instructions at their peak, 1.05 with the reads of
// their fragments from LDS and 1.4 to 1.5 with the loads into it, so the loads
// (64 KiB a step, from the XCD's L2) bound it; 10 us are the outputs.
template <int BK>
__device__ __forceinline__ int swizzle(int row) {
    return BK == 128 ? row & 7 : (row >> 2) & 3;
}

__device__ __align__(16) const int8_t kZeros[16] = {};

template <int BM, int BN, int WM, int WN, int BK, int S, bool GATED, bool GROUPED>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_i8_big(I8Args p, int tiles_m, int tiles_n) {
    constexpr int kW = WM * WN, kChunks = BK / 16, kRows = 64 / kChunks;  // rows of one 1 KiB load
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int NA = BM / kRows / kW, NB = BN / kRows / kW, NL = NA + NB;  // loads of a wave and tile
    constexpr int OUT_N = GATED ? BN / 2 : BN;
    constexpr int kTile = (BM + BN) * BK;
    static_assert(NA * kW * kRows == BM && NB * kW * kRows == BN, "loads divide");
    static_assert(S >= 2 && S <= 4 && (S - 2) * NL < 64, "stages");
    constexpr int kStage = kW * Stage<FM, FN, GATED>::kBytes;
    // an array for each stage: only then does the compiler see that reads of
    // one need not wait for loads into another
    __shared__ __align__(16) int8_t s0[kTile > kStage ? kTile : kStage];
    __shared__ __align__(16) int8_t s1[kTile];
    __shared__ __align__(16) int8_t s2[S > 2 ? kTile : 16];
    __shared__ __align__(16) int8_t s3[S > 3 ? kTile : 16];

    int tile_m, tile_n;
    if (GROUPED) tiles_m = *p.n_tiles;  // the grid has room for max_tiles
    if (!tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, &tile_m, &tile_n)) return;
    int64_t m0 = (int64_t)tile_m * BM, m_end = p.M;
    const int8_t* B = p.B;
    const float* sb = p.sb;
    const float* bias = p.bias;
    if constexpr (GROUPED) {
        const int4 t = p.tiles[tile_m];
        m0 = t.y;
        m_end = t.z;
        B += (int64_t)t.x * p.b_stride;
        sb += (int64_t)t.x * p.s_stride;
        if (bias) bias += (int64_t)t.x * p.s_stride;
    }
    const int n0 = tile_n * OUT_N;
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6);
    const int lrow = lane / kChunks, chunk = ((lane % kChunks) ^ swizzle<BK>(lrow)) * 16;
    auto a_row = [&](int i) __attribute__((always_inline)) {
        int64_t m = m0 + (wave * NA + i) * kRows + lrow;
        if (m >= m_end) m = m_end - 1;  // a valid row, its products are not stored
        if (GROUPED && p.a_rows) m = p.a_rows[m];
        return p.A + m * p.lda + chunk;
    };
    auto b_row = [&](int i) __attribute__((always_inline)) {
        const int c = (wave * NB + i) * kRows + lrow;
        int n = GATED ? n0 + (c >> 5) * 16 + (c & 15) : n0 + c;
        if (n >= p.N) n = p.N - 1;
        if (GATED && (c & 16)) n += p.N;
        return B + (int64_t)n * p.ldb + chunk;
    };
    const int8_t* pa[NA];
    const int8_t* pb[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) pa[i] = a_row(i);
#pragma unroll
    for (int i = 0; i < NB; ++i) pb[i] = b_row(i);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const Rows<FM> rows = rows_of<FM, GROUPED>(p, m0 + wm, m_end);
    v4i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};

    // Tile 0 holds the whole chunks past the last whole tile, if any; the last
    // K % 16 codes come after all.
    const int k16 = p.K & ~15, part = k16 % BK, tiles = (k16 + BK - 1) / BK;
    auto fetch_one = [&](int8_t* s, int k0, int l) __attribute__((always_inline)) {
        if (l < NA)
            __builtin_amdgcn_global_load_lds((GlobalPtr)(pa[l] + k0), (LdsPtr)(s + (wave * NA + l) * 1024), 16, 0, 0);
        else
            __builtin_amdgcn_global_load_lds((GlobalPtr)(pb[l - NA] + k0),
                                             (LdsPtr)(s + BM * BK + (wave * NB + l - NA) * 1024), 16, 0, 0);
    };
    // where tile t > 0 of several starts; past the end the last, loaded and not used
    auto k_of = [&](int t) __attribute__((always_inline)) { return ((t < tiles ? t : tiles - 1) - (part ? 1 : 0)) * BK; };
    // Tile 0 where it is partial: chunks past its end are zeros.
    auto fetch_part = [&](int8_t* s) __attribute__((always_inline)) {
        const bool in = chunk < part;
#pragma unroll
        for (int l = 0; l < NL; ++l) {
            const int8_t* row = l < NA ? pa[l < NA ? l : 0] : pb[l < NA ? 0 : l - NA];
            const int8_t* from = in ? row + (k16 - part) : kZeros;
            __builtin_amdgcn_global_load_lds(
                (GlobalPtr)from, (LdsPtr)(s + (l < NA ? wave * NA + l : BM / kRows + wave * NB + l - NA) * 1024), 16, 0,
                0);
        }
    };
    auto fetch = [&](int8_t* s, int t) __attribute__((always_inline)) {
#pragma unroll
        for (int l = 0; l < NL; ++l) fetch_one(s, k_of(t), l);
    };
    // One tile multiplied, with the loads of another (k0 of it, to `next`)
    // spread between: a wave that issues its loads in one go waits for the
    // address unit, and its matrix instructions with it.  Each group is one row
    // fragment against all channel fragments; fragments are read two groups
    // (channels: one k step) ahead.
    constexpr int KK = BK / 64, G = KK * FM;
    auto multiply = [&](auto with_loads, const int8_t* s, int8_t* next, int k0) __attribute__((always_inline)) {
        const int r = lane & 15;
        v4i fa[3], fb[2][FN];
        auto read_a = [&](int g) __attribute__((always_inline)) {
            const int c = ((g / FM * 4 + (lane >> 4)) ^ swizzle<BK>(r)) * 16;
            fa[g % 3] = *reinterpret_cast<const v4i*>(s + (wm + g % FM * 16 + r) * BK + c);
        };
        auto read_b = [&](int kk, int j) __attribute__((always_inline)) {
            const int c = ((kk * 4 + (lane >> 4)) ^ swizzle<BK>(r)) * 16;
            fb[kk & 1][j] = *reinterpret_cast<const v4i*>(s + (BM + wn + j * 16 + r) * BK + c);
        };
        read_a(0);
#pragma unroll
        for (int j = 0; j < FN; ++j) read_b(0, j);
        if (G > 1) read_a(1);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int kk = g / FM, i = g % FM;
            if (g + 2 < G) read_a(g + 2);
            if (kk + 1 < KK) {
#pragma unroll
                for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) read_b(kk + 1, j);
            }
            if constexpr (with_loads.value) {
#pragma unroll
                for (int l = 0; l < NL; ++l)
                    if (l * G / NL == g) fetch_one(next, k0, l);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[kk & 1][j], fa[g % 3], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Tile t is in s; the loads of tile t + S - 1 go to `next`, whose tile
    // every wave has read before the barrier.  No branch between loads and
    // waits, so the number in flight is known everywhere and the compiler adds
    // no waits of its own.
    auto step = [&](const int8_t* s, int8_t* next, int t) __attribute__((always_inline)) {
        wait_loads<(S - 2) * NL>();
        barrier();
        multiply(std::true_type{}, s, next, k_of(t + S - 1));
    };
    if constexpr (S == 2) {
        // Two stages, the barrier before a tile's last two groups: by then all
        // its fragments are in registers, so the next tile's first ones are
        // read, and the loads of the one after that are issued into its LDS,
        // while the matrix instructions go on.
        static_assert(G % 4 == 0 && G >= 4, "the ring of fragments comes round with the tile");
        const int r = lane & 15;
        v4i fa[4], fb[2][FN];
        auto read_a = [&](const int8_t* s, int g) __attribute__((always_inline)) {
            const int c = ((g / FM * 4 + (lane >> 4)) ^ swizzle<BK>(r)) * 16;
            fa[g % 4] = *reinterpret_cast<const v4i*>(s + (wm + g % FM * 16 + r) * BK + c);
        };
        auto read_b = [&](const int8_t* s, int kk, int j) __attribute__((always_inline)) {
            const int c = ((kk * 4 + (lane >> 4)) ^ swizzle<BK>(r)) * 16;
            fb[kk & 1][j] = *reinterpret_cast<const v4i*>(s + (BM + wn + j * 16 + r) * BK + c);
        };
        auto first = [&](const int8_t* s) __attribute__((always_inline)) {
            read_a(s, 0);
#pragma unroll
            for (int j = 0; j < FN; ++j) read_b(s, 0, j);
            read_a(s, 1);
        };
        // A tile's first kEarly loads go out behind the barrier that frees its
        // LDS, the others between the first groups of the next tile: all at
        // once they hold up the fragment reads.
        constexpr int kEarly = 2, kPer = (NL - kEarly + G / 2 - 3) / (G / 2 - 2 > 0 ? G / 2 - 2 : 1);
        static_assert(kEarly + kPer * (G - 2) >= NL, "all loads go out");
        auto run = [&](int8_t* s, int8_t* next, int t) __attribute__((always_inline)) {
            const int k0 = k_of(t + 2), k1 = k_of(t + 1);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int kk = g / FM, i = g % FM;
                if (g + 2 < G) read_a(s, g + 2);
                if (kk + 1 < KK) {
#pragma unroll
                    for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) read_b(s, kk + 1, j);
                }
                if (g == G - 2) {
                    wait_loads<0>();
                    barrier();
                    first(next);
                }
                if (g >= G - 2) fetch_one(s, k0, g - (G - 2));
                else
#pragma unroll
                    for (int l = kEarly + g * kPer; l < kEarly + (g + 1) * kPer && l < NL; ++l) fetch_one(next, k1, l);
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[kk & 1][j], fa[g % 4], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // at least two tiles (deep_ok)
        if (part) fetch_part(s0);
        else fetch(s0, 0);
        wait_loads<0>();
#pragma unroll
        for (int l = 0; l < kEarly; ++l) fetch_one(s1, k_of(1), l);
        barrier();
        first(s0);
        for (int t = 0; t < tiles; t += 2) {
            run(s0, s1, t);
            if (t + 1 < tiles) run(s1, s0, t + 1);
        }
    } else if (tiles == 1) {  // nothing to load ahead
        if (part) fetch_part(s0);
        else fetch(s0, 0);
        wait_loads<0>();
        barrier();
        multiply(std::false_type{}, s0, s0, 0);
    } else if (tiles > 1) {
        if (part) fetch_part(s0);
        else fetch(s0, 0);
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
        if (t < tiles) multiply(std::false_type{}, s0, s0, 0);
        if (t + 1 < tiles) multiply(std::false_type{}, s1, s1, 0);
        if (S > 3 && t + 2 < tiles) multiply(std::false_type{}, s2, s2, 0);
    }
    if (S > 2 && k16 < p.K) {
        v4i end[NL];
#pragma unroll
        for (int l = 0; l < NL; ++l)
            end[l] = load16((l < NA ? a_row(l) : b_row(l - NA)) - chunk, k16 + chunk, p.K);
        __syncthreads();
#pragma unroll
        for (int l = 0; l < NL; ++l)
            *reinterpret_cast<v4i*>(s0 + (l < NA ? wave * NA + l : BM / kRows + wave * NB + l - NA) * 1024 +
                                    lane * 16) = end[l];
        __syncthreads();
        multiply(std::false_type{}, s0, s0, 0);
    }
    wait_loads<0>();  // also those past the end: the stage takes their place
    barrier();
    epilogue<FM, FN, GATED>(p, acc, rows, m0 + wm, m_end, n0, wn, sb, bias,
                            reinterpret_cast<float*>(s0) + wave * (Stage<FM, FN, GATED>::kBytes / 4));
}

// Rows of codes to rows on 128 bytes with zeros behind them, 16 codes a thread.
__global__ __launch_bounds__(256) void k_realign(const int8_t* __restrict__ from, int64_t ld, int64_t rows, int K,
                                                 int8_t* __restrict__ to, int64_t ld_to) {
    const int64_t per = ld_to / 16, n = rows * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
        const int64_t r = at / per;
        const int k = (int)(at - r * per) * 16;
        *reinterpret_cast<v4i*>(to + r * ld_to + k) = load16(from + r * ld, k, K);
    }
}

// Rows that 16-byte loads to LDS can take.
bool aligned16(const I8Args& a) {
    return (((uintptr_t)a.A | (uintptr_t)a.B | (uintptr_t)a.lda | (uintptr_t)a.ldb | (uintptr_t)a.b_stride) & 15) == 0;
}

// What the two-stage tiles ask of K: whole chunks, and two tiles at least.
constexpr int kDeepK = 256;
bool deep_k(int K) { return K % 16 == 0 && K >= kDeepK; }
bool deep_ok(const I8Args& a) { return aligned16(a) && deep_k(a.K); }

int64_t tiles_of(int64_t M, int N, int bm, int bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); }

}  // namespace

int launch_realign(vdttfs_ctx* ctx, const int8_t* from, int64_t ld, int64_t rows, int K, int8_t* to, int64_t ld_to) {
    const int64_t blocks = (rows * (ld_to / 16) + 255) / 256;
    if (blocks <= 0) return VDTTFS_OK;
    k_realign<<<dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), 256, 0, ctx->stream>>>(from, ld, rows, K, to,
                                                                                               ld_to);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

// Whether a product is large enough for rows that the two-stage tiles do not
// take to be copied first, rather than read unaligned through registers (us,
// with copies and without): 8192x4096x4095 147, 394; 4000x1000x1000 23, 17.  Of
// rows quantised in scratch only the weights are copied (from BF16, with and
// without): 4000x1000x1001 22.5, 27.1; 1000x1000x1001 13.6, 16.2; 8000x200x301
// 15.6, 16.5; 6165x337x571 25.3, 24.6.
bool i8_wants_aligned(const I8Args& a) {
    return a.K >= kDeepK && !deep_ok(a) && (double)a.M * a.N * a.K >= (a.a_padded ? 2e8 : 1e10) &&
           tiles_of(a.M, a.N, 64, 64) >= 192;
}

template <int BM, int BN, int WM, int WN, int BK, int S>
int run_big(vdttfs_ctx* ctx, const I8Args& a) {
    const int64_t tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    k_i8_big<BM, BN, WM, WN, BK, S, false, false>
        <<<dim3((unsigned)(tm * tn)), WM * WN * 64, 0, ctx->stream>>>(a, (int)tm, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

template <int BM, int BN>
int run_tile(vdttfs_ctx* ctx, const I8Args& a) {
    const int64_t tn = (a.N + BN - 1) / BN, blocks = (a.M + BM - 1) / BM * tn;
    k_i8_tile<BM, BN, 2, 2, false, false><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, (int)tn);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

// Rows on 16 bytes take the tiles that go to LDS directly: the largest tile of
// which there are enough to fill the chip, as below that a CU's time goes by
// the number of steps in K, whatever the tile.  Measured (us, K last):
//   8192x4096x4096: 256x256 125, 128x128 155, 64x128 183, 64x64 219
//   1536x8192x2048 (192 tiles of 256): 32, 36, 37, 45;  2560x8192x2048 (320, so
//   two rounds, the second a quarter full): 62, 53, 58, 72
//   1024x4096x4096 (256 of 128): 128x128 28, 64x128 23, 64x64 27
//   256x4096x4096: 64x128 14.7, 64x64 10.2, 32x32 14.2;  64x4096x4096: 64x64
//   9.6, 32x32 7.6;  333x1111x1024: 64x64 7.3, 32x32 4.6
// Rows off 16 bytes and not worth a copy go through registers.
I8Tile i8_dense_tile(int64_t M, int N, int K, bool aligned) {
    auto tiles = [&](int bm, int bn) { return tiles_of(M, N, bm, bn); };
    if (!aligned) return tiles(64, 64) >= 192 ? I8Tile{64, 64} : I8Tile{32, 32};
    const int64_t big = tiles(256, 256), rounds = (big + 255) / 256;
    const bool deep = deep_k(K);
    if (deep && (rounds == 1 ? big >= 160 : big * 10 >= rounds * 256 * 7)) return I8Tile{256, 256};
    if (deep && tiles(128, 128) >= 384) return I8Tile{128, 128};
    if (tiles(64, 128) >= 384) return I8Tile{64, 128};
    return tiles(64, 64) >= 192 ? I8Tile{64, 64} : I8Tile{32, 32};
}

static int run_dense(vdttfs_ctx* ctx, const I8Args& a, I8Tile t, bool aligned) {
    if (!aligned) return t.bm == 64 ? run_tile<64, 64>(ctx, a) : run_tile<32, 32>(ctx, a);
    if (t.bm == 256) return run_big<256, 256, 2, 4, 128, 2>(ctx, a);
    if (t.bm == 128) return run_big<128, 128, 2, 2, 128, 2>(ctx, a);
    if (t.bn == 128) return run_big<64, 128, 2, 2, 128, 3>(ctx, a);
    return t.bm == 64 ? run_big<64, 64, 2, 2, 128, 4>(ctx, a) : run_big<32, 32, 2, 2, 128, 4>(ctx, a);
}

int launch_i8_dense(vdttfs_ctx* ctx, const I8Args& a) {
    if (a.M <= 0 || a.N <= 0) return VDTTFS_OK;
    const bool aligned = aligned16(a);
    const I8Tile t = i8_dense_tile(a.M, a.N, a.K, aligned);
    // as many rows a launch as its tiles allow: one tile of rows at least, with
    // VDTTFS_I8_MAX_N channels
    const int64_t rows = max_blocks(512) / ((a.N + t.bn - 1) / t.bn) * t.bm;
    for (int64_t m = 0; m < a.M; m += rows) {
        I8Args part = a;
        part.A += m * a.lda;
        part.sa += m;
        part.out = static_cast<char*>(a.out) + m * a.ldo * (a.out_elem == VDTTFS_ELEM_F32 ? 4 : 2);
        part.M = a.M - m < rows ? a.M - m : rows;
        VD_TRY(run_dense(ctx, part, t, aligned));
    }
    return VDTTFS_OK;
}

// Rows of the tiles of a layer's two products: the largest that an expert's
// rows fill on average, of which there are enough for the chip.
int i8_tile_rows(int64_t pairs, const vdttfs_expert_layer& L) {
    const int64_t mean = pairs / L.n_experts;
    const int k_min = L.d_in < L.d_hidden ? L.d_in : L.d_hidden;
    const int64_t hidden = L.gated ? 2 * (int64_t)L.d_hidden : L.d_hidden;
    auto enough = [&](int bm, int bn) {
        const int64_t rows = pairs / bm + L.n_experts / 2;
        return rows * ((hidden + bn - 1) / bn) >= 192 && rows * ((L.d_out + bn - 1) / bn) >= 192;
    };
    if (k_min >= kDeepK && mean >= 256 && enough(256, 256)) return 256;
    if (k_min >= kDeepK && mean >= 96 && enough(128, 128)) return 128;
    return mean >= 40 && enough(64, 64) ? 64 : 32;
}

template <int BM, int BN, int WM, int WN, int S, bool GATED>
int run_grouped(vdttfs_ctx* ctx, const I8Args& a) {
    constexpr int kOut = GATED ? BN / 2 : BN;
    const int64_t tn = (a.N + kOut - 1) / kOut, blocks = a.max_tiles * tn;
    if (blocks > max_blocks(WM * WN * 64))
        return set_error(VDTTFS_E_UNSUPPORTED, "experts: %lld tiles, at most %lld", (long long)blocks,
                         (long long)max_blocks(WM * WN * 64));
    if (S == 2 ? deep_ok(a) : aligned16(a) || a.K == 0) {  // of no terms nothing is read
        k_i8_big<BM, BN, WM, WN, 128, S, GATED, true>
            <<<dim3((unsigned)blocks), WM * WN * 64, 0, ctx->stream>>>(a, a.max_tiles, (int)tn);
    } else {
        if constexpr (BM > 32)
            return set_error(VDTTFS_E_UNSUPPORTED, "product of codes: rows off 16 bytes in large tiles");
        else
            k_i8_tile<BM, BN, WM, WN, GATED, true>
                <<<dim3((unsigned)blocks), WM * WN * 64, 0, ctx->stream>>>(a, (int)tn);
    }
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

template <bool GATED>
int run_grouped_rows(vdttfs_ctx* ctx, const I8Args& a, int bm) {
    if (bm == 256) return run_grouped<256, 256, 2, 4, 2, GATED>(ctx, a);
    if (bm == 128) return run_grouped<128, 128, 2, 2, 2, GATED>(ctx, a);
    if (bm == 64) return run_grouped<64, 64, 2, 2, 4, GATED>(ctx, a);
    return run_grouped<32, 64, 2, 2, 4, GATED>(ctx, a);
}

int launch_i8_grouped(vdttfs_ctx* ctx, const I8Args& a, bool gated, int bm) {
    if (a.max_tiles <= 0 || a.N <= 0) return VDTTFS_OK;
    return gated ? run_grouped_rows<true>(ctx, a, bm) : run_grouped_rows<false>(ctx, a, bm);
}

}  // namespace vdttfs
