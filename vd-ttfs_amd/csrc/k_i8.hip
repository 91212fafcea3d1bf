// Products of 8-bit codes on the matrix cores, dense and by expert.
//
// out[m][n] = act(float(sum_k A[m][k] B[n][k]) * sa[m] * sb[n] + bias[n]), the
// sum in 32-bit integers (v_mfma_i32_16x16x64_i8), so no order of k matters.
#include "elem.h"
#include "head.h"
#include "wave.h"

namespace vdttfs {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(1))) Bytes16 {
    v4i v;
};

// 16 codes at p, of which the first `valid` exist; the others are 0.  p may
// have any alignment (gfx950 loads 16 bytes from any address).
__device__ __forceinline__ v4i load16(const int8_t* p, int valid) {
    if (valid >= 16) return reinterpret_cast<const Bytes16*>(p)->v;
    v4i r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < valid) r[i >> 2] |= (int)(uint32_t)(uint8_t)p[i] << (8 * (i & 3));
    return r;
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
    __shared__ __align__(16) int8_t sA[BM * kBK];
    __shared__ __align__(16) int8_t sB[BN * kBK];

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
    v4i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};

    v4i ra[NA], rb[NB];
    auto fetch = [&](int k0) {
        const int valid = p.K - k0 - chunk;
#pragma unroll
        for (int i = 0; i < NA; ++i) ra[i] = load16(pa[i] + k0 + chunk, valid);
#pragma unroll
        for (int i = 0; i < NB; ++i) rb[i] = load16(pb[i] + k0 + chunk, valid);
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

    // A lane's four sums of a fragment: row m = lane & 15, channels
    // (lane >> 4) * 4 + 0..3.
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t m = m0 + wm + i * 16 + (lane & 15);
        if (m >= m_end) continue;
        const int64_t ar = GROUPED && p.a_rows ? p.a_rows[m] : m;
        const float sa = p.sa[ar];
        const int64_t orow = (GROUPED && p.o_rows ? p.o_rows[m] : m) * p.ldo;
#pragma unroll
        for (int j = 0; j < FN; j += GATED ? 2 : 1) {
            const int c = wn + j * 16 + (lane >> 4) * 4;
            const int n = n0 + (GATED ? (c >> 5) * 16 + (c & 15) : c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (n + e >= p.N) continue;
                float v = (float)acc[i][j][e] * sa * sb[n + e];
                if (bias) v += bias[n + e];
                v = apply_act(v, p.act);
                if constexpr (GATED) {
                    float u = (float)acc[i][j + 1][e] * sa * sb[p.N + n + e];
                    if (bias) u += bias[p.N + n + e];
                    v *= u;
                }
                store_elem(p.out, orow + n + e, v, p.out_elem);
            }
        }
    }
}

int check_grid(int64_t blocks) {
    if (blocks > 0x7fffffffll) return set_error(VDTTFS_E_UNSUPPORTED, "product of codes: too many tiles");
    return VDTTFS_OK;
}

}  // namespace

int launch_i8_dense(vdttfs_ctx* ctx, const I8Args& a) {
    if (a.M <= 0 || a.N <= 0) return VDTTFS_OK;
    const int tiles_n = (a.N + 63) / 64;
    const int64_t blocks = (a.M + 63) / 64 * tiles_n;
    VD_TRY(check_grid(blocks));
    k_i8_tile<64, 64, 2, 2, false, false><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, tiles_n);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int i8_tile_rows(int64_t pairs, int n_experts) {
    (void)pairs;
    (void)n_experts;
    return 64;
}

int launch_i8_grouped(vdttfs_ctx* ctx, const I8Args& a, bool gated, int bm) {
    if (a.max_tiles <= 0 || a.N <= 0) return VDTTFS_OK;
    (void)bm;
    const int out_n = gated ? 32 : 64;
    const int tiles_n = (a.N + out_n - 1) / out_n;
    const int64_t blocks = (int64_t)a.max_tiles * tiles_n;
    VD_TRY(check_grid(blocks));
    if (gated)
        k_i8_tile<64, 64, 2, 2, true, true><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, tiles_n);
    else
        k_i8_tile<64, 64, 2, 2, false, true><<<dim3((unsigned)blocks), 256, 0, ctx->stream>>>(a, tiles_n);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
