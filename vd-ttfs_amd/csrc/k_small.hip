// Products of few rows: the weights stream once from memory into the matrix
// instructions, and the rows are quantised inside the kernel, so a call is one
// launch (experts: two or three).
#include "codes.h"
#include "head.h"
#include "quant.h"

namespace vdttfs {
namespace {

constexpr int kCodes = kElemCodes;  // rows that are codes already
constexpr int kWaves = 8, kThreads = kWaves * 64;
constexpr int kAhead = 8;  // weight loads a wave has in flight
constexpr int kRows = 16;

// Who turns which values into codes: 2^lanes_log threads share a row, each
// with `turns` runs of eight of it, and the workgroup takes as many rows at a
// time as it has such teams.  All of it in kUnits runs a thread, or none.
struct Share {
    int lanes_log, turns, passes;
};
constexpr int kUnits = 2;
Share share_of(int rows, int K) {
    const int per = (K + 63) / 64 * 8;  // runs of a row, a multiple of eight
    int log = 3;
    while (log < 9 && (1 << log) < per) ++log;
    const int teams = kThreads >> log;
    return Share{log, (per + (1 << log) - 1) >> log, (rows + teams - 1) / teams};
}

// The workgroup turns rows into codes in LDS, `stride` bytes apart (zeros from
// K to the next 64), and their scales.  Every value is loaded once, all loads
// at once; a row's largest magnitude is a maximum over LDS of its bits (those
// of a NaN are above infinity's, and no order of maxima matters).  row(r):
// where row r starts in x.  Ends with a barrier.
template <int ELEM, typename RowAt>
__device__ __forceinline__ void rows_to_lds(const void* x, RowAt row, int rows, int K, Share sh, float tfs, int T,
                                            int8_t* to, int stride, float* scale, int* peak) {
    const int end = (K + 63) & ~63;
    if constexpr (ELEM == kCodes) {
        const int total = rows * (end / 16);
        for (int u = threadIdx.x; u < total; u += kThreads) {
            const int r = u / (end / 16), c = u % (end / 16) * 16;
            *reinterpret_cast<v4i*>(to + r * stride + c) = load16(static_cast<const int8_t*>(x) + row(r), c, K);
        }
        __syncthreads();
    } else {
        const int teams = kThreads >> sh.lanes_log, units = sh.passes * sh.turns;
        // run i of this thread: row r[i], column c[i]
        int r[kUnits], c[kUnits];
        {
            const int c0 = (threadIdx.x & ((1 << sh.lanes_log) - 1)) * 8, cstep = 8 << sh.lanes_log;
            int row_i = threadIdx.x >> sh.lanes_log, turn = 0;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                r[i] = row_i;
                c[i] = c0 + turn * cstep;
                const bool wrap = ++turn == sh.turns;
                turn = wrap ? 0 : turn;
                row_i += wrap ? teams : 0;
            }
        }
        auto there = [&](int i) __attribute__((always_inline)) { return i < units && r[i] < rows && c[i] < end; };
        // the same in a loop that is not unrolled
        auto each_again = [&](unsigned which, auto what) __attribute__((always_inline)) {
            const int c0 = (threadIdx.x & ((1 << sh.lanes_log) - 1)) * 8, cstep = 8 << sh.lanes_log;
            int at_r = threadIdx.x >> sh.lanes_log, at_c = c0;
#pragma unroll 1
            for (int i = 0; i < units; ++i) {
                if (which >> i & 1) what(at_r, at_c);
                at_c += cstep;
                if (at_c >= c0 + sh.turns * cstep) {
                    at_c = c0;
                    at_r += teams;
                }
            }
        };
        // A kernel that runs for some microseconds pays for every instruction
        // it fetches: unrolled is only what holds values in registers, and runs
        // that need more than that (the end of a row inside, a quotient near a
        // half) are loaded again in loops.
        Raw8<ELEM> raw[kUnits];
        unsigned ends = 0;  // runs that the row's end is inside of
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            raw[i] = nothing8<ELEM>();
            if (there(i)) {
                if (c[i] + 8 <= K) raw[i] = raw8<ELEM>(x, row(r[i]) + c[i]);
                else if (c[i] < K) ends |= 1u << i;
            }
        }
        auto put = [&](int r, int c, const int (&k)[8]) __attribute__((always_inline)) {
            *reinterpret_cast<uint2*>(to + r * stride + c) = pack8(k);
        };
        int k[8];
        float f[8];
        if constexpr (ELEM == VDTTFS_ELEM_TIMES) {
            const int levels = T < 127 ? T : 127;
            if ((int)threadIdx.x < rows) scale[threadIdx.x] = 1.0f / (float)levels;
            auto code = [&](int r, int c) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = time_code(f[e], tfs, T, levels);
                put(r, c, k);
            };
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (there(i)) {
                    unpack8<ELEM>(raw[i], f);
                    code(r[i], c[i]);
                }
            if (K & 7)
                each_again(ends, [&](int r, int c) __attribute__((always_inline)) {
                    load8<ELEM>(x, row(r), c, K, f);
                    code(r, c);
                });
        } else {
            if ((int)threadIdx.x < rows) peak[threadIdx.x] = 0;
            __syncthreads();
            auto magnitude = [&]() __attribute__((always_inline)) {
                int a = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) a = max(a, __float_as_int(f[e]) & 0x7fffffff);
                return a;
            };
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (i < units) {
                    unpack8<ELEM>(raw[i], f);
                    int a = magnitude();
                    // eight lanes are on one row (or past the last, with zeros)
                    a = max(a, __builtin_amdgcn_update_dpp(a, a, 0xB1, 0xf, 0xf, false));
                    a = max(a, __builtin_amdgcn_update_dpp(a, a, 0x4E, 0xf, 0xf, false));
                    a = max(a, __builtin_amdgcn_update_dpp(a, a, 0x141, 0xf, 0xf, false));
                    if ((threadIdx.x & 7) == 0 && a > 0) atomicMax(&peak[r[i]], a);
                }
            if (K & 7)
                each_again(ends, [&](int r, int c) __attribute__((always_inline)) {
                    load8<ELEM>(x, row(r), c, K, f);
                    atomicMax(&peak[r], magnitude());
                });
            __syncthreads();
            if ((int)threadIdx.x < rows) scale[threadIdx.x] = scale_of(__int_as_float(peak[threadIdx.x]));
            __syncthreads();
            unsigned again = ends;
#pragma unroll
            for (int i = 0; i < kUnits; ++i)
                if (there(i)) {
                    unpack8<ELEM>(raw[i], f);
                    if (codes8_fast(f, coder_of(scale[r[i]]), k)) again |= 1u << i;
                    put(r[i], c[i], k);
                }
            if (__any(again != 0))
                each_again(again, [&](int r, int c) __attribute__((always_inline)) {
                    load8<ELEM>(x, row(r), c, K, f);
                    codes8_exact(f, coder_of(scale[r]), k);
                    put(r, c, k);
                });
        }
        __syncthreads();
    }
}

// The codes of a row lie `stride` bytes apart: K rounded up to 64, and 16 more,
// so that 16 rows read at one place come from different banks.
__host__ __device__ __forceinline__ int lds_stride(int K) { return ((K + 63) & ~63) + 16; }

// One of `of` parts of K for PARTS runs of 16 channels (a lane holds 16 codes of
// channel lane & 15 at a time): its first loads are issued by begin(), before
// anything waits for the rows.  The last K % 64 codes are the last part's.
template <int PARTS>
struct Weights {
    static constexpr int kHeld = kAhead / PARTS;
    const int8_t* row[PARTS];
    v4i ahead[PARTS][kHeld], tail[PARTS];
    int first, last, K, at_tail;  // steps of 64 codes

    __device__ __forceinline__ void begin(int K_, int part, int of) {
        K = K_;
        const int steps = K / 64, per = (steps + of - 1) / of, g = (lane_id() >> 4) * 16;
        first = part * per;
        last = first + per < steps ? first + per : steps;
        at_tail = part == of - 1 && K > steps * 64 ? steps * 64 : -1;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) row[p] += g;
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                if (first + i < last)
                    ahead[p][i] = reinterpret_cast<const Bytes16*>(row[p] + (first + i) * 64)->v;
        if (at_tail >= 0) {
#pragma unroll 1
            for (int p = 0; p < PARTS; ++p) {
                const v4i t = load16(row[p] - g, at_tail + g, K);
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    if (q == p) tail[q] = t;
            }
        }
    }
    // acc[p] += channels x rows; rows: the lane's row of codes (lane & 15), zeros
    // in its place unless `keep`
    __device__ __forceinline__ void multiply(const int8_t* rows, v4i (&acc)[PARTS], bool keep = true) const {
        rows += (lane_id() >> 4) * 16;
        auto codes = [&](int k) __attribute__((always_inline)) {
            const v4i a = *reinterpret_cast<const v4i*>(rows + k);
            return keep ? a : v4i{0, 0, 0, 0};
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (first + i < last) {
                const v4i a = codes((first + i) * 64);
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    acc[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ahead[p][i], a, acc[p], 0, 0, 0);
            }
#pragma unroll 2
        for (int s = first + kHeld; s < last; ++s) {
            const v4i a = codes(s * 64);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                acc[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    reinterpret_cast<const Bytes16*>(row[p] + s * 64)->v, a, acc[p], 0, 0, 0);
        }
        if (at_tail >= 0) {
            const v4i a = codes(at_tail);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                acc[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(tail[p], a, acc[p], 0, 0, 0);
        }
    }
};

// Sum of the waves' parts for output (row m, channel n) of a 16 x 16 tile.
__device__ __forceinline__ int gather(const int* part, int m, int n) {
    int v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += part[w * 256 + (m + 16 * (n >> 2)) * 4 + (n & 3)];
    return v;
}

struct SmallArgs {
    const void* x;
    int64_t ldx;
    const float* sa;  // scales of rows that are codes already
    const int8_t* w;
    int64_t ldw;
    const float* sb;
    const float* bias;
    void* out;
    int64_t ldo;
    int64_t M;
    int N, K, act, out_elem;
    float tfs;
    int T;
    Share sh;
};

// 16 rows x 16 channels a workgroup, its eight waves sharing K.
template <int ELEM>
__global__ __launch_bounds__(kThreads) void k_i8_small(SmallArgs p) {
    extern __shared__ __align__(16) int8_t codes[];
    __shared__ int part[kWaves * 256];
    __shared__ float scale[kRows];
    __shared__ int peak[kRows];
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), stride = lds_stride(p.K);
    const int n0 = blockIdx.x * 16;
    const int64_t m0 = (int64_t)blockIdx.y * kRows;
    const int rows = p.M - m0 < kRows ? (int)(p.M - m0) : kRows;
    Weights<1> w;
    {
        const int n = n0 + (lane & 15);
        w.row[0] = p.w + (int64_t)(n < p.N ? n : p.N - 1) * p.ldw;
    }
    w.begin(p.K, wave, kWaves);
    if (ELEM == kCodes && (int)threadIdx.x < rows) scale[threadIdx.x] = p.sa[m0 + threadIdx.x];
    rows_to_lds<ELEM>(p.x, [&](int r) { return (m0 + r) * p.ldx; }, rows, p.K, p.sh, p.tfs, p.T, codes, stride,
                      scale, peak);
    const int r = lane & 15;
    v4i acc[1] = {v4i{0, 0, 0, 0}};
    w.multiply(codes + (r < rows ? r : rows - 1) * stride, acc);
    *reinterpret_cast<v4i*>(part + wave * 256 + lane * 4) = acc[0];
    __syncthreads();
    const int m = threadIdx.x >> 4, n = threadIdx.x & 15;
    if (m < rows && n0 + n < p.N) {
        float v = (float)gather(part, m, n) * scale[m] * p.sb[n0 + n];
        if (p.bias) v += p.bias[n0 + n];
        store_elem(p.out, (m0 + m) * p.ldo + n0 + n, apply_act(v, p.act), p.out_elem);
    }
}

// ---- experts of few pairs ---------------------------------------------------------
// No sort and no tiles: a workgroup finds the pairs (row, slot) of its expert by
// looking through the whole idx, at most kMaxPairs of them.  blockIdx.y names
// the expert where there are no more experts than pairs; else it names a pair,
// and the first pair of an expert stands for it.
constexpr int kMaxPairs = 512;
struct PairArgs {
    const int32_t* idx;
    int pairs, top_k, n_experts, by_pair;
};

// The pairs of the workgroup's expert, in order, to list; their number, 0 where
// another workgroup has them.
__device__ __forceinline__ int find_pairs(const PairArgs& a, int* list, int* counts, int* expert) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    const int e = a.by_pair ? a.idx[blockIdx.y] : (int)blockIdx.y;
    *expert = e;
    if (e < 0 || e >= a.n_experts) return 0;  // the same in every thread
    int before = 0;
    for (int p0 = 0; p0 < a.pairs; p0 += kThreads) {
        const int p = p0 + threadIdx.x;
        const bool mine = p < a.pairs && a.idx[p] == e;
        const uint64_t m = __ballot(mine);
        if (lane == 0) counts[wave] = __popcll(m);
        __syncthreads();
        int at = before;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += counts[w];
            before += counts[w];
        }
        if (mine) list[at + __popcll(m & lanemask_lt())] = p;
        __syncthreads();
    }
    if (a.by_pair && list[0] != (int)blockIdx.y) return 0;
    return before;
}

struct ExpertArgs {
    PairArgs pairs;
    const void* x;
    int64_t ldx;
    const float* sa;  // scales of rows that are codes already
    const int8_t* w;  // [E][channels][K]
    const float* sb;  // [E][channels]
    const float* bias;
    float* out;  // [pairs][N]
    int N, K, act, channels;
    float tfs;
    int T;
    int cap;  // rows at a time
    Share sh;  // of so many
};

// The experts' first product: out[pair] for 16 columns (of gate and up if
// GATED) of the rows of one expert, `cap` at a time, every gridDim.z-th here.
template <int ELEM, bool GATED>
__global__ __launch_bounds__(kThreads) void k_expert_small(ExpertArgs p) {
    extern __shared__ __align__(16) int8_t codes[];
    constexpr int kParts = GATED ? 2 : 1;
    __shared__ int part[kParts * kWaves * 256];
    __shared__ float scale[kRows];
    __shared__ int peak[kRows];
    __shared__ int list[kMaxPairs];
    __shared__ int counts[kWaves];
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), stride = lds_stride(p.K);
    int e;
    const int n_rows = find_pairs(p.pairs, list, counts, &e);
    const int n0 = blockIdx.x * 16;
    if ((int)blockIdx.z * p.cap >= n_rows) return;
    const int64_t ch0 = (int64_t)e * p.channels;
    Weights<kParts> w;
    {
        const int n = n0 + (lane & 15) < p.N ? n0 + (lane & 15) : p.N - 1;
#pragma unroll
        for (int q = 0; q < kParts; ++q) w.row[q] = p.w + (ch0 + n + q * p.N) * p.K;
    }
    w.begin(p.K, wave, kWaves);
    for (int r0 = blockIdx.z * p.cap; r0 < n_rows; r0 += gridDim.z * p.cap) {
        const int rows = n_rows - r0 < p.cap ? n_rows - r0 : p.cap;
        auto x_row = [&](int r) { return list[r0 + r] / p.pairs.top_k; };
        if (ELEM == kCodes && (int)threadIdx.x < rows) scale[threadIdx.x] = p.sa[x_row(threadIdx.x)];
        rows_to_lds<ELEM>(p.x, [&](int r) { return (int64_t)x_row(r) * p.ldx; }, rows, p.K, p.sh, p.tfs, p.T, codes,
                          stride, scale, peak);
        const int r = lane & 15;
        v4i acc[kParts];
#pragma unroll
        for (int q = 0; q < kParts; ++q) acc[q] = v4i{0, 0, 0, 0};
        w.multiply(codes + (r < rows ? r : rows - 1) * stride, acc);
#pragma unroll
        for (int q = 0; q < kParts; ++q)
            *reinterpret_cast<v4i*>(part + (q * kWaves + wave) * 256 + lane * 4) = acc[q];
        __syncthreads();
        const int m = threadIdx.x >> 4, n = threadIdx.x & 15;
        if (m < rows && n0 + n < p.N) {
            const int64_t ch = ch0 + n0 + n;
            float v = (float)gather(part, m, n) * scale[m] * p.sb[ch];
            if (p.bias) v += p.bias[ch];
            v = apply_act(v, p.act);
            if constexpr (GATED) {
                float u = (float)gather(part + kWaves * 256, m, n) * scale[m] * p.sb[ch + p.N];
                if (p.bias) u += p.bias[ch + p.N];
                v *= u;
            }
            p.out[(int64_t)list[r0 + m] * p.N + n0 + n] = v;
        }
        __syncthreads();
    }
}

// The experts' second product and its sum over the slots: out for 16 columns of
// a few rows, whose pairs (16 at most) are the rows of one fragment.  Their
// experts, each once, are shared out over the waves, and K too where there are
// fewer; a pair's codes count in the products of its own expert alone, so one
// accumulator serves them all.
struct OutArgs {
    const void* h;  // [pairs][K]
    int64_t ldh;
    const float* sa;  // scales of rows that are codes already
    const int8_t* w;  // [E][N][K]
    const float* sb;  // [E][N]
    const float* bias;
    const int32_t* idx;
    const float* wt;
    void* out;
    int64_t ldo;
    int64_t M;
    int out_elem, N, K, top_k, n_experts;
    int m_rows;  // rows of a workgroup
    Share sh;
};

template <int ELEM>
__global__ __launch_bounds__(kThreads) void k_expert_out(OutArgs p) {
    extern __shared__ __align__(16) int8_t codes[];
    __shared__ int part[kWaves * 256];
    __shared__ float scale[kRows];
    __shared__ int peak[kRows];
    __shared__ float z[kRows][17];
    const int lane = lane_id(), wave = uniform(threadIdx.x >> 6), stride = lds_stride(p.K);
    const int n0 = blockIdx.x * 16;
    const int64_t m0 = (int64_t)blockIdx.y * p.m_rows, q0 = m0 * p.top_k;
    const int m_here = p.M - m0 < p.m_rows ? (int)(p.M - m0) : p.m_rows, pairs = m_here * p.top_k;
    // the expert of pair lane & 15, -1 where it has none
    int e = (lane & 15) < pairs ? p.idx[q0 + (lane & 15)] : -1;
    if (e < 0 || e >= p.n_experts) e = -1;
    int distinct = 0;
    uint32_t firsts = 0;  // the first pair of each expert
    for (int j = 0; j < pairs; ++j) {
        const int ej = __builtin_amdgcn_readlane(e, j);
        const uint32_t same = (uint32_t)__ballot(e == ej) & 0xffff;
        if (ej >= 0 && __builtin_ctz(same) == j) {
            firsts |= 1u << j;
            ++distinct;
        }
    }
    // expert number d (by its first pair); -1: the wave has none
    auto expert_of = [&](int d) __attribute__((always_inline)) {
        uint32_t left = firsts;
        for (; d > 0; --d) left &= left - 1;
        return __builtin_amdgcn_readlane(e, __builtin_ctz(left));
    };
    const int parts = distinct > 0 && distinct < kWaves ? kWaves / distinct : 1;
    const int share = distinct < kWaves ? distinct : kWaves;  // waves of one part
    const int my_part = share > 0 ? wave / share : parts;
    int d = share > 0 ? wave % share : 0;
    const int n_lane = n0 + (lane & 15) < p.N ? n0 + (lane & 15) : p.N - 1;
    Weights<1> w;
    int my_e = -1;
    auto begin = [&]() __attribute__((always_inline)) {
        my_e = expert_of(d);
        w.row[0] = p.w + ((int64_t)my_e * p.N + n_lane) * p.K;
        w.begin(p.K, my_part, parts);
    };
    if (my_part < parts) begin();
    // what thread (pair, column) needs at the end
    const int pair = threadIdx.x >> 4, n = n0 + (threadIdx.x & 15);
    float sb = 0.0f, bias = 0.0f, wt = 0.0f;
    int pe = -1;
    if (pair < pairs && n < p.N) {
        pe = p.idx[q0 + pair];
        if (pe >= 0 && pe < p.n_experts) {
            sb = p.sb[(int64_t)pe * p.N + n];
            if (p.bias) bias = p.bias[(int64_t)pe * p.N + n];
            wt = p.wt[q0 + pair];
        } else {
            pe = -1;
        }
    }
    if (ELEM == kCodes && (int)threadIdx.x < pairs) scale[threadIdx.x] = p.sa[q0 + threadIdx.x];
    rows_to_lds<ELEM>(p.h, [&](int r) { return (q0 + r) * p.ldh; }, pairs, p.K, p.sh, 0.0f, 1, codes, stride, scale,
                      peak);
    v4i acc[1] = {v4i{0, 0, 0, 0}};
    if (my_part < parts) {
        const int r = lane & 15;
        const int8_t* row = codes + (r < pairs ? r : 0) * stride;
        w.multiply(row, acc, e == my_e);
        for (d += kWaves; d < distinct; d += kWaves) {
            begin();
            w.multiply(row, acc, e == my_e);
        }
    }
    *reinterpret_cast<v4i*>(part + wave * 256 + lane * 4) = acc[0];
    __syncthreads();
    if (pair < kRows) {
        float v = 0.0f;
        if (pe >= 0) {
            v = (float)gather(part, pair, threadIdx.x & 15) * scale[pair] * sb;
            if (p.bias) v += bias;
            v *= wt;
        }
        z[pair][threadIdx.x & 15] = v;
    }
    __syncthreads();
    if (pair < m_here && n < p.N) {  // a row here
        float sum = 0.0f;
        for (int j = 0; j < p.top_k; ++j) sum += z[pair * p.top_k + j][threadIdx.x & 15];
        store_elem(p.out, (m0 + pair) * p.ldo + n, sum, p.out_elem);
    }
}

}  // namespace

// Few rows, or layers so small that launches count.  Every workgroup quantises
// its rows, some 1.1 us for each run of eight a thread has, so two at most; past
// that a launch of its own does it (5x4096x4096 of BF16: 12.3 us, so 9.8).
// Measured (us, against quantisation and tiles): 1x4096x4096 of BF16 6.7, 11.2;
// 16x512x512 5.5, 7.3; 128x512x512 5.6, 7.4; 256x512x512 7.7, 6.8, of spike
// times 5.7, 7.2, 512 rows of them 8.6, 6.9.  Codes, 1x4096x4096: 5.2 (3.2 TB/s
// of weights, and a launch), tiles 7.5; 5 rows 5.8, 7.6.  Long rows of codes
// leave a CU one workgroup, which the tiles beat (64x64x8192: 17.8, 16.0) unless
// rows off 16 bytes take them through registers (215x57x7276: 15.4, 28.6;
// 26x3942x7254: 33, 38; 100x1000x1003: 5.5, 6.8).
bool small_ok(int64_t M, int N, int K, int elem, bool off16) {
    const int64_t rows = M < kRows ? M : kRows;
    const Share sh = share_of((int)rows, K);
    if (elem != kElemCodes && sh.passes * sh.turns > kUnits) return false;
    if (rows * lds_stride(K) > (elem == kElemCodes && off16 ? 144 : 56) * 1024) return false;
    const int64_t blocks = (M + kRows - 1) / kRows * ((N + 15) / 16);
    return M <= kRows || blocks <= (elem == VDTTFS_ELEM_TIMES || (elem == kElemCodes && off16) ? 512 : 256);
}

int launch_i8_small(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, const float* sa, const I8Args& a) {
    const SmallArgs p{x,    ldx, sa,  a.B, a.ldb, a.sb,       a.bias,     a.out,      a.ldo,
                      a.M,  a.N, a.K, a.act, a.out_elem, ctx->c.tfs, ctx->c.T,
                      share_of((int)(a.M < kRows ? a.M : kRows), a.K)};
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + kRows - 1) / kRows));
    const int rows = a.M < kRows ? (int)a.M : kRows;
    const size_t lds = (size_t)rows * lds_stride(a.K);
    switch (elem) {
        case VDTTFS_ELEM_F32: k_i8_small<VDTTFS_ELEM_F32><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_BF16: k_i8_small<VDTTFS_ELEM_BF16><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_F16: k_i8_small<VDTTFS_ELEM_F16><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_TIMES: k_i8_small<VDTTFS_ELEM_TIMES><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        default: k_i8_small<kCodes><<<grid, kThreads, lds, ctx->stream>>>(p);
    }
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

// Rows that a workgroup of the experts' kernels takes at a time, 0 where none.
static int expert_rows(int64_t pairs, int K, bool codes) {
    for (int rows = pairs < kRows ? (int)pairs : kRows; rows > 0; rows /= 2) {
        const Share sh = share_of(rows, K);
        if ((codes || sh.passes * sh.turns <= kUnits) && rows * lds_stride(K) <= 32 * 1024) return rows;
    }
    return 0;
}

// Every workgroup reads all experts of its rows' pairs, and quantises the pairs
// if `fuse`, so it pays while there are few; else the pairs are sorted.  Measured
// (us, joined and, before the sort was as fast, with launches of their own for
// product and sum; workgroups, MB of weights read):
//   1 x 6 of 64, 1024-512-1024 gated (64, 3)      11.6  13.2
//   256 x 2 of 8, 512-512-10 (32, 2)              17.2  19.3
//   16 x 16 of 64, 512-512-512 (512, 64)          29.5  31.9
//   40 x 4 of 32, 512-2048-512 (320, 160)         56.1  40.6
//   256 x 2 of 8, 512-512-512 gated (1024, 64)    28.9  23.3
static bool expert_out_ok(int64_t pairs, int top_k, const vdttfs_expert_layer& L, bool fuse) {
    if (top_k > kRows) return false;
    const int rows = (pairs < kRows ? (int)pairs : kRows) / top_k * top_k;
    const int64_t blocks = (pairs + rows - 1) / rows * ((L.d_out + 15) / 16);
    if (blocks > 512 || blocks * (rows < L.n_experts ? rows : L.n_experts) * 16 * L.d_hidden > 64 << 20) return false;
    const Share sh = share_of(rows, L.d_hidden);
    if (fuse && sh.passes * sh.turns > kUnits) return false;
    return rows * lds_stride(L.d_hidden) <= 48 * 1024;
}

// Measured (us; rows x slots of experts, d_in-d_hidden-d_out; quantising in the
// products, before them, and sorted with tiles):
//   1 x 6 of 64, 1024-512-1024 gated   11.4  15.7  21.8
//   32 x 2 of 8, 512-512-512           14.7  16.6  21.9 (the second before: 14.1)
//   256 x 2 of 8, 512-512-10           22.9  18.9  23.5 (the first before: 17.2)
// Past two workgroups a CU in the first product, sorted tiles are as good or
// better, but for one row, which shares no weights (these kernels, and tiles;
// the tiles have since lost another 3 us):
//   2 x 4 of 16, 2048-1024-2048 gated (512 workgroups)    19.0  27.1
//   4 x 2 of 8, 4096-1024-4096 gated (512)                27.2  34.8
//   16 x 2 of 16, 2048-1024-2048 gated (1024)             41.4  35.3
//   32 x 4 of 32, 512-512-512 (1024)                      22.8  23.8
//   128 x 4 of 64, 512-512-512 gated (2048)               37.2  30.5
//   1 x 4 of 8, 4096-4096-4096 gated (1024)               55.9  65.9
//   1 x 8 of 128, 4096-2048-4096 gated (1024)             59.7  57.1
bool experts_small_ok(int64_t pairs, int top_k, const vdttfs_expert_layer& L, bool* fuse1, bool* fuse2) {
    // every 16 columns quantise an expert's rows again
    auto fuse = [&](int K, int N) { return pairs * K <= 32768 || N <= 32; };
    *fuse1 = fuse(L.d_in, L.d_hidden) && expert_rows(pairs, L.d_in, false) > 0;
    *fuse2 = fuse(L.d_hidden, L.d_out) && expert_out_ok(pairs, top_k, L, true);
    const int64_t blocks = (pairs < L.n_experts ? pairs : L.n_experts) * ((L.d_hidden + 15) / 16);
    if (pairs > kMaxPairs || (blocks > 512 && pairs > top_k)) return false;
    return expert_rows(pairs, L.d_in, !*fuse1) > 0 && expert_out_ok(pairs, top_k, L, *fuse2);
}

template <bool GATED>
static void expert_elem(vdttfs_ctx* ctx, const ExpertArgs& p, int elem, dim3 grid, size_t lds) {
    switch (elem) {
        case VDTTFS_ELEM_F32: k_expert_small<VDTTFS_ELEM_F32, GATED><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_BF16: k_expert_small<VDTTFS_ELEM_BF16, GATED><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_F16: k_expert_small<VDTTFS_ELEM_F16, GATED><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        case VDTTFS_ELEM_TIMES: k_expert_small<VDTTFS_ELEM_TIMES, GATED><<<grid, kThreads, lds, ctx->stream>>>(p); break;
        default: k_expert_small<kCodes, GATED><<<grid, kThreads, lds, ctx->stream>>>(p);
    }
}

int launch_expert_product(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, const float* sa, const int32_t* idx,
                          int64_t pairs, int top_k, const vdttfs_expert_layer& L, float* out) {
    const bool by_pair = pairs < L.n_experts;
    const PairArgs pa{idx, (int)pairs, top_k, L.n_experts, by_pair};
    const unsigned y = (unsigned)(by_pair ? pairs : L.n_experts);
    const int K = L.d_in, N = L.d_hidden;
    if (N <= 0) return VDTTFS_OK;
    const int cap = expert_rows(pairs, K, elem == kCodes);
    const ExpertArgs p{pa,  x, ldx, sa,    L.w1,  L.s1, L.b1, out, N, K, L.act, L.gated ? 2 * N : N, ctx->c.tfs,
                       ctx->c.T, cap, share_of(cap, K)};
    // parts of an expert's rows: as many as its mean needs, while the chip holds
    // all workgroups at once
    const unsigned cols = (unsigned)((N + 15) / 16), want = (unsigned)((pairs / y + cap - 1) / cap);
    const unsigned room = 512 / (cols * y);
    const dim3 grid(cols, y, want < room ? want : room > 0 ? room : 1);
    const size_t lds = (size_t)cap * lds_stride(K);
    if (L.gated) expert_elem<true>(ctx, p, elem, grid, lds);
    else expert_elem<false>(ctx, p, elem, grid, lds);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_expert_out(vdttfs_ctx* ctx, const void* h, bool is_codes, int64_t ldh, const float* sa, const int32_t* idx,
                      const float* wt, int64_t M, int top_k, const vdttfs_expert_layer& L, void* out, int out_elem,
                      int64_t ldo) {
    int m_rows = kRows / top_k;
    if (M < m_rows) m_rows = (int)M;
    const OutArgs p{h,   ldh, sa, L.w2,     L.s2,    L.b2,       idx,   wt,          out,
                    ldo, M,   out_elem, L.d_out, L.d_hidden, top_k, L.n_experts, m_rows,
                    share_of(m_rows * top_k, L.d_hidden)};
    const dim3 grid((unsigned)((L.d_out + 15) / 16), (unsigned)((M + m_rows - 1) / m_rows));
    const size_t lds = (size_t)m_rows * top_k * lds_stride(L.d_hidden);
    if (is_codes) k_expert_out<kCodes><<<grid, kThreads, lds, ctx->stream>>>(p);
    else k_expert_out<VDTTFS_ELEM_F32><<<grid, kThreads, lds, ctx->stream>>>(p);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
