// Rows to the order of their experts and back, and the gradients of both.
//
// A pair is (row m, slot j), number m * top_k + j; its place is its rank among
// the pairs with an expert, by expert and then by number.  Rows move as they are;
// sums over slots are in 32 bits, in the order of the slots.
#include <algorithm>
#include <type_traits>

#include "elem.h"
#include "head.h"
#include "mx4.h"
#include "quant.h"
#include "sort.h"
#include "wave.h"

namespace vdttfs {
namespace {

constexpr int kPairs = 2048;  // pairs of a workgroup of the sort
constexpr int kWaves = 16;    // of such a workgroup
constexpr int kEachPairs = 16384;  // pairs of which every workgroup counts all
constexpr int kSumBlocks = 512;  // workgroups that sum the counts by themselves

__device__ __forceinline__ int expert_of(const PlaceArgs& a, int64_t q, int64_t pairs) {
    const int e = q < pairs ? a.idx[q] : -1;
    return e >= 0 && e < a.E ? e : -1;
}

// The lanes with this lane's value of 0 <= e < E (none where e is below 0).
__device__ __forceinline__ uint64_t lanes_like(int e, int bits) {
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
        const bool on = e >> b & 1;
        const uint64_t with = __ballot(on);
        same &= on ? with : ~with;
    }
    return e >= 0 ? same : 0;
}

// Pairs of each workgroup by expert: hist[block][expert].
__global__ __launch_bounds__(1024) void k_place_count(PlaceArgs a, int* __restrict__ hist) {
    __shared__ int h[kMaxExperts];
    const int64_t pairs = a.M * a.top_k, q0 = (int64_t)blockIdx.x * kPairs + threadIdx.x;
    const int e0 = expert_of(a, q0, pairs), e1 = expert_of(a, q0 + 1024, pairs);
    if ((int)threadIdx.x < a.E) h[threadIdx.x] = 0;
    __syncthreads();
    if (e0 >= 0) atomicAdd(&h[e0], 1);
    if (e1 >= 0) atomicAdd(&h[e1], 1);
    __syncthreads();
    if ((int)threadIdx.x < a.E) hist[(int64_t)blockIdx.x * a.E + threadIdx.x] = h[threadIdx.x];
}

// One workgroup: hist[block][expert] becomes the place of the block's first pair
// of the expert.  2^log threads go over the experts, and share the blocks in
// 1024 >> log runs.
__global__ __launch_bounds__(1024) void k_place_scan(PlaceArgs a, int* __restrict__ hist, int blocks, int log) {
    __shared__ int lds[16];
    __shared__ int sums[1024];
    __shared__ int starts[kMaxExperts];
    const int e = threadIdx.x & ((1 << log) - 1), run = threadIdx.x >> log, runs = 1024 >> log;
    const int per = (blocks + runs - 1) / runs;
    const int b0 = run * per < blocks ? run * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
    int n = 0;
    if (e < a.E)
#pragma unroll 4
        for (int b = b0; b < b1; ++b) n += hist[(int64_t)b * a.E + e];
    sums[threadIdx.x] = n;
    __syncthreads();
    int total = 0;
    if (run == 0)
        for (int r = 0; r < runs; ++r) total += sums[(r << log) + e];
    int all;
    const int first = block_excl_scan(total, lds, &all);
    if (run == 0) starts[e] = first;
    if (a.start && run == 0 && e < a.E) a.start[e] = first;
    if (a.start && threadIdx.x == 0) a.start[a.E] = all;
    __syncthreads();
    if (e >= a.E) return;
    int at = starts[e];
    for (int r = 0; r < run; ++r) at += sums[(r << log) + e];
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int64_t i = (int64_t)b * a.E + e;
        const int h = hist[i];
        hist[i] = at;
        at += h;
    }
}

// The places of a workgroup's pairs: each wave has N runs of 64 neighbouring ones,
// counts them by expert, adds what the waves before it have, and ranks a run's lanes
// among themselves.  first(), called by all threads: the place of the workgroup's first
// pair of expert threadIdx.x (unused from E on).
template <int N, class F>
__device__ __forceinline__ void place_block(const PlaceArgs& a, int64_t q0, int* at, int bits, const F& first) {
    const int64_t pairs = a.M * a.top_k;
    const int wave = threadIdx.x >> 6, lane = lane_id();
    q0 += wave * (N * 64) + lane;
    int e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = expert_of(a, q0 + 64 * i, pairs);
    for (int i = threadIdx.x; i < kWaves * a.E; i += 1024) at[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (e[i] >= 0) atomicAdd(&at[wave * a.E + e[i]], 1);
    __syncthreads();
    int sum = first();
    if ((int)threadIdx.x < a.E)
        for (int w = 0; w < kWaves; ++w) {
            const int n = at[w * a.E + threadIdx.x];
            at[w * a.E + threadIdx.x] = sum;
            sum += n;
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t same = lanes_like(e[i], bits);
        const int rank = __popcll(same & lanemask_lt());
        int to = -1;
        if (e[i] >= 0) to = at[wave * a.E + e[i]] + rank;
        wave_sync();  // read by all before the first of them moves it on
        if (e[i] >= 0 && rank == 0) at[wave * a.E + e[i]] = to + __popcll(same);
        wave_sync();
        if (q0 + 64 * i < pairs) a.place[q0 + 64 * i] = to;
    }
}

// ... from the scanned counts.
__global__ __launch_bounds__(1024) void k_place(PlaceArgs a, const int* __restrict__ hist, int bits) {
    extern __shared__ int at[];  // [kWaves][E]
    place_block<kPairs / 1024>(a, (int64_t)blockIdx.x * kPairs, at, bits, [&] {
        return (int)threadIdx.x < a.E ? hist[(int64_t)blockIdx.x * a.E + threadIdx.x] : 0;
    });
}

// ... from the counts, which every workgroup sums by itself: one launch less.  2^bits
// threads go over the experts, and share the blocks.
__global__ __launch_bounds__(1024) void k_place_sum(PlaceArgs a, const int* __restrict__ hist, int blocks, int bits) {
    extern __shared__ int at[];
    __shared__ int before[1024], total[1024];
    __shared__ int lds[16];
    place_block<kPairs / 1024>(a, (int64_t)blockIdx.x * kPairs, at, bits, [&] {
        const int e = threadIdx.x & ((1 << bits) - 1), run = threadIdx.x >> bits, runs = 1024 >> bits;
        int mine = 0, all = 0;
        if (e < a.E)
#pragma unroll 4
            for (int b = run; b < blocks; b += runs) {
                const int n = hist[b * a.E + e];
                all += n;
                mine += b < (int)blockIdx.x ? n : 0;
            }
        before[threadIdx.x] = mine;
        total[threadIdx.x] = all;
        __syncthreads();
        mine = all = 0;
        if (run == 0)
            for (int r = 0; r < runs; ++r) {
                mine += before[(r << bits) + e];
                all += total[(r << bits) + e];
            }
        int used;
        const int start = block_excl_scan(all, lds, &used);
        if (blockIdx.x == 0 && a.start) {
            if ((int)threadIdx.x < a.E) a.start[threadIdx.x] = start;
            if (threadIdx.x == 0) a.start[a.E] = used;
        }
        return start + mine;
    });
}

// ... from all pairs, which every workgroup counts by itself: no launch before it, and
// no scratch.
__global__ __launch_bounds__(1024) void k_place_each(PlaceArgs a, int bits) {
    extern __shared__ int at[];
    __shared__ int before[kMaxExperts], total[kMaxExperts];
    __shared__ int lds[16];
    const int64_t q0 = (int64_t)blockIdx.x * kPairs;
    place_block<kPairs / 1024>(a, q0, at, bits, [&] {
        const int pairs = (int)(a.M * a.top_k);
        before[threadIdx.x] = total[threadIdx.x] = 0;
        __syncthreads();
        for (int q = threadIdx.x; q < pairs; q += 4 * 1024) {
            int e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = expert_of(a, q + i * 1024, pairs);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e[i] >= 0) atomicAdd(q + i * 1024 < q0 ? &before[e[i]] : &total[e[i]], 1);
        }
        __syncthreads();
        const int mine = before[threadIdx.x];
        int used;
        const int start = block_excl_scan(mine + total[threadIdx.x], lds, &used);
        if (blockIdx.x == 0 && a.start) {
            if ((int)threadIdx.x < a.E) a.start[threadIdx.x] = start;
            if (threadIdx.x == 0) a.start[a.E] = used;
        }
        return start + mine;
    });
}

// A row's bytes to another; both may start anywhere that their type allows.
// A workgroup reads a row once and writes it to its slots.  Bound by memory: 16384 x 8
// rows of 2048 BF16 109 us, 0.6 GB at 5.5 TB/s.  Rows off 16 bytes keep to the caches,
// where neighbours' parts of a line meet (16384 x 8 of 2047 with their places 145 us,
// past them 161; 4412 x 6 of 2427 46 and 45).
constexpr int kCopy = 256;
template <bool PAST>
__device__ __forceinline__ void copy_to_slots(void* z, int64_t ld_bytes, const void* x_row, int64_t bytes, int unit,
                                              const int* place, int n, int64_t rows) {
    const char* from = static_cast<const char*>(x_row);
    const int64_t whole = bytes / 16 * 16;
    for (int64_t b = (int64_t)threadIdx.x * 16; b < whole; b += kCopy * 16) {
        const v4u v = reinterpret_cast<const AnyUint4*>(from + b)->v;
        for (int j = 0; j < n; ++j) {
            const int p = place[j];
            if (p < 0 || p >= rows) continue;
            char* to = static_cast<char*>(z) + p * ld_bytes + b;
            if (PAST) put16(to, v);
            else reinterpret_cast<AnyUint4*>(to)->v = v;
        }
    }
    for (int64_t b = whole + (int64_t)threadIdx.x * unit; b < bytes; b += kCopy * unit)
        for (int j = 0; j < n; ++j) {
            const int p = place[j];
            if (p < 0 || p >= rows) continue;
            char* to = static_cast<char*>(z) + p * ld_bytes + b;
            if (unit == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from + b);
            else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from + b);
        }
}
template <bool PAST>
__global__ __launch_bounds__(kCopy) void k_dispatch_rows(PlaceArgs a, void* __restrict__ z, int64_t ldz,
                                                         const void* __restrict__ x, int64_t ldx, int cols, int unit) {
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x)
        copy_to_slots<PAST>(z, ldz * unit, static_cast<const char*>(x) + m * ldx * unit, (int64_t)cols * unit, unit,
                            a.place + m * a.top_k, a.top_k, a.M * a.top_k);
}

// Up to kFewPairs pairs in one launch: a workgroup per row looks through all pairs
// for the ranks of its own, and one more counts the experts' starts; up to kFewWork of
// them to look at in a workgroup.  (Rows of 1024 F32 of 60 experts, us, and with a launch
// that places and one that copies: 1 x 6 3.9 and 6.6, 512 x 2 5.2 and 7.5, 128 x 8 7.1
// and 7.9, but 16 x 64 35 and 13.)
constexpr int kFewPairs = 1024, kFewWork = 8 * kFewPairs;
__global__ __launch_bounds__(kCopy) void k_dispatch_few(PlaceArgs a, void* __restrict__ z, int64_t ldz,
                                                        const void* __restrict__ x, int64_t ldx, int cols, int unit) {
    __shared__ int e[kFewPairs];
    __shared__ __align__(16) int hist[kMaxExperts];  // read in fours
    __shared__ int mine[64];  // top_k <= 64
    __shared__ int sums[kCopy / 64];
    const int pairs = (int)(a.M * a.top_k), wave = threadIdx.x >> 6, lane = lane_id();
    for (int q = threadIdx.x; q < kFewPairs; q += kCopy) e[q] = expert_of(a, q, pairs);
    if (blockIdx.x == a.M) {  // the starts: four neighbouring experts a thread
        for (int i = threadIdx.x; i < kMaxExperts; i += kCopy) hist[i] = 0;
        __syncthreads();
        for (int q = threadIdx.x; q < kFewPairs; q += kCopy)
            if (e[q] >= 0) atomicAdd(&hist[e[q]], 1);
        __syncthreads();
        const int4 n = reinterpret_cast<const int4*>(hist)[threadIdx.x];
        const int all = n.x + n.y + n.z + n.w, incl = wave_incl_scan(all);
        if (lane == 63) sums[wave] = incl;
        __syncthreads();
        int at = incl - all;
        for (int w = 0; w < wave; ++w) at += sums[w];
        const int four[4] = {at, at + n.x, at + n.x + n.y, at + n.x + n.y + n.z};
        for (int i = 0; i < 4; ++i)
            if ((int)threadIdx.x * 4 + i < a.E) a.start[threadIdx.x * 4 + i] = four[i];
        if (threadIdx.x == kCopy - 1) a.start[a.E] = at + all;
        return;
    }
    __syncthreads();
    const int m = blockIdx.x;
    for (int j = wave; j < a.top_k; j += kCopy / 64) {
        const int p = m * a.top_k + j, own = e[p];
        int before = 0;
        for (int q = lane; q < (pairs + 63) / 64 * 64; q += 64)
            before += __popcll(__ballot(e[q] >= 0 && (e[q] < own || (e[q] == own && q < p))));
        if (lane == 0) {
            mine[j] = own >= 0 ? before : -1;
            a.place[p] = mine[j];
        }
    }
    __syncthreads();
    copy_to_slots<true>(z, ldz * unit, static_cast<const char*>(x) + m * ldx * unit, (int64_t)cols * unit, unit, mine,
                        a.top_k, pairs);
}

// ---- sums over slots, and their gradients --------------------------------------------
// T lanes share a row (a part of a wave, a wave, or the workgroup), eight neighbours a
// lane and turn.  Up to eight slots' loads are in flight at a time; a wave that has a
// row to itself finds its places by scalar loads.  Bound by memory: sums of 16384 x 8
// rows of 2048 BF16 103 us, 0.6 GB at 5.8 TB/s; their gradients 200 us, 1.1 GB at 5.7.
constexpr int kRow = 256, kSlots = 8;
template <int T>
__device__ __forceinline__ int64_t row_of(int64_t m) {
    if constexpr (T >= 64) return (int64_t)__builtin_amdgcn_readfirstlane((int)m);
    return m;
}
struct Slots {
    int place[kSlots];
    float w[kSlots];
};
// The slots j0 .. j0 + 7 of a row: places of -1 past the last.
__device__ __forceinline__ Slots slots_of(const int32_t* place, const float* wt, int64_t q, int n, int64_t rows) {
    Slots s;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
        const int p = j < n ? place[q + j] : -1;
        s.place[j] = p >= 0 && p < rows ? p : -1;
    }
#pragma unroll
    for (int j = 0; j < kSlots; ++j) s.w[j] = wt && s.place[j] >= 0 ? wt[q + j] : 1.0f;
    return s;
}
// Where fewer than eight columns are left a lane takes the row's last eight, and
// computes and stores what its neighbour does for those they share (gradients of
// 16384 x 4 rows of 1591: 114 us, with the last one by one 182).  Rows of fewer than
// eight go one by one.
__device__ __forceinline__ int from_column(int c, int cols) { return cols - c >= 8 || cols < 8 ? c : cols - 8; }
template <int ELEM>
__device__ __forceinline__ void values8(const Raw8<ELEM>& raw, const void* x, int64_t row, int cols, float (&f)[8]) {
    unpack8<ELEM>(raw, f);
    if (cols < 8) tail8<ELEM>(x, row, 0, cols, f);
}
__device__ __forceinline__ void store8(void* p, int64_t row, int c, int cols, int elem, const float (&f)[8]) {
    if (cols >= 8) {
        put8(p, row + c, elem, f);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < cols) store_elem(p, row + i, f[i], elem);
}

template <int ZE, int T>
__global__ __launch_bounds__(kRow) void k_gather_sum(void* __restrict__ out, int out_elem, int64_t ldo,
                                                     const void* __restrict__ z, int64_t ldz,
                                                     const int32_t* __restrict__ place, const float* __restrict__ wt,
                                                     int64_t M, int top_k, int cols) {
    constexpr int kRows = kRow / T;
    const int lane = threadIdx.x % T;
    const int64_t rows = M * top_k;
    for (int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / T; at < M; at += (int64_t)gridDim.x * kRows) {
        const int64_t m = row_of<T>(at);
        for (unsigned run = (blockIdx.y * T + lane) * 8; run < (unsigned)cols; run += gridDim.y * T * 8) {
            const int c = from_column((int)run, cols);
            float sum[8] = {};
            for (int j0 = 0; j0 < top_k; j0 += kSlots) {
                const Slots s = slots_of(place, wt, m * top_k + j0, top_k - j0, rows);
                Raw8<ZE> raw[kSlots];
#pragma unroll
                for (int j = 0; j < kSlots; ++j) {
                    raw[j] = nothing8<ZE>();
                    if (s.place[j] >= 0 && cols >= 8) raw[j] = raw8<ZE>(z, s.place[j] * ldz + c);
                }
#pragma unroll
                for (int j = 0; j < kSlots; ++j) {
                    if (s.place[j] < 0) continue;
                    float f[8];
                    values8<ZE>(raw[j], z, s.place[j] * ldz, cols, f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] += s.w[j] * f[i];
                }
            }
            store8(out, m * ldo, c, cols, out_elem, sum);
        }
    }
}

// Eight sums over T lanes at once: lanes exchange halves of the values they hold until
// each has one, so ten moves do for eight sums of a wave.  Lane l has that of slot
// slot_of(l) in the end.
__device__ __forceinline__ int slot_of(int lane) {
    return (lane >> 5 & 1) * 4 + (lane >> 4 & 1) * 2 + (lane >> 3 & 1);
}
__device__ __forceinline__ float wave_sum8(float (&v)[kSlots]) {
    const int lane = lane_id();
#pragma unroll
    for (int o = 32, n = 4; o >= 8; o /= 2, n /= 2) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor(give, o, 64);
        }
    }
    float s = v[0];
#pragma unroll
    for (int o = 4; o > 0; o /= 2) s += __shfl_xor(s, o, 64);
    return s;
}

// dout is read once for eight slots, every slot's z once, and dz written once.
template <int ZE, int OE, int T>
__global__ __launch_bounds__(kRow) void k_combine_grad(void* __restrict__ dz, int64_t lddz, float* __restrict__ dw,
                                                       const void* __restrict__ z, int64_t ldz,
                                                       const void* __restrict__ dout, int64_t ldo,
                                                       const int32_t* __restrict__ place, const float* __restrict__ wt,
                                                       int64_t M, int top_k, int cols) {
    constexpr int kRows = kRow / T;
    __shared__ float part[2][kRow / 64][kSlots];
    const int lane = threadIdx.x % T, wave = threadIdx.x >> 6;
    const int64_t rows = M * top_k;
    int turn = 0;
    for (int64_t at = (int64_t)blockIdx.x * kRows + threadIdx.x / T; at < M; at += (int64_t)gridDim.x * kRows) {
        const int64_t m = row_of<T>(at);
        for (int j0 = 0; j0 < top_k; j0 += kSlots) {
            const Slots s = slots_of(place, wt, m * top_k + j0, top_k - j0, rows);
            float dot[kSlots] = {};
            for (unsigned run = lane * 8; run < (unsigned)cols; run += T * 8) {
                const int c = from_column((int)run, cols), shared = (int)run - c;  // with the neighbour
                Raw8<ZE> raw[kSlots];
                float d[8];
                if (dw) {
#pragma unroll
                    for (int j = 0; j < kSlots; ++j) {
                        raw[j] = nothing8<ZE>();
                        if (s.place[j] >= 0 && cols >= 8) raw[j] = raw8<ZE>(z, s.place[j] * ldz + c);
                    }
                }
                values8<OE>(cols >= 8 ? raw8<OE>(dout, m * ldo + c) : nothing8<OE>(), dout, m * ldo, cols, d);
                if (dz) {
#pragma unroll
                    for (int j = 0; j < kSlots; ++j) {
                        if (s.place[j] < 0) continue;
                        float f[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = s.w[j] * d[i];
                        store8(dz, s.place[j] * lddz, c, cols, ZE, f);
                    }
                }
                if (dw) {
#pragma unroll
                    for (int j = 0; j < kSlots; ++j) {
                        if (s.place[j] < 0) continue;
                        float f[8];
                        values8<ZE>(raw[j], z, s.place[j] * ldz, cols, f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float more = __builtin_fmaf(d[i], f[i], dot[j]);
                            dot[j] = i >= shared ? more : dot[j];
                        }
                    }
                }
            }
            if (!dw) continue;
            const int64_t q = m * top_k + j0;
            if constexpr (T < 64) {
#pragma unroll
                for (int j = 0; j < kSlots; ++j) {
#pragma unroll
                    for (int o = T / 2; o > 0; o /= 2) dot[j] += __shfl_xor(dot[j], o, 64);
                    if (lane == 0 && j < top_k - j0) dw[q + j] = dot[j];
                }
            } else {
                const int l = lane_id(), j = slot_of(l);
                float sum = wave_sum8(dot);
                if constexpr (T > 64) {
                    if ((l & 7) == 0) part[turn][wave][j] = sum;
                    __syncthreads();
                    sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < T / 64; ++w) sum += part[turn][w][j];
                    turn ^= 1;
                }
                if ((T == 64 || wave == 0) && (l & 7) == 0 && j < top_k - j0) dw[q + j] = sum;
            }
        }
    }
}

unsigned grid_of(int64_t blocks, unsigned most) { return (unsigned)(blocks < most ? blocks : most); }

}  // namespace

size_t dispatch_place_bytes(int64_t pairs, int n_experts) {
    return pairs <= kEachPairs ? 0 : (size_t)((pairs + kPairs - 1) / kPairs) * n_experts * 4;
}

// By pairs (rows of 16 bytes sorted and moved, us, of 60 experts unless said):
//   to kEachPairs  place at once (8028: 9.7, counting first 11.3; 16056: 10.9 and 11.7, of
//                  4 experts 13.7 and 14.7; 32768: 14.1 and 13.3)
//   beyond         count, place (32768: with a scan 15.4)
//   beyond         kSumBlocks workgroups a scan between, as too many would read the counts
//                  (1048576 of 1024 experts 158, with a scan 180; 2097152 422 and 358; of
//                  60 experts 100 and 103, 197 and 194)
int launch_place(vdttfs_ctx* ctx, const PlaceArgs& a, int* hist) {
    const int64_t pairs = a.M * a.top_k;
    const int blocks = (int)((pairs + kPairs - 1) / kPairs);
    const size_t lds = (size_t)kWaves * a.E * 4;
    int bits = 0;
    while ((1 << bits) < a.E) ++bits;
    if (pairs <= kEachPairs) {
        k_place_each<<<dim3((unsigned)std::max(blocks, 1)), 1024, lds, ctx->stream>>>(a, bits);
        VD_HIP(hipGetLastError());
        return VDTTFS_OK;
    }
    k_place_count<<<dim3((unsigned)blocks), 1024, 0, ctx->stream>>>(a, hist);
    VD_HIP(hipGetLastError());
    if (blocks <= kSumBlocks) {
        k_place_sum<<<dim3((unsigned)blocks), 1024, lds, ctx->stream>>>(a, hist, blocks, bits);
        VD_HIP(hipGetLastError());
        return VDTTFS_OK;
    }
    k_place_scan<<<dim3(1), 1024, 0, ctx->stream>>>(a, hist, blocks, bits);
    VD_HIP(hipGetLastError());
    k_place<<<dim3((unsigned)blocks), 1024, lds, ctx->stream>>>(a, hist, bits);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

bool dispatch_few_ok(int64_t pairs, int top_k) {
    return pairs > 0 && pairs <= kFewPairs && pairs * top_k <= kFewWork;
}
int launch_dispatch_few(vdttfs_ctx* ctx, const PlaceArgs& a, void* z, int64_t ldz, const void* x, int elem, int64_t ldx,
                        int cols) {
    k_dispatch_few<<<dim3((unsigned)(a.M + (a.start ? 1 : 0))), kCopy, 0, ctx->stream>>>(
        a, z, ldz, x, ldx, cols, elem == VDTTFS_ELEM_F32 ? 4 : 2);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_dispatch_rows(vdttfs_ctx* ctx, const PlaceArgs& a, void* z, int64_t ldz, const void* x, int elem, int64_t ldx,
                         int cols) {
    if (a.M <= 0 || cols <= 0) return VDTTFS_OK;
    const int unit = elem == VDTTFS_ELEM_F32 ? 4 : 2;
    const dim3 grid(grid_of(a.M, 1 << 20));
    if (ldz * unit % 16) k_dispatch_rows<false><<<grid, kCopy, 0, ctx->stream>>>(a, z, ldz, x, ldx, cols, unit);
    else k_dispatch_rows<true><<<grid, kCopy, 0, ctx->stream>>>(a, z, ldz, x, ldx, cols, unit);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

namespace {

// Lanes of a row: as many as have a run of eight, up to a wave; past that a wave where
// rows are many and each has no more than `few` values in its slots (its barrier and its
// sum over lanes are then most of its time), else the workgroup.  BF16, us, a wave and a
// workgroup a row:
//   sums       10450 x 1 x 1024 10.5 and 14.6, 16384 x 2 x 1024 17.4 and 21.9, 9039 x 4 x
//              1792 26.7 and 25.6, 500 x 8 x 1024 5.1 and 4.7
//   gradients  10450 x 1 x 1024 18 and 47, 16384 x 1 x 4096 67 and 95, 9039 x 4 x 1792 49
//              and 56, 16384 x 8 x 1024 99 and 113, x 2048 251 and 233, 500 x 8 x 1024 8.3
//              and 7.3
constexpr int kFewOfSum = 4096, kFewOfGrad = 8192;
template <class F>
void by_lanes(int64_t M, int top_k, int cols, int few, const F& f) {
    if (cols <= 64) f(std::integral_constant<int, 8>{});
    else if (cols <= 128) f(std::integral_constant<int, 16>{});
    else if (cols <= 256) f(std::integral_constant<int, 32>{});
    else if (cols <= 512 || (M >= 2048 && (int64_t)cols * std::min(top_k, kSlots) <= few))
        f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, kRow>{});
}
template <class F>
void by_elem(int elem, const F& f) {
    if (elem == VDTTFS_ELEM_F32) f(std::integral_constant<int, VDTTFS_ELEM_F32>{});
    else if (elem == VDTTFS_ELEM_BF16) f(std::integral_constant<int, VDTTFS_ELEM_BF16>{});
    else f(std::integral_constant<int, VDTTFS_ELEM_F16>{});
}
dim3 grid_rows(int64_t M, int lanes) { return dim3(grid_of((M + kRow / lanes - 1) / (kRow / lanes), 1 << 20)); }

}  // namespace

int launch_gather_sum(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const void* z, int z_elem, int64_t ldz,
                      const int32_t* place, const float* wt, int64_t M, int top_k, int cols) {
    by_lanes(M, top_k, cols, kFewOfSum, [&](auto t) {
        dim3 grid = grid_rows(M, t.value);
        // few long rows: their columns over several workgroups (1 x 8 rows of 8192 BF16 4.2
        // us, by one 7.5; 100 x 8 4.1 and 7.8)
        if (t.value == kRow && M < 256)
            grid.y = grid_of(((int64_t)cols + kRow * 8 - 1) / (kRow * 8), 512 / (unsigned)M);
        by_elem(z_elem, [&](auto ze) {
            k_gather_sum<ze.value, t.value>
                <<<grid, kRow, 0, ctx->stream>>>(out, out_elem, ldo, z, ldz, place, wt, M, top_k, cols);
        });
    });
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_combine_grad(vdttfs_ctx* ctx, void* dz, int64_t lddz, float* dw, const void* z, int z_elem, int64_t ldz,
                        const void* dout, int out_elem, int64_t ldo, const int32_t* place, const float* wt, int64_t M,
                        int top_k, int cols) {
    by_lanes(M, top_k, cols, kFewOfGrad, [&](auto t) {
        by_elem(z_elem, [&](auto ze) {
            by_elem(out_elem, [&](auto oe) {
                k_combine_grad<ze.value, oe.value, t.value><<<grid_rows(M, t.value), kRow, 0, ctx->stream>>>(
                    dz, lddz, dw, z, ldz, dout, ldo, place, wt, M, top_k, cols);
            });
        });
    });
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
