// Routing of rows to experts, the sort of the chosen pairs by expert, and the
// weighted sum of the experts' outputs.
#include "elem.h"
#include "head.h"
#include "sort.h"
#include "wave.h"

namespace vdttfs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kSortPairs = 2048;  // pairs a workgroup of the sort takes

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// Another lane's value by a data-parallel-primitive move (no LDS trip); of all
// lanes, or only of the rows in a mask, the others keeping theirs.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp_bits(int v) {
    if constexpr (ROWS == 0xf) return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true);
    else return __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(dpp_bits<CTRL, ROWS>(__float_as_int(v)));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kBcast15 = 0x142, kBcast31 = 0x143;

// The wave's largest value, in every lane (scalar).
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<kXor1>(v));
    v = fmaxf(v, dpp<kXor2>(v));
    v = fmaxf(v, dpp<kHalfMirror>(v));
    v = fmaxf(v, dpp<kMirror>(v));
    v = fmaxf(v, dpp<kBcast15, 0xa>(v));
    v = fmaxf(v, dpp<kBcast31, 0xc>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<kXor1>(v);
    v += dpp<kXor2>(v);
    v += dpp<kHalfMirror>(v);
    v += dpp<kMirror>(v);
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), r * 16));
    return s;
}

// exp and 1 / x of the scores, by the hardware's exp2 and reciprocal; equal inputs
// give equal scores.  Of 32-bit logits the exponent's rounding, which grows with
// |x|, is taken out again: neighbours past 11 would share a score without it.  The
// bounds keep what it multiplies finite, and give 0 and a sigmoid of 0 as the exp
// itself does.  16-bit logits lie 2^13 times as far apart as that rounding: the
// relative error is below (2 + |x|) 2^-23.
template <int ELEM>
__device__ __forceinline__ float fast_exp(float x) {
    constexpr float kHi = 1.44269504088896341f, kLo = 1.925963033500e-8f, kLn2 = 0.693147180559945f;
    if constexpr (ELEM != VDTTFS_ELEM_F32) return __builtin_amdgcn_exp2f(x * kHi);
    const float c = __builtin_amdgcn_fmed3f(x, -120.0f, 88.0f), t = c * kHi;
    const float r = __builtin_fmaf(c, kLo, __builtin_fmaf(c, kHi, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, r * kLn2, e);
}
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// What a group is worth from its two largest values t0 >= t1.  Their sum is
// rounded to 24 bits as any float; past the largest float it is formed of halves,
// so groups are told apart there too, and one of lowest values is above one that
// has none.
__device__ __forceinline__ double group_worth(float t0, float t1, int group_top) {
    if (group_top != 2 || !(t1 > neg_inf())) return t0;
    const float s = t0 + t1;
    return fabsf(s) < -neg_inf() ? (double)s : 2.0 * (double)(0.5f * t0 + 0.5f * t1);
}

struct RouteArgs {
    int32_t* idx;
    float* wt;
    int32_t* count;
    const void* logits;
    int64_t ld;
    const float* bias;
    const uint8_t* row_mask;
    int64_t M;
    int E, k, score, groups, top_groups, group_top, renorm;
    float scale;
};

// The workgroup's counts into the call's, which a launch before has cleared where
// there are several workgroups (2 us more than a call without counts; 65536 rows
// of 256 experts 5): nothing is kept between calls, whose graphs may run side by
// side.  Whole numbers, so no order matters.
__device__ __forceinline__ void finish_counts(const RouteArgs& a, const int* hist) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        if (gridDim.x == 1) a.count[e] = hist[e];
        else if (hist[e]) atomicAdd(&a.count[e], hist[e]);
    }
}

// A wave per row, NPL neighbouring experts a lane: the largest value of the
// wave is then first in index order at the first lane that holds it.
template <int ELEM, int NPL>
__global__ __launch_bounds__(kThreads) void k_route(RouteArgs a) {
    __shared__ int hist[kMaxExperts];
    __shared__ float group_c[kWaves][64 * NPL];
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    if (a.count) {
        for (int e = threadIdx.x; e < a.E; e += kThreads) hist[e] = 0;
        __syncthreads();
    }
    float bias[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int e = lane * NPL + i;
        bias[i] = a.bias && e < a.E ? a.bias[e] : 0.0f;
    }
    const int per = a.E / a.groups;
    for (int64_t m = (int64_t)blockIdx.x * kWaves + wave; m < a.M; m += (int64_t)gridDim.x * kWaves) {
        const bool row = !a.row_mask || a.row_mask[m] != 0;
        float p[NPL], c[NPL];
        float mx = neg_inf();
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int e = lane * NPL + i;
            const float l = row && e < a.E ? load_elem<ELEM>(a.logits, m * a.ld + e) : neg_inf();
            c[i] = l > neg_inf() ? l : neg_inf();  // NaN: not choosable
            mx = fmaxf(mx, c[i]);
        }
        if (a.score == VDTTFS_SCORE_SOFTMAX) {
            mx = wave_max(mx);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                p[i] = c[i] > neg_inf() ? (c[i] == mx ? 1.0f : fast_exp<ELEM>(c[i] - mx)) : 0.0f;
                sum += p[i];
            }
            sum = 1.0f / wave_sum(sum);  // of a row without experts: not read
#pragma unroll
            for (int i = 0; i < NPL; ++i) p[i] *= sum;
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) p[i] = fast_rcp(1.0f + fast_exp<ELEM>(-c[i]));
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float v = p[i] + bias[i];
            c[i] = c[i] > neg_inf() && v > neg_inf() ? v : neg_inf();
        }
        if (a.groups > 1) {
            // the group's value: g of lane 0..groups-1, or of every lane of it
            float t0 = neg_inf(), t1 = neg_inf();
            auto take = [&](float v) {
                t1 = fmaxf(t1, fminf(t0, v));
                t0 = fmaxf(t0, v);
            };
            const bool in_lanes = per % NPL == 0 && (per / NPL == 1 || per / NPL == 2 || per / NPL == 4 ||
                                                     per / NPL == 8 || per / NPL == 16);
            const int span = in_lanes ? per / NPL : 1;  // lanes of a group
            auto merge = [&](float o0, float o1) {
                t1 = fmaxf(fminf(t0, o0), fmaxf(t1, o1));
                t0 = fmaxf(t0, o0);
            };
            if (in_lanes) {
#pragma unroll
                for (int i = 0; i < NPL; ++i) take(c[i]);
                if (span > 1) merge(dpp<kXor1>(t0), dpp<kXor1>(t1));
                if (span > 2) merge(dpp<kXor2>(t0), dpp<kXor2>(t1));
                if (span > 4) merge(dpp<kHalfMirror>(t0), dpp<kHalfMirror>(t1));
                if (span > 8) merge(dpp<kMirror>(t0), dpp<kMirror>(t1));
            } else {
#pragma unroll
                for (int i = 0; i < NPL; ++i) group_c[wave][lane * NPL + i] = c[i];
                wave_sync();
                if (lane < a.groups)
                    for (int i = 0; i < per; ++i) take(group_c[wave][lane * per + i]);
                wave_sync();
            }
            const double g = group_worth(t0, t1, a.group_top);
            // a group stays if fewer than top_groups come before it
            const int mine = in_lanes ? lane / span : lane;
            int rank = 0;
            for (int o = 0; o < a.groups; ++o) {
                const double v = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(g), o * span),
                                                  __builtin_amdgcn_readlane(__double2loint(g), o * span));
                rank += v > g || (v == g && o < mine) ? 1 : 0;
            }
            const bool stays = rank < a.top_groups;
            if (in_lanes) {
#pragma unroll
                for (int i = 0; i < NPL; ++i)
                    if (!stays) c[i] = neg_inf();
            } else {
                const uint64_t keep = __ballot(stays);
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    const int e = lane * NPL + i;
                    if (e < a.E && !((keep >> (e / per)) & 1)) c[i] = neg_inf();
                }
            }
        }
        int my_idx = -1;
        float my_w = 0.0f;
        for (int j = 0; j < a.k; ++j) {
            float bv = c[0];
#pragma unroll
            for (int i = 1; i < NPL; ++i) bv = fmaxf(bv, c[i]);
            const float best = wave_max(bv);
            if (!(best > neg_inf())) break;
            const int src = __builtin_ctzll(__ballot(bv == best));  // the lowest index is in the first such lane
            // that lane's first value equal to it leaves
            int bi = 0;
            float bp = 0.0f;
            bool found = lane != src;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const bool hit = !found && c[i] == best;
                bi = hit ? i : bi;
                bp = hit ? p[i] : bp;
                c[i] = hit ? neg_inf() : c[i];
                found = found || hit;
            }
            const int e = src * NPL + __builtin_amdgcn_readlane(bi, src);
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(bp), src));
            if (lane == j) {
                my_idx = e;
                my_w = w;
            }
        }
        if (a.renorm) {
            const float sum = wave_sum(my_w);
            my_w = sum > 0.0f ? my_w / sum : 0.0f;
        }
        if (lane < a.k) {
            a.idx[m * a.k + lane] = my_idx;
            a.wt[m * a.k + lane] = my_w * a.scale;
            if (a.count && my_idx >= 0) atomicAdd(&hist[my_idx], 1);
        }
    }
    if (a.count) finish_counts(a, hist);
}

// ---- four rows a wave -----------------------------------------------------------
// A key orders the choice: the choice value as a double, whose low 29 bits a
// 32-bit value leaves free, with the expert's index in them so that equal
// values differ, the lower index above.  A maximum is then one instruction with
// no second value to carry.
// kFar, past all floats and the sums of two, stands for an infinity, which has
// no such bits; minus infinity is not choosable.
constexpr double kFar = 0x1p300;
__device__ __forceinline__ double with_index(double d, int e) {
    const int hi = __double2hiint(d), lo = __double2loint(d);
    return __hiloint2double(hi, lo | (((255 - e) ^ hi >> 31) & 255));
}
__device__ __forceinline__ double make_key(float c, int e) {
    return with_index(__builtin_fmin(__builtin_fmax((double)c, -kFar), kFar), e);
}
// The choice value of a key as an integer of the same order, and the expert
// from it and the key's low word.  kFar is infinity again; kNone: the value of a
// key that is below all floats, minus infinity.
__device__ __forceinline__ int key_value(double key) {
    const int f = __float_as_int((float)key);
    return f ^ ((f >> 31) & 0x7fffffff);
}
__device__ __forceinline__ int key_expert(int value, int low) { return 255 - ((low ^ value >> 31) & 255); }
constexpr int kNone = (int)(0xff800000u ^ 0x7fffffffu);
// key[p0 .. p0 + N) in descending order, by Batcher's odd-even merges (K. E.
// Batcher, "Sorting networks and their applications", 1968).
template <int N>
__device__ __forceinline__ void exchange(double (&key)[N], int i, int j) {
    const double x = key[i], y = key[j];
    key[i] = __builtin_fmax(x, y);
    key[j] = __builtin_fmin(x, y);
}
template <int COUNT, int N>
__device__ __forceinline__ void sort_keys(double (&key)[N], int p0) {
#pragma unroll
    for (int p = 1; p < COUNT; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < COUNT; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < COUNT && (i + j) / (2 * p) == (i + j + q) / (2 * p))
                        exchange(key, p0 + i + j, p0 + i + j + q);
}
// The largest over 16 lanes.
__device__ __forceinline__ int row16_max(int v) {
    v = max(v, dpp_bits<kXor1>(v));
    v = max(v, dpp_bits<kXor2>(v));
    v = max(v, dpp_bits<kHalfMirror>(v));
    return max(v, dpp_bits<kMirror>(v));
}
__device__ __forceinline__ float row16_maxf(float v) {
    v = fmaxf(v, dpp<kXor1>(v));
    v = fmaxf(v, dpp<kXor2>(v));
    v = fmaxf(v, dpp<kHalfMirror>(v));
    return fmaxf(v, dpp<kMirror>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp<kXor1>(v);
    v += dpp<kXor2>(v);
    v += dpp<kHalfMirror>(v);
    return v + dpp<kMirror>(v);
}

// Sixteen lanes per row, NPL neighbouring experts a lane: each lane sorts its
// keys once and gives up its first whenever that is the row's largest, so a
// choice costs a maximum over 16 lanes and a shift, for four rows at a time.
// Bound by these instructions: 65536 rows of 256 experts, 8 chosen of 4 groups
// of 8, take 36 us with counts (7 by their bytes; some 800 vector instructions for four
// rows, 200 of them the lanes' sorts), and 80 with a wave per row and a search
// for every choice.  At most kPop choices; a group has `span` lanes, a power of
// two, the last of which may have fewer experts or none.
constexpr int kPop = 8;
template <int ELEM, int NPL>
__global__ __launch_bounds__(1024) void k_route16(RouteArgs a, int span, int vec) {
    __shared__ int hist[256];
    __shared__ int chosen[64][kPop];  // of each row, from the lanes that held them
    __shared__ __align__(16) double group_keys[64][16];
    const int lane = lane_id() & 15;
    const uint64_t before = ((1ull << lane) - 1) << (lane_id() & 48);  // lanes of the row
    const int rows = blockDim.x / 16;
    if (a.count) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
        __syncthreads();
    }
    // the lane's experts: e0 .. e0 + here - 1
    const int per = a.E / a.groups, group = lane / span;
    const int e0 = group * per + lane % span * NPL, left = group < a.groups ? per - lane % span * NPL : 0;
    const int here = left < NPL ? left : NPL;
    float bias[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) bias[i] = a.bias && i < here ? a.bias[e0 + i] : 0.0f;
    const int64_t groups_of_rows = (a.M + rows - 1) / rows;
    for (int64_t b = blockIdx.x; b < groups_of_rows; b += gridDim.x) {
        const int64_t m = b * rows + threadIdx.x / 16;
        const bool row = m < a.M && (!a.row_mask || a.row_mask[m] != 0);
        float l[NPL];
        if (row && vec && here == NPL) {
            if constexpr (ELEM == VDTTFS_ELEM_F32) {
                const float4* p =
                    reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + m * a.ld + e0);
#pragma unroll
                for (int i = 0; i < NPL / 4; ++i) {
                    const float4 v = p[i];
                    l[4 * i] = v.x, l[4 * i + 1] = v.y, l[4 * i + 2] = v.z, l[4 * i + 3] = v.w;
                }
            } else {
                const uint2* p =
                    reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.logits) + m * a.ld + e0);
#pragma unroll
                for (int i = 0; i < NPL / 4; ++i) {
                    const uint2 v = p[i];
                    const uint16_t h[4] = {(uint16_t)v.x, (uint16_t)(v.x >> 16), (uint16_t)v.y, (uint16_t)(v.y >> 16)};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        l[4 * i + q] = ELEM == VDTTFS_ELEM_BF16 ? bf16_to_f32(h[q]) : f16_to_f32(h[q]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i)
                l[i] = row && i < here ? load_elem<ELEM>(a.logits, m * a.ld + e0 + i) : neg_inf();
        }
        float mx = neg_inf(), inv = 1.0f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            l[i] = l[i] > neg_inf() ? l[i] : neg_inf();  // NaN: not choosable
            mx = __builtin_amdgcn_fmed3f(mx, l[i], -neg_inf());
        }
        float c[NPL];
        if (a.score == VDTTFS_SCORE_SOFTMAX) {
            mx = row16_maxf(mx);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                const float x = fast_exp<ELEM>(l[i] - mx);
                c[i] = l[i] == mx ? 1.0f : x;  // an infinity less itself is none
                sum += c[i];
            }
            inv = 1.0f / row16_sum(sum);  // a row without experts has some too, not used
#pragma unroll
            for (int i = 0; i < NPL; ++i) c[i] *= inv;
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) c[i] = fast_rcp(1.0f + fast_exp<ELEM>(-l[i]));
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const float v = c[i] + bias[i];
            c[i] = fmaxf(l[i] > neg_inf() ? v : neg_inf(), neg_inf());
        }
        if (a.groups > 1) {
            float t0 = neg_inf(), t1 = neg_inf();
#pragma unroll
            for (int i = 0; i < NPL; ++i) {
                t1 = __builtin_amdgcn_fmed3f(t0, t1, c[i]);  // t1 <= t0
                t0 = fmaxf(t0, c[i]);
            }
            auto merge = [&](float o0, float o1) {
                t1 = fmaxf(fminf(t0, o0), fmaxf(t1, o1));
                t0 = fmaxf(t0, o0);
            };
            if (span > 1) merge(dpp<kXor1>(t0), dpp<kXor1>(t1));
            if (span > 2) merge(dpp<kXor2>(t0), dpp<kXor2>(t1));
            if (span > 4) merge(dpp<kHalfMirror>(t0), dpp<kHalfMirror>(t1));
            if (span > 8) merge(dpp<kMirror>(t0), dpp<kMirror>(t1));
            const double g = group_worth(t0, t1, a.group_top);
            // a group stays if fewer than top_groups come before it: keys again,
            // the row's through LDS
            const double k = with_index(__builtin_fmin(__builtin_fmax(g, -kFar), kFar), group);
            double* keys = group_keys[threadIdx.x / 16];
            if (lane % span == 0 && group < a.groups) keys[group] = k;
            if (lane >= a.groups) keys[lane] = -2 * kFar;
            wave_sync();
            int rank = 0;
#pragma unroll
            for (int o = 0; o < 8; ++o) rank += keys[o] > k ? 1 : 0;
            if (a.groups > 8) {
#pragma unroll
                for (int o = 8; o < 16; ++o) rank += keys[o] > k ? 1 : 0;
            }
            wave_sync();
            if (rank >= a.top_groups) {
#pragma unroll
                for (int i = 0; i < NPL; ++i) c[i] = neg_inf();
            }
        }
        double key[NPL];
#pragma unroll
        for (int i = 0; i < NPL; ++i) key[i] = make_key(c[i], e0 + i);
        if constexpr (NPL == 2 * kPop) {
            // Of two sorted halves the larger of each first and the other's last:
            // the first kPop of all, rising and then falling, so that exchanges
            // over 4, 2 and 1 sort them.
            sort_keys<kPop>(key, 0);
            sort_keys<kPop>(key, kPop);
#pragma unroll
            for (int i = 0; i < kPop; ++i) key[i] = __builtin_fmax(key[i], key[2 * kPop - 1 - i]);
#pragma unroll
            for (int q = kPop / 2; q >= 1; q /= 2)
#pragma unroll
                for (int i = 0; i < kPop; ++i)
                    if ((i & q) == 0) exchange(key, i, i + q);
        } else {
            static_assert(NPL <= kPop, "a lane's keys");
            sort_keys<NPL>(key, 0);
        }
        // Heads are compared by value; of lanes with the same the first, which has
        // the lower experts, wins.
        constexpr int kHeld = NPL < kPop ? NPL : kPop;
        int value[kHeld], low[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            value[i] = key_value(key[i]);
            low[i] = __double2loint(key[i]);
        }
        int mine = kNone;
#pragma unroll
        for (int j = 0; j < kPop; ++j) {
            if (j < a.k) {
                const int best = row16_max(value[0]);
                const uint64_t heads = __ballot(value[0] == best);
                const bool win = value[0] == best && (heads & before) == 0;
                if (win) chosen[threadIdx.x / 16][j] = low[0];
#pragma unroll
                for (int i = 0; i + 1 < kHeld && i + 1 < kPop - j; ++i) {
                    const int v = value[i + 1], w = low[i + 1];
                    value[i] = win ? v : value[i];
                    low[i] = win ? w : low[i];
                }
                if (kHeld < kPop - j) value[kHeld - 1] = win ? kNone : value[kHeld - 1];
                mine = lane == j ? best : mine;
            }
        }
        wave_sync();
        int e = -1;
        float w = 0.0f;
        if (mine > kNone) {
            e = key_expert(mine, chosen[threadIdx.x / 16][lane]);
            const float v = load_elem<ELEM>(a.logits, m * a.ld + e);
            w = a.score != VDTTFS_SCORE_SOFTMAX ? fast_rcp(1.0f + fast_exp<ELEM>(-v))
                                                : (v == mx ? 1.0f : fast_exp<ELEM>(v - mx)) * inv;
        }
        if (a.renorm) {
            const float sum = row16_sum(w);
            w = sum > 0.0f ? w / sum : 0.0f;
        }
        if (m < a.M && lane < a.k) {
            a.idx[m * a.k + lane] = e;
            a.wt[m * a.k + lane] = w * a.scale;
            if (a.count && e >= 0) atomicAdd(&hist[e], 1);
        }
        wave_sync();
    }
    if (a.count) finish_counts(a, hist);
}

__global__ void k_zero(int* p, int n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) p[i] = 0;
}
void clear_counts(vdttfs_ctx* ctx, int* count, int E) {
    if (count) k_zero<<<dim3(1), kThreads, 0, ctx->stream>>>(count, E);
}

// Four rows a wave where it can: up to 256 experts, 8 slots, and groups that
// fit its lanes; else a wave per row (29887 rows of 12 experts in groups of 6: 27
// us, four rows a wave 13).
template <int ELEM>
void route_elem(vdttfs_ctx* ctx, const RouteArgs& a) {
    const int size = ELEM == VDTTFS_ELEM_F32 ? 4 : 2, per = a.E / a.groups;
    // the fewest experts a lane with which the groups' lanes fit
    int npl = 4, span = 16;
    for (; npl <= 16; npl *= 2) {
        for (span = 1; span * npl < per; span *= 2) {
        }
        if (span * a.groups <= 16) break;
    }
    if (a.E <= 256 && a.k <= kPop && npl <= 16) {
        // one workgroup a CU at most, of 16 waves where there are rows for them
        const int threads = a.M > 1024 ? 1024 : kThreads;
        const int64_t blocks = (a.M + threads / 16 - 1) / (threads / 16);
        const dim3 grid((unsigned)(blocks < 256 ? blocks : 256));
        if (blocks > 1) clear_counts(ctx, a.count, a.E);
        const int vec = per % 4 == 0 && (((uintptr_t)a.logits | (uintptr_t)(a.ld * size)) & (4 * size - 1)) == 0;
        if (npl == 4) k_route16<ELEM, 4><<<grid, threads, 0, ctx->stream>>>(a, span, vec);
        else if (npl == 8) k_route16<ELEM, 8><<<grid, threads, 0, ctx->stream>>>(a, span, vec);
        else k_route16<ELEM, 16><<<grid, threads, 0, ctx->stream>>>(a, span, vec);
        return;
    }
    const int64_t blocks = (a.M + kWaves - 1) / kWaves;
    const dim3 grid((unsigned)(blocks < 1024 ? blocks : 1024));
    if (blocks > 1) clear_counts(ctx, a.count, a.E);
    if (a.E <= 64) k_route<ELEM, 1><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 128) k_route<ELEM, 2><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 256) k_route<ELEM, 4><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (a.E <= 512) k_route<ELEM, 8><<<grid, kThreads, 0, ctx->stream>>>(a);
    else k_route<ELEM, 16><<<grid, kThreads, 0, ctx->stream>>>(a);
}

// Experts of each workgroup's pairs: hist[block][expert].
__global__ __launch_bounds__(1024) void k_sort_count(const int32_t* __restrict__ idx, int64_t pairs, int E,
                                                     int* __restrict__ hist) {
    __shared__ int h[kMaxExperts];
    const int64_t q0 = (int64_t)blockIdx.x * kSortPairs + threadIdx.x, q1 = q0 + 1024;
    const int e0 = q0 < pairs ? idx[q0] : -1, e1 = q1 < pairs ? idx[q1] : -1;
    if ((int)threadIdx.x < E) h[threadIdx.x] = 0;
    __syncthreads();
    if (e0 >= 0 && e0 < E) atomicAdd(&h[e0], 1);
    if (e1 >= 0 && e1 < E) atomicAdd(&h[e1], 1);
    __syncthreads();
    if ((int)threadIdx.x < E) hist[(int64_t)blockIdx.x * E + threadIdx.x] = h[threadIdx.x];
}

// One workgroup: hist[block][expert] becomes the sorted position of the
// block's first pair of the expert; the row tiles of every expert follow.
// 2^log threads go over the experts, and share the blocks in 1024 >> log runs.
__global__ __launch_bounds__(1024) void k_sort_plan(int* __restrict__ hist, int blocks, int E, int log, int bm,
                                                    int4* __restrict__ tiles, int* __restrict__ n_tiles) {
    __shared__ int lds[16];
    __shared__ int sums[1024];
    __shared__ int starts[kMaxExperts];
    const int e = threadIdx.x & ((1 << log) - 1), run = threadIdx.x >> log, runs = 1024 >> log;
    const int per = (blocks + runs - 1) / runs;
    const int b0 = run * per, b1 = b0 + per < blocks ? b0 + per : blocks;
    int n = 0;
    if (e < E)
#pragma unroll 4
        for (int b = b0; b < b1; ++b) n += hist[(int64_t)b * E + e];
    sums[threadIdx.x] = n;
    __syncthreads();
    // the first run's threads have an expert's total
    int total = 0;
    if (run == 0)
        for (int r = 0; r < runs; ++r) total += sums[(r << log) + e];
    int all, t_all;
    const int start = block_excl_scan(total, lds, &all);
    const int t = (total + bm - 1) / bm;
    const int t0 = block_excl_scan(t, lds, &t_all);
    for (int i = 0; i < t; ++i) tiles[t0 + i] = make_int4(e, start + i * bm, start + total, 0);
    if (threadIdx.x == 0) *n_tiles = t_all;
    if (run == 0) starts[e] = start;
    __syncthreads();
    if (e >= E) return;
    int at = starts[e];
    for (int r = 0; r < run; ++r) at += sums[(r << log) + e];
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int h = hist[(int64_t)b * E + e];
        hist[(int64_t)b * E + e] = at;
        at += h;
    }
}

// Each pair to its place.  The order of an expert's pairs within a workgroup
// is that of its LDS atomics; nothing that is computed depends on it.
__global__ __launch_bounds__(1024) void k_sort_place(const int32_t* __restrict__ idx, int64_t pairs, int E, int top_k,
                                                     const int* __restrict__ hist, int* __restrict__ pair,
                                                     int* __restrict__ row) {
    __shared__ int at[kMaxExperts];
    const int64_t q[2] = {(int64_t)blockIdx.x * kSortPairs + threadIdx.x,
                          (int64_t)blockIdx.x * kSortPairs + threadIdx.x + 1024};
    const int e[2] = {q[0] < pairs ? idx[q[0]] : -1, q[1] < pairs ? idx[q[1]] : -1};
    if ((int)threadIdx.x < E) at[threadIdx.x] = hist[(int64_t)blockIdx.x * E + threadIdx.x];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (e[i] >= 0 && e[i] < E) {
            const int to = atomicAdd(&at[e[i]], 1);
            pair[to] = (int)q[i];
            row[to] = (int)(q[i] / top_k);
        }
}

__global__ __launch_bounds__(1024) void k_sort_one(SortOne a) { sort_one(a); }

// The slots' outputs summed in order, four neighbouring columns a thread; eight
// slots' loads are in flight at a time.
__global__ __launch_bounds__(kThreads) void k_combine(void* __restrict__ out, int out_elem, int64_t ldo,
                                                      const float* __restrict__ z, int64_t ldz,
                                                      const int32_t* __restrict__ idx, const float* __restrict__ wt,
                                                      int64_t M, int N, int top_k, int E) {
    constexpr int VEC = 4, kSlots = 8;
    typedef float zvec __attribute__((ext_vector_type(VEC)));
    const int n = (blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (n >= N) return;
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
        float sum[VEC] = {};
        for (int j0 = 0; j0 < top_k; j0 += kSlots) {
            zvec v[kSlots];
            float w[kSlots];
            bool on[kSlots];
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
                const int64_t q = m * top_k + j0 + j;
                const int e = j0 + j < top_k ? idx[q] : -1;
                on[j] = e >= 0 && e < E;
                w[j] = 0.0f;
                v[j] = zvec(0.0f);
                if (on[j]) {
                    w[j] = wt[q];
                    v[j] = *reinterpret_cast<const zvec*>(z + q * ldz + n);
                }
            }
#pragma unroll
            for (int j = 0; j < kSlots; ++j)
                if (on[j])
#pragma unroll
                    for (int i = 0; i < VEC; ++i) sum[i] += w[j] * v[j][i];
        }
        const int64_t o = m * ldo + n;
        const bool bf16 = out_elem == VDTTFS_ELEM_BF16;
        if (out_elem != VDTTFS_ELEM_F32 && n + VEC <= N &&
            (((uintptr_t)out | (uintptr_t)(ldo * 2)) & (VEC * 2 - 1)) == 0) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) =
                make_uint2(pack2(sum[0], sum[1], bf16), pack2(sum[2], sum[3], bf16));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (n + i < N) store_elem(out, o + i, sum[i], out_elem);
        }
    }
}

}  // namespace

int launch_route(vdttfs_ctx* ctx, int32_t* idx, float* wt, int32_t* count, const void* logits, int elem, int64_t ld,
                 const float* bias, const uint8_t* row_mask, int64_t M, const vdttfs_route_opts& o) {
    if (M <= 0) {
        clear_counts(ctx, count, o.n_experts);
        VD_HIP(hipGetLastError());
        return VDTTFS_OK;
    }
    const RouteArgs a{idx,         wt,      count,   logits,   ld,           bias,        row_mask, M,
                      o.n_experts, o.top_k, o.score, o.groups, o.top_groups, o.group_top, o.renorm, o.scale};
    if (elem == VDTTFS_ELEM_F32) route_elem<VDTTFS_ELEM_F32>(ctx, a);
    else if (elem == VDTTFS_ELEM_BF16) route_elem<VDTTFS_ELEM_BF16>(ctx, a);
    else route_elem<VDTTFS_ELEM_F16>(ctx, a);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int dispatch_blocks(int64_t pairs) { return (int)((pairs + kSortPairs - 1) / kSortPairs); }

int launch_dispatch(vdttfs_ctx* ctx, const int32_t* idx, int64_t pairs, int top_k, int n_experts, int bm,
                    const Dispatch& d) {
    const int blocks = dispatch_blocks(pairs);
    if (pairs <= kSortOne) {
        k_sort_one<<<dim3(1), 1024, 0, ctx->stream>>>(
            SortOne{idx, (int)pairs, n_experts, top_k, bm, d.tiles, d.n_tiles, d.pair, d.row});
        VD_HIP(hipGetLastError());
        return VDTTFS_OK;
    }
    int log = 0;
    while ((1 << log) < n_experts) ++log;
    k_sort_count<<<dim3((unsigned)blocks), 1024, 0, ctx->stream>>>(idx, pairs, n_experts, d.hist);
    VD_HIP(hipGetLastError());
    k_sort_plan<<<dim3(1), 1024, 0, ctx->stream>>>(d.hist, blocks, n_experts, log, bm, d.tiles, d.n_tiles);
    VD_HIP(hipGetLastError());
    k_sort_place<<<dim3((unsigned)blocks), 1024, 0, ctx->stream>>>(idx, pairs, n_experts, top_k, d.hist, d.pair,
                                                                   d.row);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

int launch_combine(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const float* z, int64_t ldz,
                   const int32_t* idx, const float* wt, int64_t M, int N, int top_k, int n_experts) {
    const dim3 grid((unsigned)(((N + 3) / 4 + kThreads - 1) / kThreads), (unsigned)(M < 65535 ? M : 65535));
    k_combine<<<grid, kThreads, 0, ctx->stream>>>(out, out_elem, ldo, z, ldz, idx, wt, M, N, top_k, n_experts);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
