// Rows over their root mean square, with a residual's addition before it, as
// floats, 8-bit codes or microscaled 4-bit codes.
//
// h = x + r, u = h g, y = u / sqrt(mean(h^2) + eps).  Bound by memory: a row is
// held in registers between the two, so x and r are read once and the sum and y
// written once (16384 x 4096 BF16 with a residual 96 us, 0.54 GB at 5.6 TB/s).  Codes
// of 8 bits cost as many instructions again: 8192 x 2048 24 to 25 us, 4.8 TB/s.
#include "elem.h"
#include "head.h"
#include "mx4.h"
#include "quant.h"

namespace vdttfs {
namespace {

constexpr int kNoRes = -1;

struct __attribute__((packed, aligned(1))) AnyUint2 {
    uint32_t v[2];
};
__device__ __forceinline__ void store8(void* p, int64_t row, int c, int cols, int elem, const float (&f)[8]) {
    if (cols - c >= 8) {
        put8(p, row + c, elem, f);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < cols - c) store_elem(p, row + c + i, f[i], elem);
}
__device__ __forceinline__ void store_codes8(int8_t* q, int64_t row, int c, int cols, const int (&k)[8]) {
    if (cols - c >= 8) {
        const uint2 w = pack8(k);
        AnyUint2* to = reinterpret_cast<AnyUint2*>(q + row + c);
        to->v[0] = w.x;
        to->v[1] = w.y;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < cols - c) q[row + c + i] = (int8_t)k[i];
}

// Sums and largest magnitudes (as bits: those of a NaN are above all others, so it
// wins) over the LANES lanes that share a row, in every one of them.  `turn` alternates
// between calls, so that one barrier a call does.
template <int LANES>
struct Shared {
    float sum[2][LANES > 64 ? LANES / 64 : 1];
    uint32_t top[2][LANES > 64 ? LANES / 64 : 1];
};
template <int LANES, bool TOP>
__device__ __forceinline__ void over_row(float& sum, uint32_t& top, Shared<LANES>& s, int turn) {
#pragma unroll
    for (int o = 1; o < LANES && o < 64; o *= 2) {
        sum += __shfl_xor(sum, o, 64);
        if (TOP) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    }
    if constexpr (LANES > 64) {
        const int wave = threadIdx.x >> 6;
        if (lane_id() == 0) {
            s.sum[turn][wave] = sum;
            if (TOP) s.top[turn][wave] = top;
        }
        __syncthreads();
        sum = s.sum[turn][0];
        if (TOP) top = s.top[turn][0];
#pragma unroll
        for (int i = 1; i < LANES / 64; ++i) {
            sum += s.sum[turn][i];
            if (TOP) top = max(top, s.top[turn][i]);
        }
    }
}

// 1 / sqrt(mean + eps) of a row as f * r, f a power of two.  Squares of values
// past 2^63 or below 2^-60 or so leave the range of 32 bits: such a row is summed
// again with its largest value brought near 1 (the sum of (h f)^2), and its root
// taken in 64 bits.  Where h g passes the largest float, though y does not, the gain
// is taken of h f; else u stays the 32-bit product that its 8-bit codes are defined
// by.  Zeros alone with an eps of 0 give 0.
constexpr float kFewest = 0x1p-100f, kMost = 0x1p120f;
struct Root {
    float f, r;
};
// mean + eps too: with an eps at the largest float a mean of 2^103 passes it
__device__ __forceinline__ bool in_range(float sum, float eps) {
    return sum >= kFewest && sum <= kMost && eps < 0x1p127f;
}
__device__ __forceinline__ Root plain_root(float sum, int cols, float eps) {
    return Root{1.0f, 1.0f / sqrtf(sum / (float)cols + eps)};
}
__device__ __forceinline__ float factor_of(uint32_t top) {
    int e = (int)(top >> 23) - 127;
    e = e < -126 ? -126 : e > 126 ? 126 : e;
    return __uint_as_float((uint32_t)(127 - e) << 23);
}
__device__ __forceinline__ Root far_root(float sum, float top, float f, int cols, float eps) {
    if (!(top > 0.0f)) return Root{1.0f, top == 0.0f ? (eps > 0.0f ? 1.0f / sqrtf(eps) : 0.0f) : __builtin_nanf("")};
    if (top == __builtin_inff()) return Root{1.0f, 0.0f};
    // mean(h^2) + eps = (mean((h f)^2) + eps f^2) / f^2
    const double v = (double)sum / cols + (double)eps * f * f;
    return Root{f, (float)(1.0 / sqrt(v))};
}

// The factor taken before the gain: of a row of finite values, the largest `most`, of
// whose u some, `lost` of them, are not.
__device__ __forceinline__ float before_gain(float lost, uint32_t most, float f) {
    return lost > 0.0f && most < 0x7f800000u ? f : 1.0f;
}

// Eight values, `by` of them further on, then zeros.
__device__ __forceinline__ void further(float (&f)[8], int by) {
#pragma unroll
    for (int o = 4; o > 0; o /= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = by & o ? (i + o < 8 ? f[i + o] : 0.0f) : f[i];
}

enum { kFloats, kCodes8, kCodes4 };

// LANES lanes hold a row, eight values a lane and turn (NV turns).  Gains stay in
// registers over the workgroup's rows.  Where fewer than eight are left, a lane loads
// the row's last eight with the others' loads and moves them (7552 x 1165 to 8 bits
// with a residual 17 us; loaded one by one behind the others 10 more).  The sum, which
// may take the residual's place, is stored behind the barrier that all loads come before.
template <int XE, int RE, int NV, int LANES, int THREADS>
__global__ __launch_bounds__(THREADS, NV == 2 ? 4 : 1) void k_norm(NormArgs a) {
    static_assert(LANES <= 64 || LANES == THREADS, "a row has a part of a wave, a wave or the workgroup");
    __shared__ Shared<LANES> lds;
    constexpr int kRows = THREADS / LANES;
    const int lane = threadIdx.x % LANES;
    float g[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * LANES + lane) * 8;
        if (a.gain) load8<VDTTFS_ELEM_F32>(a.gain, 0, c, a.cols, g[v]);
    }
    int turn = 0;
    for (int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES; m < a.rows; m += (int64_t)gridDim.x * kRows) {
        Raw8<XE> rx[NV];
        Raw8<RE == kNoRes ? VDTTFS_ELEM_F32 : RE> rr[RE == kNoRes ? 1 : NV];
        float h[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * LANES + lane) * 8;
            const int from = c + 8 <= a.cols ? c : a.cols - 8;
            rx[v] = nothing8<XE>();
            if (c < a.cols && from >= 0) rx[v] = raw8<XE>(a.x, m * a.ldx + from);
            if constexpr (RE != kNoRes) {
                rr[v] = nothing8<RE>();
                if (c < a.cols && from >= 0) rr[v] = raw8<RE>(a.res, m * a.ldr + from);
            }
        }
        float sum = 0.0f;
        uint32_t top = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * LANES + lane) * 8;
            const bool part = c < a.cols && c + 8 > a.cols;
            unpack8<XE>(rx[v], h[v]);
            if (part && a.cols < 8) tail8<XE>(a.x, m * a.ldx, c, a.cols, h[v]);
            if constexpr (RE != kNoRes) {
                float r[8];
                unpack8<RE>(rr[v], r);
                if (part && a.cols < 8) tail8<RE>(a.res, m * a.ldr, c, a.cols, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[v][i] += r[i];
            }
            if (part && a.cols >= 8) further(h[v], c + 8 - a.cols);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(h[v][i], h[v][i], sum);
        }
        float u[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) u[v][i] = a.gain ? h[v][i] * g[v][i] : h[v][i];
        if (a.kind == kCodes8) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, magnitude(u[v][i]));
            over_row<LANES, true>(sum, top, lds, turn);
        } else {
            over_row<LANES, false>(sum, top, lds, turn);
        }
        turn ^= 1;
        if constexpr (RE != kNoRes) {
            if (a.sum) {
#pragma unroll
                for (int v = 0; v < NV; ++v) store8(a.sum, m * a.lds, (v * LANES + lane) * 8, a.cols, RE, h[v]);
            }
        }
        Root root = plain_root(sum, a.cols, a.eps);
        if (!in_range(sum, a.eps)) {  // the same in all lanes of the row
            float lost = 0.0f, again = 0.0f;
            uint32_t most = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    most = max(most, magnitude(h[v][i]));
                    // of half of h, whose products with the gain need not be kept
                    if (fabsf(a.gain ? (h[v][i] * 0.5f) * g[v][i] : h[v][i] * 0.5f) >= 0x1p127f) lost = 1.0f;
                }
            over_row<LANES, true>(lost, most, lds, turn);
            turn ^= 1;
            const float f = factor_of(most), before = before_gain(lost, most, f);
            top = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    again += (h[v][i] * f) * (h[v][i] * f);
                    u[v][i] = a.gain ? (h[v][i] * before) * g[v][i] : h[v][i] * before;
                    top = max(top, magnitude(u[v][i]));
                }
            over_row<LANES, true>(again, top, lds, turn);
            turn ^= 1;
            root = far_root(again, __uint_as_float(most), f, a.cols, a.eps);
            if (before != 1.0f) root.f = 1.0f;
        }
        if (a.kind == kCodes8) {
            // codes are those of u: a row's codes do not change with a factor of all of it
            const float s = scale_of(__uint_as_float(top));
            if (lane == 0) a.scale[m] = (float)((double)s * root.f * root.r);
            const Coder coder = coder_of(s);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                int k[8];
                codes8(u[v], coder, k);
                store_codes8(static_cast<int8_t*>(a.q), m * a.ldq, (v * LANES + lane) * 8, a.cols, k);
            }
            continue;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * LANES + lane) * 8;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = u[v][i] * root.f * root.r;
            if (a.kind == kFloats) {
                store8(a.y, m * a.ldy, c, a.cols, a.y_elem, y);
            } else {
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) most = max(most, magnitude(y[i]));
                const int s = mx4_scale(quad_max(most));
                mx4_store8(static_cast<uint8_t*>(a.q) + m * a.ldq, a.ms + m * a.ldms, c, a.cols, mx4_codes8(y, s), s);
            }
        }
    }
}

// Rows past what a workgroup holds: a workgroup each, which reads its row twice
// (the second time from the caches), and four times where its squares leave the range.
// F32 with a residual, its sum and floats out: 1 and 64 rows of 20000 8.8 and 9.9 us, of
// 65536 22 and 32, where the bytes of 64 take 12.  The sum is written in the second reading, as
// it may take the residual's place; a thread has the same columns in both.
template <int XE, int RE>
__device__ __forceinline__ void load_h(const NormArgs& a, int64_t m, int c, float (&h)[8]) {
    load8<XE>(a.x, m * a.ldx, c, a.cols, h);
    if constexpr (RE != kNoRes) {
        float r[8];
        load8<RE>(a.res, m * a.ldr, c, a.cols, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
}
__device__ __forceinline__ void times_gain(const NormArgs& a, int c, float f, float (&h)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= f;
    if (!a.gain) return;
    float g[8];
    load8<VDTTFS_ELEM_F32>(a.gain, 0, c, a.cols, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] *= g[i];
}
constexpr int kLong = 1024;
template <int XE, int RE>
__global__ __launch_bounds__(kLong) void k_norm_long(NormArgs a) {
    __shared__ Shared<kLong> lds;
    int turn = 0;
    // unsigned: a thread's column goes past the row's end, and past 2^31
    const unsigned cols = (unsigned)a.cols, ends = (cols + kMxBlock - 1) / kMxBlock * kMxBlock;
    for (int64_t m = blockIdx.x; m < a.rows; m += gridDim.x) {
        uint32_t top = 0;
        double total = 0.0;  // a thread has up to 2^18 runs
        for (unsigned c = threadIdx.x * 8; c < cols; c += kLong * 8) {
            float h[8], part = 0.0f;
            load_h<XE, RE>(a, m, (int)c, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) part = __builtin_fmaf(h[i], h[i], part);
            total += part;
            times_gain(a, (int)c, 1.0f, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, magnitude(h[i]));
        }
        float sum = (float)total;
        over_row<kLong, true>(sum, top, lds, turn);
        turn ^= 1;
        Root root = plain_root(sum, a.cols, a.eps);
        float before = 1.0f;  // the factor taken before the gain
        if (!in_range(sum, a.eps)) {
            float lost = 0.0f, again = 0.0f;
            uint32_t most = 0;
            for (unsigned c = threadIdx.x * 8; c < cols; c += kLong * 8) {
                float h[8];
                load_h<XE, RE>(a, m, (int)c, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = max(most, magnitude(h[i]));
            }
            if (top >= 0x7f800000u) lost = 1.0f;
            over_row<kLong, true>(lost, most, lds, turn);
            turn ^= 1;
            const float f = factor_of(most);
            before = before_gain(lost, most, f);
            double total_f = 0.0;
            top = 0;
            for (unsigned c = threadIdx.x * 8; c < cols; c += kLong * 8) {
                float h[8];
                load_h<XE, RE>(a, m, (int)c, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) total_f += (double)((h[i] * f) * (h[i] * f));
                times_gain(a, (int)c, before, h);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, magnitude(h[i]));
            }
            again = (float)total_f;
            over_row<kLong, true>(again, top, lds, turn);
            turn ^= 1;
            root = far_root(again, __uint_as_float(most), f, a.cols, a.eps);
            if (before != 1.0f) root.f = 1.0f;
        }
        const float s8 = scale_of(__uint_as_float(top));
        const Coder coder = coder_of(s8);
        if (a.kind == kCodes8 && threadIdx.x == 0) a.scale[m] = (float)((double)s8 * root.f * root.r);
        for (unsigned c = threadIdx.x * 8; c < ends; c += kLong * 8) {
            float h[8];
            load_h<XE, RE>(a, m, (int)c, h);
            if constexpr (RE != kNoRes) {
                if (a.sum && c < cols) store8(a.sum, m * a.lds, (int)c, a.cols, RE, h);
            }
            times_gain(a, (int)c, before, h);
            if (a.kind == kCodes8) {
                int k[8];
                codes8(h, coder, k);
                if (c < cols) store_codes8(static_cast<int8_t*>(a.q), m * a.ldq, (int)c, a.cols, k);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = h[i] * root.f * root.r;
            if (a.kind == kFloats) {
                if (c < cols) store8(a.y, m * a.ldy, (int)c, a.cols, a.y_elem, h);
            } else {
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) most = max(most, magnitude(h[i]));
                const int s = mx4_scale(quad_max(most));
                mx4_store8(static_cast<uint8_t*>(a.q) + m * a.ldq, a.ms + m * a.ldms, (int)c, a.cols, mx4_codes8(h, s),
                           s);
            }
        }
    }
}

template <int XE, int RE, int NV, int LANES, int THREADS>
void norm_nv(vdttfs_ctx* ctx, const NormArgs& a) {
    constexpr int kRows = THREADS / LANES;
    const int64_t blocks = (a.rows + kRows - 1) / kRows;
    const unsigned most = 256 * 2048 / THREADS;  // as many as the CUs hold at once
    k_norm<XE, RE, NV, LANES, THREADS>
        <<<dim3((unsigned)(blocks < most ? blocks : most)), THREADS, 0, ctx->stream>>>(a);
}

// By columns: as many lanes as a row has runs of eight, to a wave; with rows enough to
// fill the CUs a wave takes two, so that no barrier is needed; then three waves or four,
// one run a lane, then four or eight of two.  Four runs in 256 lanes instead of two in 512: 3973 x 5632 to 8
// bits 47.2 us and 40.6, 2000 x 4100 24.3 and 18.2, 4096 x 8192 to 4 bits 48.0 and 41.7;
// the other way round 4000 x 6144 of 32-bit floats throughout, 76.7 and 82.4.  One run in
// 1024 lanes 52.1, 23.1, 49.9 and 75.1.
template <int XE, int RE>
void norm_types(vdttfs_ctx* ctx, const NormArgs& a) {
    if (a.cols <= 128) norm_nv<XE, RE, 1, 16, 256>(ctx, a);
    else if (a.cols <= 256) norm_nv<XE, RE, 1, 32, 256>(ctx, a);
    else if (a.cols <= 512) norm_nv<XE, RE, 1, 64, 256>(ctx, a);
    else if (a.cols <= 1024 && a.rows >= 1024) norm_nv<XE, RE, 2, 64, 256>(ctx, a);
    else if (a.cols <= 1536) norm_nv<XE, RE, 1, 192, 192>(ctx, a);
    else if (a.cols <= 2048) norm_nv<XE, RE, 1, 256, 256>(ctx, a);
    else if (a.cols <= 4096) norm_nv<XE, RE, 2, 256, 256>(ctx, a);
    else if (a.cols <= 8192) norm_nv<XE, RE, 2, 512, 512>(ctx, a);
    else if (a.cols <= 16384) norm_nv<XE, RE, 2, 1024, 1024>(ctx, a);
    else
        k_norm_long<XE, RE><<<dim3((unsigned)(a.rows < 512 ? a.rows : 512)), kLong, 0, ctx->stream>>>(a);
}

template <int XE>
void norm_x(vdttfs_ctx* ctx, const NormArgs& a, int res_elem) {
    if (!a.res) norm_types<XE, kNoRes>(ctx, a);
    else if (res_elem == VDTTFS_ELEM_F32) norm_types<XE, VDTTFS_ELEM_F32>(ctx, a);
    else if (res_elem == VDTTFS_ELEM_BF16) norm_types<XE, VDTTFS_ELEM_BF16>(ctx, a);
    else norm_types<XE, VDTTFS_ELEM_F16>(ctx, a);
}

}  // namespace

int launch_norm(vdttfs_ctx* ctx, NormArgs a, int x_elem, int res_elem) {
    a.kind = a.y ? kFloats : a.ms ? kCodes4 : kCodes8;
    if (a.rows <= 0) return VDTTFS_OK;
    if (x_elem == VDTTFS_ELEM_F32) norm_x<VDTTFS_ELEM_F32>(ctx, a, res_elem);
    else if (x_elem == VDTTFS_ELEM_BF16) norm_x<VDTTFS_ELEM_BF16>(ctx, a, res_elem);
    else norm_x<VDTTFS_ELEM_F16>(ctx, a, res_elem);
    VD_HIP(hipGetLastError());
    return VDTTFS_OK;
}

}  // namespace vdttfs
