// C ABI entry points of the 8-bit heads: argument checks, scratch and the
// order of launches.
#include <cmath>

#include "head.h"

using namespace vdttfs;

namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 64, kMaxGroups = 64;
constexpr int64_t kMaxRows = 0x7fffffff;
constexpr int kRowBytes = 128;  // rows of codes in scratch start on whole cache lines

int bad(const char* what, const char* why) { return set_error(VDTTFS_E_INVALID, "%s: %s", what, why); }

size_t elem_size(int elem) { return elem == VDTTFS_ELEM_BF16 || elem == VDTTFS_ELEM_F16 ? 2 : 4; }

int check_float_ptr(const char* what, const void* p, size_t align) {
    if (!p) return bad(what, "null buffer");
    if ((uintptr_t)p % align) return bad(what, "a float buffer is not aligned to its type");
    return VDTTFS_OK;
}

int check_in(const char* what, const void* x, int elem, int64_t ldx, int64_t rows, int cols) {
    if (elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_TIMES) return bad(what, "unknown input element type");
    if (rows < 0 || cols < 0) return bad(what, "negative size");
    if (rows > kMaxRows) return set_error(VDTTFS_E_UNSUPPORTED, "%s: 2^31 rows or more", what);
    if (ldx < cols) return bad(what, "leading dimension below the columns");
    if (rows > 0 && cols > 0) VD_TRY(check_float_ptr(what, x, elem_size(elem)));
    return VDTTFS_OK;
}

int check_out(const char* what, const void* out, int elem, int64_t ldo, int N) {
    if (elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_F16) return bad(what, "unknown output element type");
    if (ldo < N) return bad(what, "leading dimension below the columns");
    return check_float_ptr(what, out, elem_size(elem));
}

int check_channels(const char* what, int N) {
    if (N > VDTTFS_I8_MAX_N)
        return set_error(VDTTFS_E_UNSUPPORTED, "%s: %d output channels, at most %d", what, N, VDTTFS_I8_MAX_N);
    return VDTTFS_OK;
}

// Shape and weights of one product; the outputs are not empty.
int check_product(const char* what, const int8_t* w, int64_t ldw, const float* ch, const float* bias, int act,
                  int K) {
    if (act < VDTTFS_ACT_NONE || act > VDTTFS_ACT_SILU) return bad(what, "unknown activation");
    if (K > VDTTFS_I8_MAX_K)
        return set_error(VDTTFS_E_UNSUPPORTED, "%s: %d terms a sum, at most %d fit 32 bits", what, K, VDTTFS_I8_MAX_K);
    if (ldw < K) return bad(what, "leading dimension below the columns");
    if (K > 0 && !w) return bad(what, "null buffer");
    VD_TRY(check_float_ptr(what, ch, 4));
    if (bias) VD_TRY(check_float_ptr(what, bias, 4));
    return VDTTFS_OK;
}

int check_mnk(const char* what, int64_t M, int N, int K) {
    if (M < 0 || N < 0 || K < 0) return bad(what, "negative size");
    if (M > kMaxRows) return set_error(VDTTFS_E_UNSUPPORTED, "%s: 2^31 rows or more", what);
    return check_channels(what, N);
}

// The context's scratch of these calls, at least `bytes`; a buffer whose
// address a captured graph holds is set aside until the context ends.
int head_scratch(vdttfs_ctx* ctx, size_t bytes, unsigned char** out) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    VD_HIP(hipStreamIsCapturing(ctx->stream, &cs));
    const bool capturing = cs != hipStreamCaptureStatusNone;
    if (ctx->head.bytes < bytes) {
        if (capturing)
            return set_error(VDTTFS_E_UNSUPPORTED,
                             "the context's scratch is too small and cannot grow under stream capture: run the call "
                             "once before capturing it");
        VD_HIP(hipStreamSynchronize(ctx->stream));
        if (ctx->head.captured)
            ctx->split_kept.push_back(ctx->head.buf);
        else if (ctx->head.buf)
            VD_HIP(hipFree(ctx->head.buf));
        ctx->head.buf = nullptr;
        ctx->head.bytes = 0;
        ctx->head.captured = false;
        if (hipMalloc(&ctx->head.buf, bytes) != hipSuccess) {
            ctx->head.buf = nullptr;
            (void)hipGetLastError();
            return set_error(VDTTFS_E_NOMEM, "device allocation of %zu bytes failed", bytes);
        }
        ctx->head.bytes = bytes;
    }
    ctx->head.captured |= capturing;
    *out = static_cast<unsigned char*>(ctx->head.buf);
    return VDTTFS_OK;
}

// Parts of one scratch buffer, each on a 256-byte boundary.
struct Layout {
    size_t bytes = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += (n + 255) & ~size_t(255);
        return at;
    }
};

int64_t padded(int cols) { return ((int64_t)cols + kRowBytes - 1) / kRowBytes * kRowBytes; }

I8Args product(const int8_t* A, int64_t lda, const float* sa, const int8_t* B, int64_t ldb, const float* sb,
               const float* bias, void* out, int out_elem, int64_t ldo, int64_t M, int N, int K, int act) {
    I8Args a{};
    a.A = A;
    a.lda = lda;
    a.sa = sa;
    a.B = B;
    a.ldb = ldb;
    a.sb = sb;
    a.bias = bias;
    a.out = out;
    a.ldo = ldo;
    a.M = M;
    a.N = N;
    a.K = K;
    a.act = act;
    a.out_elem = out_elem;
    return a;
}

// Copies of the operands with rows on 128 bytes and zeros behind them, where
// the product asks for it: which, and their scratch.
bool off16(const int8_t* p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)ld) & 15) != 0; }
struct Copies {
    bool a, b;
    size_t bytes;
};
Copies copies_of(const I8Args& a) {
    if (!i8_wants_aligned(a)) return Copies{false, false, 0};
    const bool part = a.K % 16 != 0;
    Copies c{off16(a.A, a.lda) || (part && !a.a_padded), off16(a.B, a.ldb) || part, 0};
    Layout l;
    if (c.a) l.take((size_t)a.M * padded(a.K));
    if (c.b) l.take((size_t)a.N * padded(a.K));
    c.bytes = l.bytes;
    return c;
}

// The product, its operands copied first where copies_of says so; scratch of
// so many bytes, or none yet.
int dense(vdttfs_ctx* ctx, I8Args a, size_t bytes, unsigned char* buf) {
    const Copies c = copies_of(a);
    const int64_t ld = padded(a.K);
    if (c.bytes > bytes) VD_TRY(head_scratch(ctx, c.bytes, &buf));
    if (c.a) {
        VD_TRY(launch_realign(ctx, a.A, a.lda, a.M, a.K, reinterpret_cast<int8_t*>(buf), ld));
        a.A = reinterpret_cast<int8_t*>(buf);
        a.lda = ld;
        buf += ((size_t)a.M * ld + 255) & ~size_t(255);
    }
    if (c.b) {
        VD_TRY(launch_realign(ctx, a.B, a.ldb, a.N, a.K, reinterpret_cast<int8_t*>(buf), ld));
        a.B = reinterpret_cast<int8_t*>(buf);
        a.ldb = ld;
        if (c.a || a.a_padded) a.K = (int)ld;  // zeros on both sides
    }
    return launch_i8_dense(ctx, a);
}

}  // namespace

extern "C" {

int vdttfs_quant_rows(vdttfs_ctx* ctx, const void* d_x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* d_q,
                      int64_t ldq, float* d_scale) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_in("quant_rows", d_x, elem, ldx, rows, cols));
    if (ldq < cols) return bad("quant_rows", "leading dimension below the columns");
    if (rows == 0) return VDTTFS_OK;
    if (cols > 0 && !d_q) return bad("quant_rows", "null buffer");
    VD_TRY(check_float_ptr("quant_rows", d_scale, 4));
    return launch_quant_rows(ctx, d_x, elem, ldx, rows, cols, d_q, ldq, cols, d_scale);
}

int vdttfs_quant_kernel(vdttfs_ctx* ctx, const float* d_kernel, int C_in, int C_out, int8_t* d_w, int64_t ldw,
                        float* d_ch_scale) {
    VD_TRY(check_ctx(ctx));
    if (C_in < 0 || C_out < 0) return bad("quant_kernel", "negative size");
    if (ldw < C_in) return bad("quant_kernel", "leading dimension below the columns");
    if (C_out == 0) return VDTTFS_OK;
    VD_TRY(check_channels("quant_kernel", C_out));
    if (C_in > 0 && !d_w) return bad("quant_kernel", "null buffer");
    if (C_in > 0) VD_TRY(check_float_ptr("quant_kernel", d_kernel, 4));
    VD_TRY(check_float_ptr("quant_kernel", d_ch_scale, 4));
    return launch_quant_kernel(ctx, d_kernel, C_in, C_out, d_w, ldw, d_ch_scale);
}

int vdttfs_i8_matmul(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const int8_t* d_q, int64_t ldq,
                     const float* d_row_scale, const int8_t* d_w, int64_t ldw, const float* d_ch_scale,
                     const float* d_bias, int act, int64_t M, int N, int K) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_mnk("i8_matmul", M, N, K));
    if (M == 0 || N == 0) return VDTTFS_OK;
    VD_TRY(check_out("i8_matmul", d_out, out_elem, ldo, N));
    if (ldq < K) return bad("i8_matmul", "leading dimension below the columns");
    if (K > 0 && !d_q) return bad("i8_matmul", "null buffer");
    VD_TRY(check_float_ptr("i8_matmul", d_row_scale, 4));
    VD_TRY(check_product("i8_matmul", d_w, ldw, d_ch_scale, d_bias, act, K));
    const I8Args a = product(d_q, ldq, d_row_scale, d_w, ldw, d_ch_scale, d_bias, d_out, out_elem, ldo, M, N, K, act);
    const bool off = off16(d_q, ldq) || off16(d_w, ldw);
    if (small_ok(M, N, K, kElemCodes, off)) return launch_i8_small(ctx, d_q, kElemCodes, ldq, d_row_scale, a);
    return dense(ctx, a, 0, nullptr);
}

int vdttfs_i8_linear(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const void* d_x, int x_elem,
                     int64_t ldx, const int8_t* d_w, int64_t ldw, const float* d_ch_scale, const float* d_bias,
                     int act, int64_t M, int N, int K) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_mnk("i8_linear", M, N, K));
    if (M == 0 || N == 0) return VDTTFS_OK;
    VD_TRY(check_out("i8_linear", d_out, out_elem, ldo, N));
    VD_TRY(check_in("i8_linear", d_x, x_elem, ldx, M, K));
    VD_TRY(check_product("i8_linear", d_w, ldw, d_ch_scale, d_bias, act, K));
    const bool off = off16(d_w, ldw);
    if (small_ok(M, N, K, x_elem, off))
        return launch_i8_small(ctx, d_x, x_elem, ldx, nullptr,
                               product(nullptr, 0, nullptr, d_w, ldw, d_ch_scale, d_bias, d_out, out_elem, ldo, M, N,
                                       K, act));
    // the codes' rows end in zeros, so a weight row may too: whole chunks
    const int64_t ldq = padded(K);
    I8Args a = product(nullptr, ldq, nullptr, d_w, ldw, d_ch_scale, d_bias, d_out, out_elem, ldo, M, N, K, act);
    a.a_padded = true;
    const bool small = small_ok(M, N, K, kElemCodes, off);
    Layout l;
    const size_t at_q = l.take((size_t)M * ldq), at_s = l.take((size_t)M * 4);
    const size_t own = l.bytes;
    if (!small) l.take(copies_of(a).bytes);
    unsigned char* buf;
    VD_TRY(head_scratch(ctx, l.bytes, &buf));
    int8_t* q = reinterpret_cast<int8_t*>(buf + at_q);
    float* s = reinterpret_cast<float*>(buf + at_s);
    VD_TRY(launch_quant_rows(ctx, d_x, x_elem, ldx, M, K, q, ldq, (int)ldq, s));
    a.A = q;
    a.sa = s;
    if (small) return launch_i8_small(ctx, q, kElemCodes, ldq, s, a);
    return dense(ctx, a, l.bytes - own, buf + own);
}

int vdttfs_route(vdttfs_ctx* ctx, int32_t* d_idx, float* d_weight, int32_t* d_count, const void* d_logits, int elem,
                 int64_t ld, const float* d_bias, const uint8_t* d_row_mask, int64_t M,
                 const vdttfs_route_opts* opts) {
    VD_TRY(check_ctx(ctx));
    if (!opts) return bad("route", "null options");
    const vdttfs_route_opts& o = *opts;
    if (M < 0 || o.n_experts < 1 || o.top_k < 1) return bad("route", "size below 1 (rows: below 0)");
    if (o.n_experts > kMaxExperts || o.top_k > kMaxTopK || o.groups > kMaxGroups || M > kMaxRows / o.top_k)
        return set_error(VDTTFS_E_UNSUPPORTED, "route: more than %d experts, %d slots, %d groups or 2^31 pairs",
                         kMaxExperts, kMaxTopK, kMaxGroups);
    if (o.top_k > o.n_experts) return bad("route", "more slots than experts");
    if (o.score != VDTTFS_SCORE_SOFTMAX && o.score != VDTTFS_SCORE_SIGMOID) return bad("route", "unknown score");
    if (o.groups < 1 || o.n_experts % o.groups) return bad("route", "groups do not divide the experts");
    if (o.top_groups < 1 || o.top_groups > o.groups) return bad("route", "top_groups outside [1, groups]");
    if (o.group_top != 1 && o.group_top != 2) return bad("route", "group_top is 1 or 2");
    if (!std::isfinite(o.scale)) return bad("route", "scale is not finite");
    if (elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_F16) return bad("route", "unknown logit type");
    if (ld < o.n_experts) return bad("route", "leading dimension below the experts");
    if (d_count) VD_TRY(check_float_ptr("route", d_count, 4));
    if (M > 0) {
        VD_TRY(check_float_ptr("route", d_idx, 4));
        VD_TRY(check_float_ptr("route", d_weight, 4));
        VD_TRY(check_float_ptr("route", d_logits, elem_size(elem)));
        if (d_bias) VD_TRY(check_float_ptr("route", d_bias, 4));
    }
    return launch_route(ctx, d_idx, d_weight, d_count, d_logits, elem, ld, d_bias, d_row_mask, M, o);
}

int vdttfs_experts(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const void* d_x, int x_elem, int64_t ldx,
                   const int32_t* d_idx, const float* d_weight, int64_t M, int top_k,
                   const vdttfs_expert_layer* layer) {
    VD_TRY(check_ctx(ctx));
    if (!layer) return bad("experts", "null layer");
    const vdttfs_expert_layer& L = *layer;
    if (M < 0 || top_k < 1 || L.n_experts < 1 || L.d_in < 0 || L.d_hidden < 0 || L.d_out < 0)
        return bad("experts", "negative size, no slot or no expert");
    if (L.n_experts > kMaxExperts || top_k > kMaxTopK || M > kMaxRows / top_k)
        return set_error(VDTTFS_E_UNSUPPORTED, "experts: more than %d experts, %d slots or 2^31 pairs", kMaxExperts,
                         kMaxTopK);
    if (L.gated && L.d_hidden > kMaxRows / 2) return bad("experts", "hidden width too large");
    if (M == 0 || L.d_out == 0) return VDTTFS_OK;
    VD_TRY(check_channels("experts", L.d_out));
    VD_TRY(check_out("experts", d_out, out_elem, ldo, L.d_out));
    VD_TRY(check_in("experts", d_x, x_elem, ldx, M, L.d_in));
    VD_TRY(check_float_ptr("experts", d_idx, 4));
    VD_TRY(check_float_ptr("experts", d_weight, 4));
    const int H = L.gated ? 2 * L.d_hidden : L.d_hidden;
    if (L.d_in > VDTTFS_I8_MAX_K)  // where there is no first product too: its rows are quantised
        return set_error(VDTTFS_E_UNSUPPORTED, "experts: %d inputs, at most %d", L.d_in, VDTTFS_I8_MAX_K);
    if (H > 0) VD_TRY(check_product("experts", L.w1, L.d_in, L.s1, L.b1, L.act, L.d_in));
    VD_TRY(check_product("experts", L.w2, L.d_hidden, L.s2, L.b2, L.act, L.d_hidden));

    const int64_t pairs = M * top_k;
    const int64_t ldq = padded(L.d_in), ldh = padded(L.d_hidden);
    bool fuse1, fuse2;
    if (experts_small_ok(pairs, top_k, L, &fuse1, &fuse2)) {
        Layout l;
        const size_t at_q = l.take(fuse1 ? 0 : (size_t)M * ldq), at_s = l.take(fuse1 ? 0 : (size_t)M * 4);
        const size_t at_h = l.take((size_t)pairs * L.d_hidden * 4);
        const size_t at_hq = l.take(fuse2 ? 0 : (size_t)pairs * ldh), at_hs = l.take(fuse2 ? 0 : (size_t)pairs * 4);
        unsigned char* buf;
        VD_TRY(head_scratch(ctx, l.bytes, &buf));
        int8_t* q = reinterpret_cast<int8_t*>(buf + at_q);
        float* s = reinterpret_cast<float*>(buf + at_s);
        float* h = reinterpret_cast<float*>(buf + at_h);
        int8_t* hq = reinterpret_cast<int8_t*>(buf + at_hq);
        float* hs = reinterpret_cast<float*>(buf + at_hs);
        if (!fuse1) VD_TRY(launch_quant_rows(ctx, d_x, x_elem, ldx, M, L.d_in, q, ldq, (int)ldq, s));
        VD_TRY(fuse1 ? launch_expert_product(ctx, d_x, x_elem, ldx, nullptr, d_idx, pairs, top_k, L, h)
                     : launch_expert_product(ctx, q, kElemCodes, ldq, s, d_idx, pairs, top_k, L, h));
        if (!fuse2)
            VD_TRY(launch_quant_rows(ctx, h, VDTTFS_ELEM_F32, L.d_hidden, pairs, L.d_hidden, hq, ldh, (int)ldh, hs));
        return fuse2 ? launch_expert_out(ctx, h, false, L.d_hidden, nullptr, d_idx, d_weight, M, top_k, L, d_out,
                                         out_elem, ldo)
                     : launch_expert_out(ctx, hq, true, ldh, hs, d_idx, d_weight, M, top_k, L, d_out, out_elem, ldo);
    }
    const int bm = i8_tile_rows(pairs, L);
    const int64_t max_tiles = pairs / bm + (pairs < L.n_experts ? pairs : L.n_experts);
    Layout l;
    const size_t at_q = l.take((size_t)M * ldq), at_s = l.take((size_t)M * 4);
    // rows of whole vectors, so that they are stored and read as such
    const int64_t ldf = ((int64_t)L.d_hidden + 3) / 4 * 4, ldz = ((int64_t)L.d_out + 3) / 4 * 4;
    const size_t at_h = l.take((size_t)pairs * ldf * 4);
    const size_t at_hq = l.take((size_t)pairs * ldh), at_hs = l.take((size_t)pairs * 4);
    // The slots' products stay in 32 bits whatever the output's type: rounded to it
    // before their sum they would add an error of their own size, not of the sum's.
    const size_t at_z = l.take((size_t)pairs * ldz * 4);
    const size_t at_pair = l.take((size_t)pairs * 4), at_row = l.take((size_t)pairs * 4);
    const size_t at_tiles = l.take((size_t)max_tiles * sizeof(int4)), at_n = l.take(4);
    const size_t at_hist = l.take((size_t)dispatch_blocks(pairs) * L.n_experts * 4);
    // weights off 16 bytes: copied where every expert has rows enough to pay for it
    const bool copy1 = bm > 32 && H > 0 && L.d_in > 0 && off16(L.w1, L.d_in);
    const bool copy2 = bm > 32 && L.d_hidden > 0 && off16(L.w2, L.d_hidden);
    const size_t at_w1 = l.take(copy1 ? (size_t)L.n_experts * H * ldq : 0);
    const size_t at_w2 = l.take(copy2 ? (size_t)L.n_experts * L.d_out * ldh : 0);
    unsigned char* buf;
    VD_TRY(head_scratch(ctx, l.bytes, &buf));
    int8_t* q = reinterpret_cast<int8_t*>(buf + at_q);
    float* s = reinterpret_cast<float*>(buf + at_s);
    float* h = reinterpret_cast<float*>(buf + at_h);
    int8_t* hq = reinterpret_cast<int8_t*>(buf + at_hq);
    float* hs = reinterpret_cast<float*>(buf + at_hs);
    float* z = reinterpret_cast<float*>(buf + at_z);
    const Dispatch d{reinterpret_cast<int*>(buf + at_pair), reinterpret_cast<int*>(buf + at_row),
                     reinterpret_cast<int4*>(buf + at_tiles), reinterpret_cast<int*>(buf + at_n),
                     reinterpret_cast<int*>(buf + at_hist)};

    VD_TRY(launch_quant_dispatch(ctx, d_x, x_elem, ldx, M, L.d_in, q, ldq, (int)ldq, s, d_idx, pairs, top_k,
                                 L.n_experts, bm, d));
    I8Args a = product(q, ldq, s, L.w1, L.d_in, L.s1, L.b1, h, VDTTFS_ELEM_F32, ldf, 0, L.d_hidden, L.d_in,
                       L.act);
    a.tiles = d.tiles;
    a.n_tiles = d.n_tiles;
    a.max_tiles = (int)max_tiles;
    a.a_rows = d.row;
    a.b_stride = (int64_t)H * L.d_in;
    if (copy1) {
        int8_t* w = reinterpret_cast<int8_t*>(buf + at_w1);
        VD_TRY(launch_realign(ctx, L.w1, L.d_in, (int64_t)L.n_experts * H, L.d_in, w, ldq));
        a.B = w;
        a.ldb = ldq;
        a.b_stride = (int64_t)H * ldq;
        a.K = (int)ldq;  // zeros on both sides
    }
    a.s_stride = H;
    VD_TRY(launch_i8_grouped(ctx, a, L.gated != 0, bm));
    VD_TRY(launch_quant_rows(ctx, h, VDTTFS_ELEM_F32, ldf, pairs, L.d_hidden, hq, ldh, (int)ldh, hs));
    I8Args b = product(hq, ldh, hs, L.w2, L.d_hidden, L.s2, L.b2, z, VDTTFS_ELEM_F32, ldz, 0, L.d_out,
                       L.d_hidden, VDTTFS_ACT_NONE);
    b.tiles = d.tiles;
    b.n_tiles = d.n_tiles;
    b.max_tiles = (int)max_tiles;
    b.o_rows = d.pair;
    b.b_stride = (int64_t)L.d_out * L.d_hidden;
    if (copy2) {
        int8_t* w = reinterpret_cast<int8_t*>(buf + at_w2);
        VD_TRY(launch_realign(ctx, L.w2, L.d_hidden, (int64_t)L.n_experts * L.d_out, L.d_hidden, w, ldh));
        b.B = w;
        b.ldb = ldh;
        b.b_stride = (int64_t)L.d_out * ldh;
        b.K = (int)ldh;
    }
    b.s_stride = L.d_out;
    VD_TRY(launch_i8_grouped(ctx, b, false, bm));
    return launch_combine(ctx, d_out, out_elem, ldo, z, ldz, d_idx, d_weight, M, L.d_out, top_k, L.n_experts);
}

}  // extern "C"
