// C ABI entry points of the heads' other operators: microscaled products, norms,
// rows to the order of their experts and back.
#include <cmath>

#include "head_check.h"

using namespace vdttfs;

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMxBlock = 32;

int64_t mx4_bytes(int cols) { return ((int64_t)cols + 1) / 2; }
int64_t mx4_blocks(int cols) { return ((int64_t)cols + kMxBlock - 1) / kMxBlock; }

int check_mx4(const char* what, const void* q, int64_t ldq, const void* s, int64_t lds, int cols) {
    if (ldq < mx4_bytes(cols)) return bad(what, "leading dimension below the codes of a row");
    if (lds < mx4_blocks(cols)) return bad(what, "leading dimension below the scales of a row");
    if (cols > 0 && (!q || !s)) return bad(what, "null buffer");
    return VDTTFS_OK;
}

int check_mx4_product(const char* what, const void* w, int64_t ldw, const void* ws, int64_t ldws, const float* bias,
                      int act, int K) {
    if (act < VDTTFS_ACT_NONE || act > VDTTFS_ACT_SILU) return bad(what, "unknown activation");
    VD_TRY(check_mx4(what, w, ldw, ws, ldws, K));
    if (bias) VD_TRY(check_float_ptr(what, bias, 4));
    return VDTTFS_OK;
}

// Rows of copies and of scratch: whole cache lines of codes.
int64_t mx4_ld(int K) { return (mx4_bytes(K) + 127) / 128 * 128; }
int64_t mx4_lds(int K) { return (mx4_ld(K) / 16 + 15) / 16 * 16; }

size_t mx4_copy_bytes(const Mx4Args& a, const Mx4Plan& p) {
    Layout l;
    if (p.a) l.take((size_t)a.M * mx4_ld(a.K));
    if (p.sa) l.take((size_t)a.M * mx4_lds(a.K));
    if (p.b) l.take((size_t)a.N * mx4_ld(a.K));
    if (p.sb) l.take((size_t)a.N * mx4_lds(a.K));
    return l.bytes;
}

// The product, its operands copied first where the plan says so.
int mx4_product(vdttfs_ctx* ctx, Mx4Args a, const Mx4Plan& p, unsigned char* buf) {
    const int64_t ld = mx4_ld(a.K), lds = mx4_lds(a.K);
    Layout l;
    Mx4Copies c{};
    c.of[0] = {a.A, a.lda, a.sa, a.ldsa, a.M, nullptr, nullptr};
    c.of[1] = {a.B, a.ldb, a.sb, a.ldsb, a.N, nullptr, nullptr};
    if (p.a) a.A = c.of[0].to_q = buf + l.take((size_t)a.M * ld), a.lda = ld;
    if (p.sa) a.sa = c.of[0].to_s = buf + l.take((size_t)a.M * lds), a.ldsa = lds;
    if (p.b) a.B = c.of[1].to_q = buf + l.take((size_t)a.N * ld), a.ldb = ld;
    if (p.sb) a.sb = c.of[1].to_s = buf + l.take((size_t)a.N * lds), a.ldsb = lds;
    VD_TRY(launch_mx4_realign(ctx, c, a.K, ld, lds));
    return launch_mx4(ctx, a, p.path);
}

int check_elem(const char* what, int elem) {
    return elem < VDTTFS_ELEM_F32 || elem > VDTTFS_ELEM_F16 ? bad(what, "unknown element type") : VDTTFS_OK;
}

int check_norm(const char* what, const void* x, int x_elem, int64_t ldx, const void* res, int res_elem, int64_t ldr,
               const void* sum, int64_t lds, const float* gain, float eps, int64_t rows, int cols) {
    VD_TRY(check_elem(what, x_elem));
    VD_TRY(check_in(what, x, x_elem, ldx, rows, cols));
    if (cols < 1) return bad(what, "rows without columns");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return bad(what, "eps is negative or not finite");
    if (sum && !res) return bad(what, "a sum without a residual");
    if (res) {
        VD_TRY(check_elem(what, res_elem));
        VD_TRY(check_in(what, res, res_elem, ldr, rows, cols));
        if (sum) {
            VD_TRY(check_out(what, sum, res_elem, lds, cols));
            if (sum == res && lds != ldr) return bad(what, "a sum in the residual's place with other rows");
        }
    }
    if (gain) VD_TRY(check_float_ptr(what, gain, 4));
    return VDTTFS_OK;
}

NormArgs norm_args(const void* x, int64_t ldx, const void* res, int64_t ldr, void* sum, int64_t lds, const float* gain,
                   float eps, int64_t rows, int cols) {
    NormArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.res = res;
    a.ldr = ldr;
    a.sum = sum;
    a.lds = lds;
    a.gain = gain;
    a.eps = eps;
    a.rows = rows;
    a.cols = cols;
    return a;
}

int check_pairs(const char* what, int64_t M, int top_k, int cols) {
    if (M < 0 || top_k < 1 || cols < 0) return bad(what, "negative size, or no slot");
    if (top_k > kMaxTopK || M > kMaxRows / top_k)
        return set_error(VDTTFS_E_UNSUPPORTED, "%s: more than %d slots or 2^31 pairs", what, kMaxTopK);
    return VDTTFS_OK;
}

// Floats of a matrix whose rows are there.
int check_matrix(const char* what, const void* p, int elem, int64_t ld, int cols) {
    VD_TRY(check_elem(what, elem));
    if (ld < cols) return bad(what, "leading dimension below the columns");
    return cols > 0 ? check_float_ptr(what, p, elem_size(elem)) : VDTTFS_OK;
}

}  // namespace

extern "C" {

int vdttfs_mx4_quant_rows(vdttfs_ctx* ctx, const void* d_x, int elem, int64_t ldx, int64_t rows, int cols,
                          uint8_t* d_q, int64_t ldq, uint8_t* d_s, int64_t lds) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_in("mx4_quant_rows", d_x, elem, ldx, rows, cols));
    if (rows == 0 || cols == 0) return VDTTFS_OK;
    VD_TRY(check_mx4("mx4_quant_rows", d_q, ldq, d_s, lds, cols));
    return launch_mx4_quant_rows(ctx, d_x, elem, ldx, rows, cols, d_q, ldq, d_s, lds);
}

int vdttfs_mx4_quant_kernel(vdttfs_ctx* ctx, const float* d_kernel, int C_in, int C_out, uint8_t* d_w, int64_t ldw,
                            uint8_t* d_ws, int64_t ldws) {
    VD_TRY(check_ctx(ctx));
    if (C_in < 0 || C_out < 0) return bad("mx4_quant_kernel", "negative size");
    if (C_in == 0 || C_out == 0) return VDTTFS_OK;
    VD_TRY(check_channels("mx4_quant_kernel", C_out));
    VD_TRY(check_mx4("mx4_quant_kernel", d_w, ldw, d_ws, ldws, C_in));
    VD_TRY(check_float_ptr("mx4_quant_kernel", d_kernel, 4));
    return launch_mx4_quant_kernel(ctx, d_kernel, C_in, C_out, d_w, ldw, d_ws, ldws);
}

int vdttfs_mx4_matmul(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const uint8_t* d_q, int64_t ldq,
                      const uint8_t* d_s, int64_t lds, const uint8_t* d_w, int64_t ldw, const uint8_t* d_ws,
                      int64_t ldws, const float* d_bias, int act, int64_t M, int N, int K) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_mnk("mx4_matmul", M, N, K));
    if (M == 0 || N == 0) return VDTTFS_OK;
    VD_TRY(check_out("mx4_matmul", d_out, out_elem, ldo, N));
    VD_TRY(check_mx4("mx4_matmul", d_q, ldq, d_s, lds, K));
    VD_TRY(check_mx4_product("mx4_matmul", d_w, ldw, d_ws, ldws, d_bias, act, K));
    const Mx4Args a{d_q, ldq, d_s, lds, d_w, ldw, d_ws, ldws, d_bias, d_out, ldo, M, N, K, act, out_elem};
    const Mx4Plan p = mx4_plan(a);
    unsigned char* buf = nullptr;
    const size_t bytes = mx4_copy_bytes(a, p);
    if (bytes) VD_TRY(head_scratch(ctx, bytes, &buf));
    return mx4_product(ctx, a, p, buf);
}

int vdttfs_mx4_linear(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const void* d_x, int x_elem,
                      int64_t ldx, const uint8_t* d_w, int64_t ldw, const uint8_t* d_ws, int64_t ldws,
                      const float* d_bias, int act, int64_t M, int N, int K) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_mnk("mx4_linear", M, N, K));
    if (M == 0 || N == 0) return VDTTFS_OK;
    VD_TRY(check_out("mx4_linear", d_out, out_elem, ldo, N));
    VD_TRY(check_in("mx4_linear", d_x, x_elem, ldx, M, K));
    VD_TRY(check_mx4_product("mx4_linear", d_w, ldw, d_ws, ldws, d_bias, act, K));
    Mx4Args a{nullptr, 0, nullptr, 0, d_w, ldw, d_ws, ldws, d_bias, d_out, ldo, M, N, K, act, out_elem};
    if (mx4_small_linear_ok(M, K)) return launch_mx4_small_linear(ctx, a, d_x, x_elem, ldx);
    a.lda = mx4_ld(K);
    a.ldsa = mx4_lds(K);
    const Mx4Plan p = mx4_plan(a);  // of the strides: the rows in scratch are aligned
    Layout l;
    const size_t at_q = l.take((size_t)M * a.lda), at_s = l.take((size_t)M * a.ldsa);
    const size_t own = l.bytes;
    l.take(mx4_copy_bytes(a, p));
    unsigned char* buf;
    VD_TRY(head_scratch(ctx, l.bytes, &buf));
    uint8_t *q = buf + at_q, *s = buf + at_s;
    VD_TRY(launch_mx4_quant_rows(ctx, d_x, x_elem, ldx, M, K, q, a.lda, s, a.ldsa));
    a.A = q;
    a.sa = s;
    return mx4_product(ctx, a, p, buf + own);
}

int vdttfs_norm_rows(vdttfs_ctx* ctx, void* d_y, int y_elem, int64_t ldy, const void* d_x, int x_elem, int64_t ldx,
                     const void* d_res, int res_elem, int64_t ldr, void* d_sum, int64_t ldsum, const float* d_gain,
                     float eps, int64_t rows, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_norm("norm_rows", d_x, x_elem, ldx, d_res, res_elem, ldr, d_sum, ldsum, d_gain, eps, rows, cols));
    if (rows == 0) return VDTTFS_OK;
    VD_TRY(check_out("norm_rows", d_y, y_elem, ldy, cols));
    NormArgs a = norm_args(d_x, ldx, d_res, ldr, d_sum, ldsum, d_gain, eps, rows, cols);
    a.y = d_y;
    a.y_elem = y_elem;
    a.ldy = ldy;
    return launch_norm(ctx, a, x_elem, res_elem);
}

int vdttfs_norm_quant(vdttfs_ctx* ctx, int8_t* d_q, int64_t ldq, float* d_scale, const void* d_x, int x_elem,
                      int64_t ldx, const void* d_res, int res_elem, int64_t ldr, void* d_sum, int64_t ldsum,
                      const float* d_gain, float eps, int64_t rows, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_norm("norm_quant", d_x, x_elem, ldx, d_res, res_elem, ldr, d_sum, ldsum, d_gain, eps, rows, cols));
    if (ldq < cols) return bad("norm_quant", "leading dimension below the columns");
    if (rows == 0) return VDTTFS_OK;
    if (!d_q) return bad("norm_quant", "null buffer");
    VD_TRY(check_float_ptr("norm_quant", d_scale, 4));
    NormArgs a = norm_args(d_x, ldx, d_res, ldr, d_sum, ldsum, d_gain, eps, rows, cols);
    a.q = d_q;
    a.ldq = ldq;
    a.scale = d_scale;
    return launch_norm(ctx, a, x_elem, res_elem);
}

int vdttfs_norm_mx4(vdttfs_ctx* ctx, uint8_t* d_q, int64_t ldq, uint8_t* d_s, int64_t lds, const void* d_x,
                    int x_elem, int64_t ldx, const void* d_res, int res_elem, int64_t ldr, void* d_sum, int64_t ldsum,
                    const float* d_gain, float eps, int64_t rows, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_norm("norm_mx4", d_x, x_elem, ldx, d_res, res_elem, ldr, d_sum, ldsum, d_gain, eps, rows, cols));
    if (rows == 0) return VDTTFS_OK;
    VD_TRY(check_mx4("norm_mx4", d_q, ldq, d_s, lds, cols));
    NormArgs a = norm_args(d_x, ldx, d_res, ldr, d_sum, ldsum, d_gain, eps, rows, cols);
    a.q = d_q;
    a.ldq = ldq;
    a.ms = d_s;
    a.ldms = lds;
    return launch_norm(ctx, a, x_elem, res_elem);
}

int vdttfs_dispatch(vdttfs_ctx* ctx, void* d_z, int64_t ldz, int32_t* d_place, int32_t* d_start, const void* d_x,
                    int elem, int64_t ldx, const int32_t* d_idx, int64_t M, int top_k, int n_experts, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_pairs("dispatch", M, top_k, cols));
    if (n_experts < 1) return bad("dispatch", "no expert");
    if (n_experts > kMaxExperts)
        return set_error(VDTTFS_E_UNSUPPORTED, "dispatch: more than %d experts", kMaxExperts);
    if (d_start) VD_TRY(check_float_ptr("dispatch", d_start, 4));
    VD_TRY(check_elem("dispatch", elem));
    if (M > 0) {
        VD_TRY(check_float_ptr("dispatch", d_place, 4));
        VD_TRY(check_float_ptr("dispatch", d_idx, 4));
        VD_TRY(check_matrix("dispatch", d_x, elem, ldx, cols));
        VD_TRY(check_matrix("dispatch", d_z, elem, ldz, cols));
    }
    const PlaceArgs a{d_place, d_start, d_idx, M, top_k, n_experts};
    if (dispatch_few_ok(M * top_k, top_k)) return launch_dispatch_few(ctx, a, d_z, ldz, d_x, elem, ldx, cols);
    unsigned char* buf = nullptr;
    const size_t bytes = dispatch_place_bytes(M * top_k, n_experts);
    if (bytes) VD_TRY(head_scratch(ctx, bytes, &buf));
    VD_TRY(launch_place(ctx, a, reinterpret_cast<int*>(buf)));
    return launch_dispatch_rows(ctx, a, d_z, ldz, d_x, elem, ldx, cols);
}

int vdttfs_combine(vdttfs_ctx* ctx, void* d_out, int out_elem, int64_t ldo, const void* d_z, int z_elem, int64_t ldz,
                   const int32_t* d_place, const float* d_weight, int64_t M, int top_k, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_pairs("combine", M, top_k, cols));
    if (M == 0 || cols == 0) return VDTTFS_OK;
    VD_TRY(check_matrix("combine", d_out, out_elem, ldo, cols));
    VD_TRY(check_matrix("combine", d_z, z_elem, ldz, cols));
    VD_TRY(check_float_ptr("combine", d_place, 4));
    if (d_weight) VD_TRY(check_float_ptr("combine", d_weight, 4));
    return launch_gather_sum(ctx, d_out, out_elem, ldo, d_z, z_elem, ldz, d_place, d_weight, M, top_k, cols);
}

int vdttfs_dispatch_grad(vdttfs_ctx* ctx, void* d_dx, int elem, int64_t lddx, const void* d_dz, int64_t lddz,
                         const int32_t* d_place, int64_t M, int top_k, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_pairs("dispatch_grad", M, top_k, cols));
    if (M == 0 || cols == 0) return VDTTFS_OK;
    VD_TRY(check_matrix("dispatch_grad", d_dx, elem, lddx, cols));
    VD_TRY(check_matrix("dispatch_grad", d_dz, elem, lddz, cols));
    VD_TRY(check_float_ptr("dispatch_grad", d_place, 4));
    return launch_gather_sum(ctx, d_dx, elem, lddx, d_dz, elem, lddz, d_place, nullptr, M, top_k, cols);
}

int vdttfs_combine_grad(vdttfs_ctx* ctx, void* d_dz, int64_t lddz, float* d_dw, const void* d_z, int z_elem,
                        int64_t ldz, const void* d_dout, int out_elem, int64_t lddo, const int32_t* d_place,
                        const float* d_weight, int64_t M, int top_k, int cols) {
    VD_TRY(check_ctx(ctx));
    VD_TRY(check_pairs("combine_grad", M, top_k, cols));
    VD_TRY(check_elem("combine_grad", z_elem));
    VD_TRY(check_elem("combine_grad", out_elem));
    if (!d_dz && !d_dw) return bad("combine_grad", "no gradient is asked for");
    if (M == 0) return VDTTFS_OK;
    VD_TRY(check_matrix("combine_grad", d_dout, out_elem, lddo, cols));
    if (d_dz) VD_TRY(check_matrix("combine_grad", d_dz, z_elem, lddz, cols));
    if (d_dw) {
        VD_TRY(check_float_ptr("combine_grad", d_dw, 4));
        VD_TRY(check_matrix("combine_grad", d_z, z_elem, ldz, cols));
    }
    VD_TRY(check_float_ptr("combine_grad", d_place, 4));
    if (d_weight) VD_TRY(check_float_ptr("combine_grad", d_weight, 4));
    return launch_combine_grad(ctx, d_dz, lddz, d_dw, d_z, z_elem, ldz, d_dout, out_elem, lddo, d_place, d_weight, M,
                               top_k, cols);
}

}  // extern "C"
