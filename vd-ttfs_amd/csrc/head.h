// Internal declarations of the 8-bit heads: quantisation, products of codes,
// routing and experts (vdttfs_quant_rows ... vdttfs_experts).
#pragma once

#include "common.h"

namespace vdttfs {

// A product of codes.  A: activations [rows][lda], B: weights [channels][ldb].
// Grouped (tiles != nullptr): row tile t belongs to expert tiles[t].x, starts
// at sorted row tiles[t].y and ends before tiles[t].z; the A row of sorted row
// i is a_rows[i] (i itself if null), its output row o_rows[i] (i if null).
struct I8Args {
    const int8_t* A;
    int64_t lda;
    const float* sa;  // per A row
    const int8_t* B;
    int64_t ldb;
    const float* sb;    // per channel
    const float* bias;  // per channel, nullable
    void* out;
    int64_t ldo;
    int64_t M;  // rows (grouped: unused)
    int N, K;   // N: output columns; gated products read 2 * N channels
    int act, out_elem;
    const int4* tiles;
    const int* n_tiles;
    const int* a_rows;
    const int* o_rows;
    int64_t b_stride;  // codes of one expert's B
    int s_stride;      // channels of one expert
    int max_tiles;     // bound on *n_tiles
    bool a_padded;     // A's rows end in zeros up to a multiple of 128
};

// Rows to codes; columns [cols, ldq_zero) of each row get 0.
int launch_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                      int64_t ldq, int cols_zero, float* scale);
int launch_quant_kernel(vdttfs_ctx* ctx, const float* kernel, int c_in, int c_out, int8_t* w, int64_t ldw,
                        float* scale);
// Rows and channels of the tile that a dense product takes.
struct I8Tile {
    int bm, bn;
};
I8Tile i8_dense_tile(int64_t M, int N, int K, bool aligned);
int launch_i8_dense(vdttfs_ctx* ctx, const I8Args& a);
bool i8_wants_aligned(const I8Args& a);
// Rows of codes to rows of ld_to, a multiple of 16, zeros from K on.
int launch_realign(vdttfs_ctx* ctx, const int8_t* from, int64_t ld, int64_t rows, int K, int8_t* to, int64_t ld_to);
// The product of few rows (a.A and a.lda unused), quantised in the kernel from
// elem, or codes with scales sa where elem is kElemCodes.
constexpr int kElemCodes = 4;
bool small_ok(int64_t M, int N, int K, int elem, bool off16);
int launch_i8_small(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, const float* sa, const I8Args& a);
// bm: rows of a tile of a grouped product (i8_tile_rows of the same call)
int launch_i8_grouped(vdttfs_ctx* ctx, const I8Args& a, bool gated, int bm);
int i8_tile_rows(int64_t pairs, const vdttfs_expert_layer& L);

// The experts of few pairs without a sort: whether to, and whether each product
// quantises its rows itself.  The first product, out float [pairs][d_hidden], x
// codes with scales sa where elem is kElemCodes; the second with the sum over
// slots, from h [pairs][d_hidden], floats quantised in the kernel, or codes.
bool experts_small_ok(int64_t pairs, int top_k, const vdttfs_expert_layer& L, bool* fuse1, bool* fuse2);
int launch_expert_product(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, const float* sa, const int32_t* idx,
                          int64_t pairs, int top_k, const vdttfs_expert_layer& L, float* out);
int launch_expert_out(vdttfs_ctx* ctx, const void* h, bool is_codes, int64_t ldh, const float* sa, const int32_t* idx,
                      const float* wt, int64_t M, int top_k, const vdttfs_expert_layer& L, void* out, int out_elem,
                      int64_t ldo);

int launch_route(vdttfs_ctx* ctx, int32_t* idx, float* wt, int32_t* count, const void* logits, int elem, int64_t ld,
                 const float* bias, const uint8_t* row_mask, int64_t M, const vdttfs_route_opts& o);

// The pairs (row, slot) sorted by expert.  pair[i]: row * top_k + slot of
// sorted row i, row[i]: its row; tiles as in I8Args with bm rows each.
struct Dispatch {
    int* pair;
    int* row;
    int4* tiles;
    int* n_tiles;
    int* hist;  // [blocks][n_experts] and scratch of the sort
};
int dispatch_blocks(int64_t pairs);
int launch_dispatch(vdttfs_ctx* ctx, const int32_t* idx, int64_t pairs, int top_k, int n_experts, int bm,
                    const Dispatch& d);
// launch_quant_rows and launch_dispatch, in one launch where they are small.
int launch_quant_dispatch(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, int8_t* q,
                          int64_t ldq, int cols_zero, float* scale, const int32_t* idx, int64_t pairs, int top_k,
                          int n_experts, int bm, const Dispatch& d);
// out[m] = sum over slots of weight * z[m * top_k + slot], z in rows of ldz, whole
// vectors of 4 floats
int launch_combine(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const float* z, int64_t ldz,
                   const int32_t* idx, const float* wt, int64_t M, int N, int top_k, int n_experts);

// Rows over their root mean square: floats to y, codes of 4 bits to q with
// scales ms, or codes of 8 bits to q with scale.
struct NormArgs {
    const void* x;
    int64_t ldx;
    const void* res;  // nullable
    int64_t ldr;
    void* sum;  // nullable; of the residual's type, and it may be the residual
    int64_t lds;
    const float* gain;  // nullable
    float eps;
    int64_t rows;
    int cols;
    void* y;
    int y_elem;
    int64_t ldy;
    void* q;
    int64_t ldq;
    float* scale;
    uint8_t* ms;
    int64_t ldms;
    int kind;  // set by the launch
};
int launch_norm(vdttfs_ctx* ctx, NormArgs a, int x_elem, int res_elem);

// Rows to microscaled codes of 4 bits.
int launch_mx4_quant_rows(vdttfs_ctx* ctx, const void* x, int elem, int64_t ldx, int64_t rows, int cols, uint8_t* q,
                          int64_t ldq, uint8_t* s, int64_t lds);
int launch_mx4_quant_kernel(vdttfs_ctx* ctx, const float* kernel, int c_in, int c_out, uint8_t* w, int64_t ldw,
                            uint8_t* s, int64_t lds);
// A product of microscaled rows: activations A [M], weights B [N].
struct Mx4Args {
    const uint8_t* A;
    int64_t lda;
    const uint8_t* sa;
    int64_t ldsa;
    const uint8_t* B;
    int64_t ldb;
    const uint8_t* sb;
    int64_t ldsb;
    const float* bias;  // per channel, nullable
    void* out;
    int64_t ldo;
    int64_t M;
    int N, K;
    int act, out_elem;
};
// The kernels of a product: fragments of 16 x 16 whose waves share K, tiles through
// registers, tiles loaded to LDS; and which operands (codes, scales) are copied first to
// rows on 16 bytes with zeros behind them.
enum Mx4Path { kMx4Few, kMx4Tile32, kMx4Tile64, kMx4Lds32, kMx4Lds64, kMx4Lds128, kMx4Lds256 };
struct Mx4Plan {
    Mx4Path path;
    bool a, sa, b, sb;
};
Mx4Plan mx4_plan(const Mx4Args& a);
struct Mx4Copies {
    struct {
        const uint8_t* q;
        int64_t ldq;
        const uint8_t* s;
        int64_t lds, rows;
        uint8_t *to_q, *to_s;  // NULL: stays
    } of[2];
};
int launch_mx4_realign(vdttfs_ctx* ctx, const Mx4Copies& c, int K, int64_t ldq_to, int64_t lds_to);
int launch_mx4(vdttfs_ctx* ctx, const Mx4Args& a, Mx4Path path);
// The product of few rows, quantised in the kernel (a.A and a.sa unused).
bool mx4_small_linear_ok(int64_t M, int K);
int launch_mx4_small_linear(vdttfs_ctx* ctx, const Mx4Args& a, const void* x, int elem, int64_t ldx);

// Rows to the order of their experts: place[row * top_k + slot], start[0 .. E]
// (nullable), and the rows themselves; hist: scratch of dispatch_place_bytes.
struct PlaceArgs {
    int32_t* place;
    int32_t* start;
    const int32_t* idx;
    int64_t M;
    int top_k, E;
};
// Few pairs: all of it in one launch, without scratch.
bool dispatch_few_ok(int64_t pairs, int top_k);
int launch_dispatch_few(vdttfs_ctx* ctx, const PlaceArgs& a, void* z, int64_t ldz, const void* x, int elem, int64_t ldx,
                        int cols);
size_t dispatch_place_bytes(int64_t pairs, int n_experts);
int launch_place(vdttfs_ctx* ctx, const PlaceArgs& a, int* hist);
int launch_dispatch_rows(vdttfs_ctx* ctx, const PlaceArgs& a, void* z, int64_t ldz, const void* x, int elem, int64_t ldx,
                         int cols);
// out[m] = sum over slots of wt * z[place] (wt null: of z[place])
int launch_gather_sum(vdttfs_ctx* ctx, void* out, int out_elem, int64_t ldo, const void* z, int z_elem, int64_t ldz,
                      const int32_t* place, const float* wt, int64_t M, int top_k, int cols);
// dz[place] = wt * dout (of z's type), dw = dout . z[place]; either nullable
int launch_combine_grad(vdttfs_ctx* ctx, void* dz, int64_t lddz, float* dw, const void* z, int z_elem, int64_t ldz,
                        const void* dout, int out_elem, int64_t ldo, const int32_t* place, const float* wt, int64_t M,
                        int top_k, int cols);

}  // namespace vdttfs
