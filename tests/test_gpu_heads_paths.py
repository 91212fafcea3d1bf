"""The large forms of the 8-bit heads, each with a remainder in every dimension:
the 256-row tiles, grouped tiles of 64, 128 and 256 rows, copied weights, the
sort in three launches, and more rows than one pass of the routing grid.  Each
test asserts by the library's own rule that its sizes take the form that it is
for.  Sampled rows are compared with the definition in 64 bits (every row is
computed for itself), among them the first and the last of the matrix."""
import ctypes as C

import numpy as np
import pytest

import headref as R
import vdttfs
from vdttfs import _lib
from test_gpu_heads import View, Out, check, codes, ctx, expert_case, run_experts  # noqa: F401
from test_gpu_heads import test_route as check_route

pytestmark = pytest.mark.gpu


def tile_rows(M, k, E, D, F, N, gated):
    """Rows of the experts' tiles, by the library's rule (one for few pairs that are not sorted)."""
    L = _lib.ExpertLayer(E, D, F, N, 0, int(gated), *[None] * 6)
    few = vdttfs.lib()["_ZN6vdttfs16experts_small_okEliRK19vdttfs_expert_layerPbS3_"]
    few.argtypes, few.restype = [C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p], C.c_bool
    rows = vdttfs.lib()["_ZN6vdttfs12i8_tile_rowsElRK19vdttfs_expert_layer"]
    rows.argtypes, rows.restype = [C.c_int64, C.c_void_p], C.c_int
    a, b = C.c_bool(), C.c_bool()
    if few(M * k, k, C.byref(L), C.byref(a), C.byref(b)):
        return 1
    return rows(M * k, C.byref(L))


class Tile(C.Structure):
    _fields_ = [("bm", C.c_int), ("bn", C.c_int)]


def dense_tile(M, N, K, aligned=True):
    f = vdttfs.lib()["_ZN6vdttfs13i8_dense_tileEliib"]
    f.argtypes, f.restype = [C.c_int64, C.c_int, C.c_int, C.c_bool], Tile
    t = f(M, N, K, aligned)
    return t.bm, t.bn


def sample(rng, M, n=150):
    """Rows at both ends, around the tiles' edges, and some between."""
    edges = [m for t in (64, 128, 256) for m in (t - 1, t, (M - 1) // t * t - 1, (M - 1) // t * t)]
    return np.unique(np.clip(np.concatenate([[0, 1, M - 2, M - 1], edges, rng.integers(0, M, n)]), 0, M - 1))


# ---- dense products ---------------------------------------------------------------
@pytest.mark.parametrize("M,N,K", [
    (4100, 2600, 256),   # two tiles of K, nothing partial
    (4100, 2600, 272),   # a partial first tile of one chunk
    (4100, 2601, 400),   # an even number of tiles
    (5300, 4361, 640),   # an odd one; two rounds of the chip, the second half full
    (5400, 4353, 1520)])
@pytest.mark.parametrize("elem,kind,bias,pad", [(R.F32, R.SILU, True, 0), (R.BF16, R.NONE, False, 16),
                                                (R.F16, R.RELU, True, 3)])
def test_matmul_of_256_row_tiles(ctx, M, N, K, elem, kind, bias, pad):
    assert dense_tile(M, N, K) == (256, 256)
    rng = np.random.default_rng(M + N + K)
    q, w = codes(rng, M, K), codes(rng, N, K)
    s = np.exp(rng.standard_normal(M)).astype(np.float32) / 50
    c = (rng.random(N) + 0.5).astype(np.float32) / 50
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    out = Out(ctx, M, N, N + pad, R.np_type(elem))
    ctx.i8_matmul(out, elem, N + pad, ctx.to_device(q), K, ctx.to_device(s), ctx.to_device(w), K, ctx.to_device(c),
                  ctx.to_device(b) if bias else None, kind, M, N, K)
    at = sample(rng, M)
    check(out.get()[at], elem, *R.product(q[at], s[at], w, c, b, kind))


@pytest.mark.parametrize("M,N,K,shift,tile", [(4100, 2700, 1601, 0, (256, 256)), (4100, 2700, 1600, 3, (256, 256)),
                                              (3100, 2100, 1603, 5, (128, 128))])
def test_matmul_of_copied_operands(ctx, M, N, K, shift, tile):
    """Rows off 16 bytes in a product that pays for their copies."""
    assert float(M) * N * K >= 1e10 and dense_tile(M, N, (K + 127) // 128 * 128 if K % 16 else K) == tile
    rng = np.random.default_rng(K)
    q, w = codes(rng, M, K), codes(rng, N, K)
    s = np.exp(rng.standard_normal(M)).astype(np.float32) / 50
    c = (rng.random(N) + 0.5).astype(np.float32) / 50
    dq = ctx.to_device(np.concatenate([np.zeros(shift, np.int8), q.ravel()]))
    dw = ctx.to_device(np.concatenate([np.zeros(shift, np.int8), w.ravel()]))
    out = Out(ctx, M, N, N + 1, np.float32)
    ctx.i8_matmul(out, R.F32, N + 1, View(dq, shift), K, ctx.to_device(s), View(dw, shift), K, ctx.to_device(c), None,
                  R.NONE, M, N, K)
    at = sample(rng, M)
    check(out.get()[at], R.F32, *R.product(q[at], s[at], w, c, None, R.NONE))


@pytest.mark.parametrize("M,N,K,shift,tile", [(4000, 1000, 1001, 0, (64, 128)), (8200, 2100, 1008, 1, (128, 128)),
                                              (8200, 2601, 301, 0, (256, 256)), (4100, 2601, 384, 0, (256, 256))])
@pytest.mark.parametrize("x_elem", [R.F32, R.BF16, R.TIMES])
def test_linear_of_large_batches(ctx, M, N, K, shift, tile, x_elem):
    """Codes in scratch, and weights copied where their rows miss 16 bytes."""
    copied = K % 16 != 0 or shift
    assert float(M) * N * K >= 2e8 and dense_tile(M, N, (K + 127) // 128 * 128 if copied else K) == tile
    rng = np.random.default_rng(M + K + x_elem)
    if x_elem == R.TIMES:
        bits = np.floor(rng.random((M, K)) * 80).astype(np.float32)
        q, s = R.quant_times(bits, 64, 0.0)
    else:
        bits = R.to_bits((rng.standard_normal((M, K)) * 3).astype(np.float32), x_elem)
        q, s = R.quant_rows(R.from_bits(bits, x_elem))
    w, c = codes(rng, N, K), (rng.random(N) / 50).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32)
    dw = ctx.to_device(np.concatenate([np.zeros(shift, np.int8), w.ravel()]))
    out = Out(ctx, M, N, N, np.float32)
    ctx.i8_linear(out, R.F32, N, ctx.to_device(bits), x_elem, K, View(dw, shift), K, ctx.to_device(c),
                  ctx.to_device(b), R.RELU, M, N, K)
    at = sample(rng, M)
    check(out.get()[at], R.F32, *R.product(q[at], s[at], w, c, b, R.RELU))


# ---- experts ----------------------------------------------------------------------
def uneven(rng, M, k, E):
    """Distinct experts of a row, the last half of them rarely; some slots and rows empty, one outside."""
    score = rng.random((M, E)) + np.where(np.arange(E) < (E + 1) // 2, 0.6, 0.0)
    idx = np.argsort(-score, axis=1)[:, :k].astype(np.int32)
    wt = (rng.random((M, k)) - 0.3).astype(np.float32)
    idx[1::19] = -1
    idx[2::17, k // 2:] = -1
    idx[5, 0] = E
    wt[5, 0] = np.nan
    return idx, wt


# M, k, E, D, F, N, gated, rows of a tile: whole 16-byte rows, and ones that are copied
LARGE = [
    (1100, 2, 11, 144, 400, 420, False, 64), (1500, 2, 20, 80, 210, 417, True, 64),
    (1301, 2, 12, 101, 403, 422, False, 64), (2700, 4, 24, 33, 330, 390, True, 64),
    (1700, 3, 12, 272, 800, 700, False, 128), (2003, 3, 16, 400, 336, 650, True, 128),
    (1500, 3, 13, 301, 777, 701, False, 128), (3001, 3, 16, 303, 357, 645, True, 128),
    (3200, 3, 4, 272, 1100, 1040, False, 256), (3300, 3, 5, 528, 560, 1090, True, 256),
    (3200, 3, 4, 299, 1101, 1041, False, 256), (3300, 3, 5, 517, 551, 1089, True, 256),
    (700, 8, 8, 2101, 300, 1300, False, 64),  # rows too long for the launch that quantises and sorts
]


@pytest.mark.parametrize("M,k,E,D,F,N,gated,tile", LARGE)
@pytest.mark.parametrize("x_elem,out_elem,bias", [(R.F32, R.F32, True), (R.BF16, R.BF16, False)])
def test_experts_of_many_rows(ctx, M, k, E, D, F, N, gated, tile, x_elem, out_elem, bias):
    assert tile_rows(M, k, E, D, F, N, gated) == tile
    rng = np.random.default_rng(M + k + D)
    weights = expert_case(rng, E, D, F, N, gated, bias)
    idx, wt = uneven(rng, M, k, E)
    bits = R.to_bits(rng.standard_normal((M, D)).astype(np.float32), x_elem)
    kind = R.SILU if gated else R.RELU
    got = run_experts(ctx, bits, x_elem, D, idx, wt, weights, kind, gated, out_elem)
    at = np.union1d(sample(rng, M, 60), [5, 20, 19])
    q, s = R.quant_rows(R.from_bits(bits[at], x_elem))
    skip = (idx[at] < 0) | (idx[at] >= E)
    y, d, _ = R.experts(q, s, np.where(skip, -1, idx[at]), np.where(skip, 0, wt[at]), *weights, kind, gated)
    check(got[at], out_elem, y, d)


@pytest.mark.parametrize("M,k,E", [(4097, 2, 5), (3000, 6, 1000), (9001, 1, 7), (50000, 3, 33)])
def test_experts_sorted_in_three_launches(ctx, M, k, E):
    """More pairs than one workgroup sorts: no, few and many rows an expert, and all on one."""
    assert M * k > 8192
    D, F, N = 40, 33, 25
    rng = np.random.default_rng(M)
    weights = expert_case(rng, E, D, F, N, False, True)
    x = rng.standard_normal((M, D)).astype(np.float32)
    for case in ("spread", "one", "none"):
        idx, wt = uneven(rng, M, k, E)
        if case != "spread":
            idx[:] = E - 1 if case == "one" else -1
        wt = np.nan_to_num(wt)
        got = run_experts(ctx, x, R.F32, D, idx, wt, weights, R.RELU, False, R.F32)
        at = sample(rng, M, 300)
        skip = (idx[at] < 0) | (idx[at] >= E)
        y, d, _ = R.experts(*R.quant_rows(x[at]), np.where(skip, -1, idx[at]), np.where(skip, 0, wt[at]), *weights,
                            R.RELU, False)
        check(got[at], R.F32, y, d)


# ---- routing ----------------------------------------------------------------------
@pytest.mark.parametrize("case", [(256, 8, 1, 8, 4, 2, True, True), (60, 4, 0, 1, 1, 1, True, False),
                                  (250, 8, 0, 2, 1, 2, False, True), (512, 8, 1, 8, 3, 2, True, True)],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("elem,M,pad", [(R.F32, 20001, 0), (R.BF16, 40007, 1)])
def test_route_of_more_rows_than_the_grid(ctx, case, elem, M, pad):
    """256 workgroups of 64 rows (past 256 experts 1024 of 4): each goes on to further rows."""
    assert M > 256 * 64
    check_route(ctx, case, elem, M, pad)
