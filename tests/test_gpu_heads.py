"""The 8-bit heads (quantisation, products of codes, routing, experts) against
their definitions in 64 bits: types, odd sizes, strides, unaligned codes, rows
without experts, infinities and NaN, lengths of zero and one, and refusals.
Bounds are those of tests/headref.py, derived from the roundings alone."""
import ctypes

import numpy as np
import pytest

import headref as R
import vdttfs
from vdttfs import _lib
from test_gpu_scratch import Captured

pytestmark = pytest.mark.gpu
GUARD = 64  # bytes before and after an output that must stay as they were


@pytest.fixture(scope="module")
def ctx(gpu_ctx_factory):
    return gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))


class View:
    """A device array from a byte offset on."""

    def __init__(self, arr, offset=0):
        self.arr, self.ptr = arr, ctypes.c_void_p(arr.ptr.value + offset)


class Out:
    """An output with leading dimension ld between guard bytes."""

    def __init__(self, ctx, rows, cols, ld, dtype):
        self.rows, self.cols, self.ld, self.dt = rows, cols, ld, np.dtype(dtype)
        self.n = rows * ld * self.dt.itemsize
        self.arr = ctx.empty(2 * GUARD + self.n, np.uint8).fill(0x5A)
        self.ptr = ctypes.c_void_p(self.arr.ptr.value + GUARD)

    def get(self):
        h = self.arr.download()
        assert (h[:GUARD] == 0x5A).all() and (h[GUARD + self.n:] == 0x5A).all()
        m = h[GUARD:GUARD + self.n].view(self.dt).reshape(self.rows, self.ld)
        gap = np.ascontiguousarray(m[:, self.cols:]).view(np.uint8)
        assert (gap == 0x5A).all(), "bytes between the rows were written"
        return m[:, :self.cols]


def strided(x, ld):
    out = np.full((x.shape[0], ld), 77, x.dtype)
    out[:, :x.shape[1]] = x
    return out


def codes(rng, rows, cols):
    return np.clip(np.rint(rng.standard_normal((rows, cols)) * 40), -128, 127).astype(np.int8)


def check(got_bits, elem, y, d):
    got = R.from_bits(got_bits, elem).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    tol = R.out_bound(y, d, elem)
    with np.errstate(invalid="ignore"):
        off = np.abs(got - y) - tol
    worst = np.nanmax(off) if off.size and not np.isnan(off).all() else -1.0
    assert worst <= 0, (worst, np.unravel_index(np.nanargmax(off), off.shape))


# ---- quantisation ---------------------------------------------------------------
@pytest.mark.parametrize("elem", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 5), (5, 64, 0), (2, 1000, 1), (9, 513, 0), (4, 5000, 8),
                                           (3, 20001, 0), (300, 100, 12), (1, 0, 3)])
def test_quant_rows_codes_are_exact(ctx, elem, rows, cols, pad):
    rng = np.random.default_rng(rows * 1000 + cols + elem)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32)
    if rows > 2:
        x[1] = 0
    bits = R.to_bits(x, elem)
    q, s = Out(ctx, rows, cols, cols + pad, np.int8), Out(ctx, 1, rows, rows, np.float32)
    ctx.quant_rows(ctx.to_device(strided(bits, cols + pad + 1)), elem, cols + pad + 1, rows, cols, q, cols + pad, s)
    rq, rs = R.quant_rows(R.from_bits(bits, elem))
    np.testing.assert_array_equal(s.get()[0], rs)
    np.testing.assert_array_equal(q.get(), rq)


def test_quant_rows_of_non_finite_and_tiny_rows(ctx):
    x = np.ones((8, 130), np.float32)
    x[0, 3], x[1, 129], x[2, 64] = np.nan, np.inf, -np.inf
    x[3], x[4] = 1e-45, 3e-38     # max / 127 underflows to nothing, and to a subnormal scale
    x[5, ::2] = -3.3e38
    x[6] = -0.0
    q, s = Out(ctx, 8, 130, 130, np.int8), Out(ctx, 1, 8, 8, np.float32)
    ctx.quant_rows(ctx.to_device(x), R.F32, 130, 8, 130, q, 130, s)
    rq, rs = R.quant_rows(x)
    assert np.isnan(rs[:3]).all() and rs[3] == 0
    np.testing.assert_array_equal(s.get()[0], rs)
    np.testing.assert_array_equal(q.get(), rq)


def test_quant_rows_half_way_quotients_go_to_even(ctx):
    x = np.arange(-254, 255, dtype=np.float32)[None, :] / 2  # scale 1, every half
    q, s = Out(ctx, 1, 509, 509, np.int8), Out(ctx, 1, 1, 1, np.float32)
    ctx.quant_rows(ctx.to_device(x), R.F32, 509, 1, 509, q, 509, s)
    np.testing.assert_array_equal(q.get()[0], np.rint(x[0]).astype(np.int8))


@pytest.mark.parametrize("T,tfs", [(1, 0.0), (64, 0.0), (64, 32.0), (80, 40.0), (127, 0.0), (128, 0.0), (255, 3.5)])
def test_quant_rows_of_spike_times(gpu_ctx_factory, T, tfs):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=T, tfs=tfs, delta=16))
    rng = np.random.default_rng(T)
    t = np.floor(rng.random((7, 301)) * (T + tfs + 4)).astype(np.float32)
    t[rng.random(t.shape) < 0.3] = 9999.0
    t[0, :4], t[1, :3] = [np.nan, np.inf, -5.0, 1e9], [T + tfs - 0.25, T + tfs, tfs - 0.5]
    q, s = Out(c, 7, 301, 304, np.int8), Out(c, 1, 7, 7, np.float32)
    c.quant_rows(c.to_device(strided(t, 303)), R.TIMES, 303, 7, 301, q, 304, s)
    rq, rs = R.quant_times(t, T, tfs)
    np.testing.assert_array_equal(q.get(), rq)
    np.testing.assert_array_equal(s.get()[0], rs)


@pytest.mark.parametrize("c_in,c_out", [(1, 1), (16, 64), (37, 65), (512, 10), (300, 130)])
def test_quant_kernel_is_quant_rows_of_the_transpose(ctx, c_in, c_out):
    w = np.random.default_rng(c_in).standard_normal((c_in, c_out)).astype(np.float32)
    w[:, 0] = 0
    q, s = Out(ctx, c_out, c_in, c_in + 3, np.int8), Out(ctx, 1, c_out, c_out, np.float32)
    ctx.quant_kernel(ctx.to_device(w), c_in, c_out, q, c_in + 3, s)
    rq, rs = R.quant_rows(np.ascontiguousarray(w.T))
    np.testing.assert_array_equal(q.get(), rq)
    np.testing.assert_array_equal(s.get()[0], rs)


# ---- products -------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 16, 64), (1, 100, 4096), (2, 33, 15), (4, 64, 127), (5, 129, 1000), (16, 17, 128),
         (17, 64, 129), (31, 300, 513), (64, 64, 256), (65, 127, 300), (129, 257, 385), (300, 10, 77), (256, 512, 512),
         (7, 1024, 8192), (513, 1030, 640), (1100, 257, 300), (1500, 512, 128), (2100, 300, 1024), (1025, 70, 90), (1024, 1024, 400), (4100, 2600, 144), (2000, 2100, 208),
         (1300, 5000, 272), (900, 700, 1000), (2600, 2600, 1500), (2561, 2500, 1601), (1100, 4100, 384)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("elem,kind,bias,pad,shift", [(R.F32, R.NONE, False, 0, 0), (R.F32, R.SILU, True, 3, 1),
                                                      (R.BF16, R.RELU, True, 16, 0), (R.F16, R.SILU, False, 0, 0),
                                                      (R.F16, R.NONE, True, 5, 7)])
def test_matmul(ctx, M, N, K, elem, kind, bias, pad, shift):
    """pad: elements between rows; shift: bytes by which the codes miss their alignment."""
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    q, w = codes(rng, M, K), codes(rng, N, K)
    s = np.exp(rng.standard_normal(M)).astype(np.float32) / 50
    c = (rng.random(N) + 0.5).astype(np.float32) / 50
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    ld = K + pad
    dq = ctx.to_device(np.concatenate([np.zeros(shift, np.int8), strided(q, ld).ravel()]))
    dw = ctx.to_device(np.concatenate([np.zeros(shift, np.int8), strided(w, ld).ravel()]))
    out = Out(ctx, M, N, N + pad, R.np_type(elem))
    ctx.i8_matmul(out, elem, N + pad, View(dq, shift), ld, ctx.to_device(s), View(dw, shift), ld, ctx.to_device(c),
                  ctx.to_device(b) if bias else None, kind, M, N, K)
    y, d = R.product(q, s, w, c, b, kind)
    check(out.get(), elem, y, d)


@pytest.mark.parametrize("M,N,K", [(1, 64, 131071), (33, 40, 131071), (140, 70, 131071)])
def test_matmul_largest_sums_fit(ctx, M, N, K):
    """All codes at -128: the sums reach 2^31 - 2^14."""
    q, w = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    s, c = np.full(M, 1.0, np.float32), np.full(N, 1.0, np.float32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.i8_matmul(out, R.F32, N, ctx.to_device(q), K, ctx.to_device(s), ctx.to_device(w), K, ctx.to_device(c), None,
                  R.NONE, M, N, K)
    assert (out.get() == np.float32(16384.0 * K)).all()


@pytest.mark.parametrize("M,N", [(1, 5), (3, 70), (200, 130)])
def test_matmul_of_no_terms_is_the_bias(ctx, M, N):
    b = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    out, one = Out(ctx, M, N, N, np.float32), ctx.to_device(np.ones(max(M, N), np.float32))
    null = View(one, 0)
    ctx.i8_matmul(out, R.F32, N, null, 0, one, null, 0, one, ctx.to_device(b), R.NONE, M, N, 0)
    np.testing.assert_array_equal(out.get(), np.broadcast_to(b, (M, N)))


def test_matmul_past_32_bit_offsets(ctx):
    """Rows of codes 2.4 GB apart from first to last."""
    M, N, K, ld = 8192, 96, 200, 300032
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((M, K)).astype(np.float32), codes(rng, N, K)
    q, s = ctx.empty(M * ld, np.int8), ctx.empty(M, np.float32)
    ctx.quant_rows(ctx.to_device(x), R.F32, K, M, K, q, ld, s)
    c = np.full(N, 0.01, np.float32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.i8_matmul(out, R.F32, N, q, ld, s, ctx.to_device(w), K, ctx.to_device(c), None, R.NONE, M, N, K)
    rq, rs = R.quant_rows(x)
    check(out.get(), R.F32, *R.product(rq, rs, w, c, None, R.NONE))
    q.free()


@pytest.mark.parametrize("M,K", [(16, 7277), (100, 7277), (33, 9001), (50, 9301), (3, 20011)])
def test_products_of_long_odd_rows(ctx, M, K):
    N = 41
    rng = np.random.default_rng(K + M)
    x, w = rng.standard_normal((M, K)).astype(np.float32), codes(rng, N, K)
    c = (rng.random(N) / 50).astype(np.float32)
    q, s = R.quant_rows(x)
    dw, dc = ctx.to_device(w), ctx.to_device(c)
    lin, mul = Out(ctx, M, N, N, np.float32), Out(ctx, M, N, N, np.float32)
    ctx.i8_linear(lin, R.F32, N, ctx.to_device(x), R.F32, K, dw, K, dc, None, R.NONE, M, N, K)
    ctx.i8_matmul(mul, R.F32, N, ctx.to_device(q), K, ctx.to_device(s), dw, K, dc, None, R.NONE, M, N, K)
    for out in (lin, mul):
        check(out.get(), R.F32, *R.product(q, s, w, c, None, R.NONE))


@pytest.mark.parametrize("M", [1, 3, 16, 20, 150])
@pytest.mark.parametrize("x_elem", [R.F32, R.BF16, R.F16, R.TIMES])
def test_linear_is_quant_rows_then_matmul(ctx, M, x_elem):
    N, K, ldx = 70, 333, 340
    rng = np.random.default_rng(M)
    if x_elem == R.TIMES:
        x = np.floor(rng.random((M, K)) * 70).astype(np.float32)
        x[rng.random(x.shape) < 0.4] = 9999
        rq, rs = R.quant_times(x, 64, 0.0)
        bits = x
    else:
        x = (rng.standard_normal((M, K)) * 3).astype(np.float32)
        if M > 2:
            x[1, 5], x[2] = np.nan, 0  # one row poisoned, one empty; the others stay
        bits = R.to_bits(x, x_elem)
        rq, rs = R.quant_rows(R.from_bits(bits, x_elem))
    w, c = codes(rng, N, K), (rng.random(N) / 50).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32)
    out = Out(ctx, M, N, N + 1, np.float32)
    ctx.i8_linear(out, R.F32, N + 1, ctx.to_device(strided(bits, ldx)), x_elem, ldx, ctx.to_device(w), K,
                  ctx.to_device(c), ctx.to_device(b), R.NONE, M, N, K)
    check(out.get(), R.F32, *R.product(rq, rs, w, c, b, R.NONE))


def test_linear_again_smaller_and_larger(ctx):
    """Scratch of another call's size is neither read nor relied on."""
    rng = np.random.default_rng(2)
    for M, N, K in [(300, 100, 700), (3, 50, 33), (40, 64, 1000), (1, 8, 1), (20, 30, 129)]:
        x, w = rng.standard_normal((M, K)).astype(np.float32), codes(rng, N, K)
        c = np.full(N, 0.02, np.float32)
        out = Out(ctx, M, N, N, np.float32)
        ctx.i8_linear(out, R.F32, N, ctx.to_device(x), R.F32, K, ctx.to_device(w), K, ctx.to_device(c), None, R.NONE,
                      M, N, K)
        rq, rs = R.quant_rows(x)
        check(out.get(), R.F32, *R.product(rq, rs, w, c, None, R.NONE))


# ---- routing --------------------------------------------------------------------
ROUTES = [  # E, k, score, groups, top_groups, group_top, bias, renorm
    (4, 1, 0, 1, 1, 1, False, False), (1, 1, 0, 1, 1, 1, False, True), (8, 8, 1, 1, 1, 1, True, True),
    (60, 4, 0, 1, 1, 1, True, False), (64, 6, 1, 1, 1, 1, False, True), (64, 8, 1, 8, 3, 2, True, True),
    (48, 5, 0, 8, 8, 1, False, True), (100, 7, 1, 4, 2, 2, True, False), (128, 2, 0, 1, 1, 1, False, True),
    (160, 6, 0, 8, 3, 1, False, False), (256, 8, 1, 8, 4, 2, True, True), (252, 8, 0, 4, 2, 2, True, True),
    (384, 8, 1, 1, 1, 1, True, True), (512, 10, 0, 64, 5, 2, False, False), (1000, 64, 1, 1, 1, 1, True, True),
    (1024, 16, 0, 32, 4, 2, True, True), (7, 7, 1, 7, 2, 2, True, True), (192, 3, 1, 64, 1, 2, False, True)]


def run_route(ctx, l, elem, bias, rows, k, score, groups, top_groups, group_top, renorm, scale, pad=0, count=True):
    M, E = l.shape
    idx, wt, n = Out(ctx, M, k, k, np.int32), Out(ctx, M, k, k, np.float32), Out(ctx, 1, E, E, np.int32)
    ctx.route(idx, wt, n if count else None, ctx.to_device(strided(l, E + pad)), elem, E + pad,
              ctx.to_device(bias) if bias is not None else None, ctx.to_device(rows) if rows is not None else None, M,
              E, k, score=score, groups=groups, top_groups=top_groups, group_top=group_top, renorm=renorm,
              scale=scale)
    gi, gw = idx.get(), wt.get()
    if count:
        np.testing.assert_array_equal(n.get()[0], np.bincount(gi[gi >= 0], minlength=E))
    return gi, gw


@pytest.mark.parametrize("case", ROUTES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("elem,M,pad", [(R.F32, 1, 0), (R.F32, 700, 3), (R.BF16, 133, 0), (R.F16, 9001, 2)])
def test_route(ctx, case, elem, M, pad):
    E, k, score, groups, top_groups, group_top, has_bias, renorm = case
    rng = np.random.default_rng(E * 31 + M)
    l = (1.5 * rng.standard_normal((M, E))).astype(np.float32)
    rows = None
    if M > 8:
        l[rng.random(l.shape) < 0.1] = -np.inf
        l[rng.random(l.shape) < 0.02] = np.nan
        l[3], l[4] = -np.inf, np.nan
        l[5, :-1] = -np.inf
        rows = (rng.random(M) > 0.1).astype(np.uint8)
        rows[5] = 255
    bias = (0.05 * rng.standard_normal(E) / (1 if score else E)).astype(np.float32) if has_bias else None
    if has_bias and E > 8:
        bias[2], bias[3] = -np.inf, np.nan
    bits = R.to_bits(l, elem)
    args = (k, score, groups, top_groups, group_top, renorm, 2.5)
    gi, gw = run_route(ctx, bits, elem, bias, rows, *args, pad=pad)
    ri, rw, decided = R.route(R.from_bits(bits, elem), bias, rows, *args)
    assert decided.mean() > 0.5  # a choice of 64 has 64 gaps
    np.testing.assert_array_equal(gi[decided], ri[decided])
    tol = R.route_bound(E) * np.abs(rw) + 1e-37
    assert (np.abs(gw.astype(np.float64) - rw) <= tol)[decided].all()
    # the other rows are a right choice up to their near ties
    for m in np.nonzero(~decided)[0]:
        there = gi[m] >= 0
        assert len(set(gi[m][there])) == there.sum() == (ri[m] >= 0).sum()


@pytest.mark.parametrize("case", [  # groups that end inside a lane's experts, or leave lanes without any
    (12, 4, 0, 2, 1, 1, False, True), (48, 5, 1, 8, 3, 2, True, True), (24, 8, 1, 4, 3, 2, True, False),
    (60, 3, 0, 3, 2, 1, False, True), (35, 8, 1, 5, 2, 2, True, True), (51, 4, 0, 1, 1, 1, True, False),
    (198, 6, 1, 6, 3, 2, True, True), (250, 8, 0, 2, 1, 2, False, True), (16, 2, 1, 16, 5, 1, True, True)],
    ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("elem,M,pad", [(R.F32, 700, 0), (R.BF16, 133, 4), (R.F16, 5001, 1)])
def test_route_groups_of_any_size(ctx, case, elem, M, pad):
    test_route(ctx, case, elem, M, pad)


@pytest.mark.parametrize("E,groups", [(16, 1), (64, 4), (200, 1), (256, 8), (1024, 1)])
@pytest.mark.parametrize("score", [0, 1])
def test_route_ties_go_to_the_lowest_index(ctx, E, groups, score):
    """Logits of three values: most neighbours are equal."""
    rng = np.random.default_rng(E)
    l = rng.integers(0, 3, (257, E)).astype(np.float32)
    l[0] = 1.0
    args = (min(8, E), score, groups, max(1, groups // 2), 2, True, 1.0)
    gi, gw = run_route(ctx, l, R.F32, None, None, *args)
    ri, rw, decided = R.route(l, None, None, *args)
    assert decided.all()
    np.testing.assert_array_equal(gi, ri)
    assert (gi[0] == np.arange(min(8, E))).all()


@pytest.mark.parametrize("score", [0, 1])
def test_route_extreme_logits(ctx, score):
    low = np.finfo(np.float32).min
    l = np.zeros((6, 8), np.float32)
    l[0] = low                              # all at the lowest value: equal
    l[1], l[1, 3] = low, 5.0
    l[2, 2] = l[2, 6] = np.inf              # two certain experts
    l[3] = [200, 100, 0, -100, -200, -300, low, -np.inf]
    l[4] = -200.0
    l[5] = -np.inf
    gi, gw = run_route(ctx, l, R.F32, None, None, 3, score, 1, 1, 1, True, 1.0)
    assert not np.isnan(gw).any()
    assert (gi[5] == -1).all() and (gw[5] == 0).all()
    np.testing.assert_array_equal(gi[0], [0, 1, 2])
    assert gi[1, 0] == 3 and (gi[2, :2] == [2, 6]).all() and (gi[3] == [0, 1, 2]).all()
    np.testing.assert_array_equal(gi[4], [0, 1, 2])
    if score == 0:
        np.testing.assert_allclose(gw[0], 1 / 3, rtol=1e-6)
        np.testing.assert_array_equal(gw[1], [1, 0, 0])
        np.testing.assert_array_equal(gw[2], [0.5, 0.5, 0])
        np.testing.assert_allclose(gw[4], 1 / 3, rtol=1e-6)
    else:
        np.testing.assert_array_equal(gw[0], 0)  # every score underflows: nothing to divide by
        np.testing.assert_array_equal(gw[1], [1, 0, 0])
        np.testing.assert_array_equal(gw[2, :2], gw[2, 0])


def test_route_no_rows_clears_the_counts(ctx):
    n = ctx.empty(10, np.int32).fill(0xFF)
    one = ctx.empty(16, np.float32)
    ctx.route(one, one, n, one, R.F32, 10, None, None, 0, 10, 2)
    assert (n.download() == 0).all()


# ---- experts --------------------------------------------------------------------
def expert_case(rng, E, D, F, N, gated, bias):
    H = 2 * F if gated else F
    w1, w2 = codes(rng, E * H, D).reshape(E, H, D), codes(rng, E * N, F).reshape(E, N, F)
    s1 = ((0.5 + rng.random((E, H))) / 40 / np.sqrt(max(D, 1))).astype(np.float32)
    s2 = ((0.5 + rng.random((E, N))) / 40 / np.sqrt(max(F, 1))).astype(np.float32)
    b1 = (0.3 * rng.standard_normal((E, H))).astype(np.float32) if bias else None
    b2 = (0.3 * rng.standard_normal((E, N))).astype(np.float32) if bias else None
    return w1, s1, b1, w2, s2, b2


def choose(rng, M, k, E):
    idx = np.argsort(rng.random((M, E)), axis=1)[:, :k].astype(np.int32)
    wt = rng.random((M, k)).astype(np.float32)
    if M > 3:
        idx[1] = -1                 # a row without experts
        idx[2, k // 2:] = -1        # some slots empty
        idx[3, 0] = E               # outside: skipped like -1
        wt[1, 0] = np.nan           # the weight of a skipped slot is not read
    return idx, wt


def run_experts(ctx, bits, x_elem, ldx, idx, wt, weights, kind, gated, out_elem, pad=0):
    w1, s1, b1, w2, s2, b2 = weights
    E, H, D = w1.shape
    N, F = w2.shape[1:]
    M, k = idx.shape
    dev = [ctx.to_device(v) if v is not None else None for v in (w1, s1, b1, w2, s2, b2)]
    out = Out(ctx, M, N, N + pad, R.np_type(out_elem))
    ctx.experts(out, out_elem, N + pad, ctx.to_device(strided(bits, ldx)), x_elem, ldx, ctx.to_device(idx),
                ctx.to_device(wt), M, k, vdttfs.ExpertWeights(E, D, F, N, kind, gated, *dev))
    return out.get()


EXPERTS = [  # M, k, E, D, F, N
    (1, 1, 1, 1, 1, 1), (1, 6, 64, 128, 64, 96), (1, 2, 4, 33, 17, 10), (2, 2, 3, 100, 70, 65), (5, 1, 2, 64, 64, 64),
    (9, 4, 8, 130, 96, 33), (40, 2, 5, 77, 50, 129), (70, 8, 8, 64, 128, 64), (257, 2, 8, 512, 512, 10),
    (600, 3, 16, 96, 40, 72), (300, 4, 4, 256, 300, 260), (3000, 2, 12, 64, 33, 40),
    (900, 3, 3, 144, 208, 130), (1500, 1, 2, 250, 90, 300)]


@pytest.mark.parametrize("M,k,E,D,F,N", EXPERTS)
@pytest.mark.parametrize("x_elem,out_elem,kind,gated,bias,pad", [
    (R.F32, R.F32, R.RELU, False, True, 3), (R.BF16, R.BF16, R.SILU, True, False, 0),
    (R.F16, R.F16, R.SILU, True, True, 1), (R.TIMES, R.F32, R.NONE, False, False, 0)])
def test_experts(ctx, M, k, E, D, F, N, x_elem, out_elem, kind, gated, bias, pad):
    rng = np.random.default_rng(M * 13 + E + D)
    weights = expert_case(rng, E, D, F, N, gated, bias)
    idx, wt = choose(rng, M, k, E)
    if x_elem == R.TIMES:
        bits = np.floor(rng.random((M, D)) * 80).astype(np.float32)
        q, s = R.quant_times(bits, 64, 0.0)
    else:
        bits = R.to_bits(rng.standard_normal((M, D)).astype(np.float32), x_elem)
        q, s = R.quant_rows(R.from_bits(bits, x_elem))
    got = run_experts(ctx, bits, x_elem, D + pad, idx, wt, weights, kind, gated, out_elem, pad)
    skip = (idx < 0) | (idx >= E)
    y, d, mag = R.experts(q, s, np.where(skip, -1, idx), np.where(skip, 0, wt), *weights, kind, gated)
    if out_elem == R.BF16:
        d = d + R.OUT_U[R.BF16] * mag  # the slots' products may pass through the output's type
    check(got, out_elem, y, d)


@pytest.mark.parametrize("M,k,E,D,F,N", [
    (16, 16, 64, 32, 200, 40),  # sixteen experts a workgroup, eight waves
    (3, 9, 20, 24, 1000, 17), (7, 5, 9, 40, 130, 31), (30, 16, 16, 16, 65, 5), (2, 17, 20, 32, 70, 20),
    (1, 3, 3, 48, 4000, 16), (11, 1, 2, 30, 64, 100)])
@pytest.mark.parametrize("x_elem,out_elem,pad", [(R.F32, R.F32, 1), (R.BF16, R.BF16, 0)])
def test_experts_of_few_rows(ctx, M, k, E, D, F, N, x_elem, out_elem, pad):
    """Slots that do and do not divide a fragment's rows, and more of them; few and many experts a workgroup."""
    rng = np.random.default_rng(M * 7 + k)
    weights = expert_case(rng, E, D, F, N, False, True)
    idx, wt = choose(rng, M, k, E)
    bits = R.to_bits(rng.standard_normal((M, D)).astype(np.float32), x_elem)
    got = run_experts(ctx, bits, x_elem, D, idx, wt, weights, R.RELU, False, out_elem, pad)
    skip = (idx < 0) | (idx >= E)
    y, d, mag = R.experts(*R.quant_rows(R.from_bits(bits, x_elem)), np.where(skip, -1, idx), np.where(skip, 0, wt),
                          *weights, R.RELU, False)
    if out_elem == R.BF16:
        d = d + R.OUT_U[R.BF16] * mag
    check(got, out_elem, y, d)


def test_experts_uneven_and_unused(ctx):
    """All rows on one expert of many, then every slot of a row on the same one."""
    rng = np.random.default_rng(3)
    E, D, F, N, M = 40, 64, 48, 50, 333
    weights = expert_case(rng, E, D, F, N, False, True)
    x = rng.standard_normal((M, D)).astype(np.float32)
    q, s = R.quant_rows(x)
    for idx in (np.full((M, 1), 37, np.int32), np.full((M, 3), 5, np.int32), np.full((M, 2), -1, np.int32)):
        wt = rng.random(idx.shape).astype(np.float32)
        got = run_experts(ctx, x, R.F32, D, idx, wt, weights, R.RELU, False, R.F32)
        check(got, R.F32, *R.experts(q, s, idx, wt, *weights, R.RELU, False)[:2])


@pytest.mark.parametrize("M", [1, 2, 50, 300])
def test_experts_empty_widths_and_poisoned_rows(ctx, M):
    rng = np.random.default_rng(4)
    E, k = 6, 2
    idx = np.argsort(rng.random((M, E)), axis=1)[:, :k].astype(np.int32)
    wt = np.full((M, k), 0.5, np.float32)
    # no hidden channel: the biases alone
    weights = expert_case(rng, E, 20, 0, 12, False, True)
    got = run_experts(ctx, np.ones((M, 20), np.float32), R.F32, 20, idx, wt, weights, R.RELU, False, R.F32)
    np.testing.assert_allclose(got, 0.5 * weights[5][idx[:, 0]] + 0.5 * weights[5][idx[:, 1]], rtol=1e-6, atol=1e-7)
    # a NaN in one row reaches that row alone
    weights = expert_case(rng, E, 20, 16, 12, False, True)
    x = np.ones((M, 20), np.float32)
    x[M // 2, 7] = np.nan
    got = run_experts(ctx, x, R.F32, 20, idx, wt, weights, R.NONE, False, R.F32)
    assert np.isnan(got[M // 2]).all() and np.isnan(got).any(axis=1).sum() == 1


# ---- the same results by any path, and again -------------------------------------
def test_rows_do_not_depend_on_the_batch(ctx):
    """A row alone, in a small batch and in a large one: the same bits."""
    rng = np.random.default_rng(6)
    K, N, E, F = 200, 90, 4, 64
    x, w = rng.standard_normal((400, K)).astype(np.float32), codes(rng, N, K)
    c = ((0.5 + rng.random(N)) / 50).astype(np.float32)
    dw, dc = ctx.to_device(w), ctx.to_device(c)
    weights = expert_case(rng, E, K, F, N, True, True)
    idx = np.argsort(rng.random((400, E)), axis=1)[:, :2].astype(np.int32)
    wt = rng.random((400, 2)).astype(np.float32)
    lin, exp = [], []
    for M in (1, 7, 30, 400):
        out = Out(ctx, M, N, N, np.float32)
        ctx.i8_linear(out, R.F32, N, ctx.to_device(x[:M]), R.F32, K, dw, K, dc, None, R.SILU, M, N, K)
        lin.append(out.get()[0].copy())
        exp.append(run_experts(ctx, x[:M], R.F32, K, idx[:M], wt[:M], weights, R.SILU, True, R.F32)[0].copy())
    for v in lin[1:]:
        np.testing.assert_array_equal(v, lin[0])
    for v in exp[1:]:
        np.testing.assert_array_equal(v, exp[0])


def test_calls_can_be_captured_once_they_have_run(gpu_ctx_factory):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    rng = np.random.default_rng(8)
    M, k, E, D, F, N = 90, 2, 6, 96, 80, 40
    weights = expert_case(rng, E, D, F, N, True, False)
    dev = [c.to_device(v) if v is not None else None for v in weights]
    ew = vdttfs.ExpertWeights(E, D, F, N, R.SILU, True, *dev)
    x, logits = c.to_device(np.zeros((M, D), np.float32)), c.to_device(np.zeros((M, E), np.float32))
    idx, wt, n = c.empty((M, k), np.int32), c.empty((M, k), np.float32), c.empty(E, np.int32)
    out = c.empty((M, N), np.float32)

    def call():
        c.route(idx, wt, n, logits, R.F32, E, None, None, M, E, k, renorm=True)
        c.experts(out, R.F32, N, x, R.F32, D, idx, wt, M, k, ew)

    call()
    c.synchronize()
    g = Captured(c, call)
    for seed in range(3):
        r = np.random.default_rng(seed)
        x.upload(r.standard_normal((M, D)).astype(np.float32))
        logits.upload(r.standard_normal((M, E)).astype(np.float32))
        out.fill(0xFF)
        n.fill(0xFF)
        g.replay()
        c.synchronize()
        got, gi, gn = out.download(), idx.download(), n.download()
        call()
        c.synchronize()
        np.testing.assert_array_equal(got, out.download())
        np.testing.assert_array_equal(gi, idx.download())
        np.testing.assert_array_equal(gn, n.download())
        assert np.isfinite(got).all() and gn.sum() == M * k
        # a larger call grows the scratch; the graph keeps its own
        big = c.empty((2000, N), np.float32)
        c.i8_linear(big, R.F32, N, c.to_device(np.ones((2000, 5000 + seed * 3000), np.float32)), R.F32,
                    5000 + seed * 3000, c.empty(N * 8000 * 2, np.int8).fill(1), 11000, c.empty(N).fill(0), None,
                    R.NONE, 2000, N, 5000 + seed * 3000)
    g.close()


def test_scratch_does_not_grow_under_capture(gpu_ctx_factory):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    x, w = c.to_device(np.ones((100, 5000), np.float32)), c.empty((30, 5000), np.int8).fill(1)
    sc, out, n = c.to_device(np.ones(30, np.float32)), c.empty((100, 30), np.float32), c.empty(4, np.int32)
    logits, small = c.to_device(np.ones((3, 4), np.float32)), c.empty((3, 2), np.int32)
    wt = c.empty((3, 2), np.float32)
    seen = []

    def call():
        with pytest.raises(vdttfs.VdttfsError) as e:
            c.i8_linear(out, R.F32, 30, x, R.F32, 5000, w, 5000, sc, None, R.NONE, 100, 30, 5000)
        seen.append(e.value.code)
        c.route(small, wt, n, logits, R.F32, 4, None, None, 3, 4, 2)  # the capture goes on

    g = Captured(c, call)
    assert seen == [_lib.E_UNSUPPORTED]
    g.replay()
    c.synchronize()
    np.testing.assert_array_equal(small.download(), [[0, 1]] * 3)
    g.close()


# ---- refusals -------------------------------------------------------------------
def refused(code, fn, *a, **k):
    with pytest.raises(vdttfs.VdttfsError) as e:
        fn(*a, **k)
    assert e.value.code == code and str(e.value)


class Null:
    ptr = None


def test_refusals(ctx):
    f, q = ctx.empty(4096, np.float32), ctx.empty(4096, np.int8)
    i = ctx.empty(64, np.int32)
    odd, two = View(f, 2), View(f, 1)
    INV, UNS = _lib.E_INVALID, _lib.E_UNSUPPORTED
    for a in [(f, 4, 8, 2, 8, q, 8, f), (f, -1, 8, 2, 8, q, 8, f), (f, 0, 7, 2, 8, q, 8, f), (f, 0, 8, 2, 8, q, 7, f),
              (f, 0, 8, -1, 8, q, 8, f), (f, 0, 8, 2, -8, q, 8, f), (Null, 0, 8, 2, 8, q, 8, f),
              (f, 0, 8, 2, 8, Null, 8, f), (f, 0, 8, 2, 8, q, 8, Null), (odd, 0, 8, 2, 8, q, 8, f),
              (two, 1, 8, 2, 8, q, 8, f), (f, 0, 8, 2, 8, q, 8, odd)]:
        refused(INV, ctx.quant_rows, *a)
    refused(UNS, ctx.quant_rows, f, 0, 8, 1 << 31, 8, q, 8, f)
    for a in [(f, -1, 4, q, 8, f), (f, 4, -1, q, 8, f), (f, 8, 4, q, 7, f), (Null, 8, 4, q, 8, f),
              (f, 8, 4, Null, 8, f), (f, 8, 4, q, 8, Null)]:
        refused(INV, ctx.quant_kernel, *a)
    good = dict(d_out=f, out_elem=0, ldo=8, d_q=q, ldq=16, d_row_scale=f, d_w=q, ldw=16, d_ch_scale=f, d_bias=None,
                act=0, M=2, N=8, K=16)
    for bad in [dict(out_elem=3), dict(out_elem=-1), dict(ldo=7), dict(ldq=15), dict(ldw=15), dict(act=3), dict(act=-1),
                dict(M=-1), dict(N=-1), dict(K=-1), dict(d_out=Null), dict(d_q=Null), dict(d_w=Null),
                dict(d_row_scale=Null), dict(d_ch_scale=Null), dict(d_out=odd), dict(d_bias=odd),
                dict(d_row_scale=odd), dict(out_elem=2, d_out=two)]:
        refused(INV, ctx.i8_matmul, **{**good, **bad})
    refused(UNS, ctx.i8_matmul, **{**good, "K": 131072, "ldq": 131072, "ldw": 131072})
    refused(UNS, ctx.i8_matmul, **{**good, "M": 1 << 31})
    lin = {k: v for k, v in good.items() if k not in ("d_q", "ldq", "d_row_scale")}
    lin.update(d_x=f, x_elem=0, ldx=16)
    for bad in [dict(x_elem=4), dict(ldx=15), dict(d_x=Null), dict(d_x=odd), dict(ldo=7), dict(d_w=Null)]:
        refused(INV, ctx.i8_linear, **{**lin, **bad})
    refused(UNS, ctx.i8_linear, **{**lin, "K": 131072, "ldx": 131072, "ldw": 131072})
    rt = dict(d_idx=i, d_weight=f, d_count=None, d_logits=f, elem=0, ld=8, d_bias=None, d_row_mask=None, M=2, E=8,
              top_k=2)
    for bad in [dict(elem=3), dict(ld=7), dict(M=-1), dict(top_k=0), dict(top_k=9), dict(E=0), dict(groups=0),
                dict(groups=3), dict(groups=2, top_groups=3), dict(top_groups=0), dict(group_top=3), dict(group_top=0),
                dict(score=2), dict(scale=float("nan")), dict(scale=float("inf")), dict(d_idx=Null),
                dict(d_weight=Null), dict(d_logits=Null), dict(d_logits=odd), dict(d_count=odd)]:
        refused(INV, ctx.route, **{**rt, **bad})
    refused(UNS, ctx.route, **{**rt, "E": 1025, "ld": 1025})
    refused(UNS, ctx.route, **{**rt, "E": 128, "ld": 128, "top_k": 65})
    refused(UNS, ctx.route, **{**rt, "E": 128, "ld": 128, "groups": 128})
    refused(UNS, ctx.route, **{**rt, "M": 1 << 31})

    def exp(x_elem=0, out_elem=0, ldo=8, ldx=8, M=2, k=2, E=4, D=8, F=8, N=8, act=0, x=f, out=f, idx=i, wt=f, w1=q,
            s1=f, b1=None, w2=q, s2=f, b2=None):
        ctx.experts(out, out_elem, ldo, x, x_elem, ldx, idx, wt, M, k,
                    vdttfs.ExpertWeights(E, D, F, N, act, False, w1, s1, b1, w2, s2, b2))

    for bad in [dict(x_elem=4), dict(out_elem=3), dict(ldo=7), dict(ldx=7), dict(M=-1), dict(k=0), dict(E=0),
                dict(D=-1), dict(F=-1), dict(N=-1), dict(act=3), dict(x=Null), dict(out=Null), dict(idx=Null),
                dict(wt=Null), dict(w1=Null), dict(s1=Null), dict(w2=Null), dict(s2=Null), dict(x=odd), dict(b1=odd)]:
        refused(INV, exp, **bad)
    refused(UNS, exp, E=1025)
    refused(UNS, exp, k=65)
    refused(UNS, exp, M=1 << 30, k=2)
    refused(UNS, exp, D=131072, ldx=131072)
    refused(UNS, exp, F=131072)


def test_empty_calls_do_nothing(ctx):
    ctx.quant_rows(Null, 0, 8, 0, 8, Null, 8, Null)
    ctx.i8_matmul(Null, 0, 8, Null, 16, Null, Null, 16, Null, None, 0, 0, 8, 16)
    ctx.i8_linear(Null, 0, 8, Null, 0, 16, Null, 16, Null, None, 0, 3, 0, 16)
    ctx.experts(Null, 0, 8, Null, 0, 8, Null, Null, 0, 2,
                vdttfs.ExpertWeights(4, 8, 8, 8, 0, False, Null, Null, None, Null, Null, None))
