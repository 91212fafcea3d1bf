"""Rows over their root mean square, with a residual: floats, 8-bit codes and
microscaled 4-bit codes against their definitions in 64 bits."""
import numpy as np
import pytest

import headref as R
import moreref as Q
import vdttfs
from test_gpu_heads import Null, Out, View, check, refused, strided
from test_gpu_scratch import Captured
from vdttfs import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(gpu_ctx_factory):
    return gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))


class Case:
    """Inputs of one call on the device and its results by definition."""

    def __init__(self, ctx, x, x_elem, res=None, res_elem=R.F32, gain=None, eps=1e-6, pad=0):
        self.M, self.K, self.ctx, self.x_elem, self.res_elem, self.pad = *x.shape, ctx, x_elem, res_elem, pad
        self.eps, self.ld = eps, x.shape[1] + pad
        xb = R.to_bits(x, x_elem)
        rb = None if res is None else R.to_bits(res, res_elem)
        self.dx = ctx.to_device(strided(xb, self.ld))
        self.dr = None if res is None else ctx.to_device(strided(rb, self.ld))
        self.dg = None if gain is None else ctx.to_device(gain)
        self.h, self.u, self.inv, self.y = Q.norm(R.from_bits(xb, x_elem),
                                                  None if res is None else R.from_bits(rb, res_elem), gain, eps)

    def rows(self, sum_=None, lds=None, res=None):
        return (self.dx, self.x_elem, self.ld, self.dr, self.res_elem, self.ld, sum_, lds or self.K, self.dg, self.eps,
                self.M, self.K)

    def sums(self):
        return Out(self.ctx, self.M, self.K, self.K + self.pad, R.np_type(self.res_elem)) if self.dr else None

    def check_sum(self, out):
        if out is not None:
            np.testing.assert_array_equal(out.get(), R.to_bits(self.h, self.res_elem))

    def check_y(self, bits, elem):
        check(bits, elem, self.y, Q.NORM_U * np.abs(self.y) + 2.0 ** -148)

    def floats(self, elem):
        out, s = Out(self.ctx, self.M, self.K, self.K + self.pad, R.np_type(elem)), self.sums()
        self.ctx.norm_rows(out, elem, self.K + self.pad, *self.rows(s, self.K + self.pad))
        self.check_y(out.get(), elem)
        self.check_sum(s)

    def codes8(self):
        q, sc, s = Out(self.ctx, self.M, self.K, self.K + self.pad, np.int8), Out(self.ctx, 1, self.M, self.M, np.float32), self.sums()
        self.ctx.norm_quant(q, self.K + self.pad, sc, *self.rows(s, self.K + self.pad))
        rq, rs = R.quant_rows(self.u)
        np.testing.assert_array_equal(q.get(), rq)
        want = rs.astype(np.float64) * self.inv[:, 0]
        got = sc.get()[0]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        with np.errstate(invalid="ignore"):
            assert not (np.abs(got - want) > Q.NORM_U * np.abs(want) + 2.0 ** -148).any()
        self.check_sum(s)

    def codes4(self):
        n, b = (self.K + 1) // 2, -(-self.K // 32)
        q, sc, s = Out(self.ctx, self.M, n, n + self.pad, np.uint8), Out(self.ctx, self.M, b, b + self.pad, np.uint8), self.sums()
        self.ctx.norm_mx4(q, n + self.pad, sc, b + self.pad, *self.rows(s, self.K + self.pad))
        got = Q.mx4_values(Q.mx4_unpack(q.get(), self.K), sc.get())
        self.check_sum(s)
        # y is known to NORM_U: where both ends of that give the same code, it is that code; else one of the two
        lo, hi = (Q.mx4_values(*Q.mx4_quant(self.y * (1 + e * Q.NORM_U))) for e in (-1, 1))
        same = (lo == hi) | (np.isnan(lo) & np.isnan(hi))
        np.testing.assert_array_equal(got[same], lo[same])
        assert ((got == lo) | (got == hi))[~same].all()
        assert same.mean() > 0.9


TYPES = [(R.F32, R.F32), (R.BF16, R.BF16), (R.F16, R.F32), (R.BF16, R.F16), (R.F32, None), (R.F16, None), (R.F16, R.F16),
         (R.F32, R.BF16), (R.BF16, None), (R.BF16, R.F32), (R.F32, R.F16), (R.F16, R.BF16)]
SIZES = [(1, 1, 0), (3, 2, 1), (1, 31, 0), (7, 33, 3), (2, 128, 0), (40, 129, 5), (33, 256, 0), (9, 500, 1), (5, 513, 0),
         (1200, 1000, 8), (1, 1024, 0), (1030, 1024, 0), (3, 2048, 2), (2, 2500, 0), (1, 4096, 0), (5, 4100, 3),
         (2, 8192, 0), (3, 8200, 1), (1, 16384, 0), (2, 16400, 0), (3, 50001, 1)]


def inputs(M, K, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)))).astype(np.float32)
    r = (rng.standard_normal((M, K)) * 2).astype(np.float32)
    return x, r, (1 + 0.3 * rng.standard_normal(K)).astype(np.float32)


@pytest.mark.parametrize("M,K,pad", SIZES)
@pytest.mark.parametrize("x_elem,res_elem", TYPES[:6])
def test_norms(ctx, M, K, pad, x_elem, res_elem):
    x, r, g = inputs(M, K, M * 31 + K)
    c = Case(ctx, x, x_elem, None if res_elem is None else r, res_elem or 0, g, 1e-6, pad)
    c.floats(R.F32)
    c.codes8()
    c.codes4()


@pytest.mark.parametrize("M,K,pad", [(4, 96, 0), (5, 700, 3), (3, 3001, 0), (1, 9000, 0), (2, 20000, 5)])
@pytest.mark.parametrize("x_elem,res_elem", TYPES)
@pytest.mark.parametrize("elem", [R.F32, R.BF16, R.F16])
def test_norms_of_all_types(ctx, M, K, pad, x_elem, res_elem, elem):
    x, r, g = inputs(M, K, K)
    Case(ctx, x, x_elem, None if res_elem is None else r, res_elem or 0, g if K % 2 else None, 1e-5, pad).floats(elem)


@pytest.mark.parametrize("K", [1, 100, 600, 3000, 20000])
def test_norms_in_place_and_unaligned(ctx, K):
    """The sum in the residual's place; rows that start where their type allows and no more."""
    M = 5
    x, r, g = inputs(M, K, K)
    for elem in (R.F32, R.BF16):
        size = 4 if elem == R.F32 else 2
        xb, rb = R.to_bits(x, elem), R.to_bits(r, elem)
        shift = lambda a: View(ctx.to_device(np.concatenate([a.ravel()[:1], a.ravel()])), size)  # noqa: E731
        dx, dr, dg = shift(xb), shift(rb), View(ctx.to_device(np.concatenate([g[:1], g])), 4)
        out = Out(ctx, M, K, K, R.np_type(elem))
        ctx.norm_rows(out, elem, K, dx, elem, K, dr, elem, K, dr, K, dg, 1e-6, M, K)
        h, _, _, y = Q.norm(R.from_bits(xb, elem), R.from_bits(rb, elem), g, 1e-6)
        check(out.get(), elem, y, Q.NORM_U * np.abs(y) + 2.0 ** -148)
        np.testing.assert_array_equal(dr.arr.download()[1:].reshape(M, K), R.to_bits(h, elem))


@pytest.mark.parametrize("M,K", [(9, 7), (40, 9), (1100, 513), (700, 1025), (900, 1541), (300, 2049), (200, 4099),
                                 (150, 8191), (60, 8195), (20, 16385)])
def test_row_ends_in_place(ctx, M, K):
    """A row's last values are read with its neighbours', which the sum replaces."""
    x, r, g = inputs(M, K, K)
    for elem in (R.F32, R.F16):
        xb, rb = R.to_bits(x, elem), R.to_bits(r, elem)
        dx, dr = ctx.to_device(xb), ctx.to_device(rb)
        out = Out(ctx, M, K, K + 1, np.float32)
        ctx.norm_rows(out, R.F32, K + 1, dx, elem, K, dr, elem, K, dr, K, ctx.to_device(g), 1e-6, M, K)
        h, _, _, y = Q.norm(R.from_bits(xb, elem), R.from_bits(rb, elem), g, 1e-6)
        check(out.get(), R.F32, y, Q.NORM_U * np.abs(y) + 2.0 ** -148)
        np.testing.assert_array_equal(dr.download(), R.to_bits(h, elem))


@pytest.mark.parametrize("K", [40, 300, 2000, 20000])
def test_norms_of_the_largest_and_smallest_rows(ctx, K):
    """Squares past either end of 32 bits, zeros, and rows that are not finite."""
    rng = np.random.default_rng(K)
    x = rng.standard_normal((12, K)).astype(np.float32)
    x[0] *= 1e38 / np.abs(x[0]).max()
    x[1] *= np.float32(1e-30)
    x[2] *= np.float32(1e-42)   # subnormals
    x[3] = 0
    x[4] = np.finfo(np.float32).max
    x[5] = 0
    x[5, K // 2] = 1e-45
    x[6] *= np.float32(2.0 ** 63)
    x[7, ::2] = 1e-25
    x[8] *= np.float32(1e19)
    x[9, 3] = np.nan
    x[10] = -0.0
    x[11, ::3] = 2e38
    g = (1 + 0.3 * rng.standard_normal(K)).astype(np.float32)
    g[g > 1] = 1  # the largest rows' u stays finite
    for eps in (0.0, 1e-6, 1e-30, 3.0):
        c = Case(ctx, x, R.F32, None, 0, g, eps)
        for run in (lambda: c.floats(R.F32), c.codes8):
            run()
        # a row of zeros is zeros whatever eps
        assert (c.y[3] == 0).all()
    c = Case(ctx, x[:9], R.F32, None, 0, g, 0.0)
    c.codes4()


def test_an_infinity_leaves_its_row_alone(ctx):
    for K in (50, 700, 20000):
        x = np.random.default_rng(K).standard_normal((4, K)).astype(np.float32)
        x[1, 7], x[2, 9] = np.inf, -np.inf
        out = Out(ctx, 4, K, K, np.float32)
        q, s = Out(ctx, 4, K, K, np.int8), Out(ctx, 1, 4, 4, np.float32)
        d = ctx.to_device(x)
        ctx.norm_rows(out, R.F32, K, d, R.F32, K, None, 0, 0, None, 0, None, 1e-6, 4, K)
        ctx.norm_quant(q, K, s, d, R.F32, K, None, 0, 0, None, 0, None, 1e-6, 4, K)
        y, sc = out.get(), s.get()[0]
        for m, c in ((1, 7), (2, 9)):  # the formula: inf / inf, and the others over inf
            assert np.isnan(y[m, c]) and (np.delete(y[m], c) == 0).all()
        assert np.isfinite(y[[0, 3]]).all() and np.isnan(sc[[1, 2]]).all() and np.isfinite(sc[[0, 3]]).all()
        assert (q.get()[1:3] == 0).all()


@pytest.mark.parametrize("M", [1, 3, 5000])
def test_rows_do_not_depend_on_the_batch(ctx, M):
    K = 96
    x, r, g = inputs(5000, K, 1)
    one = None
    for n in {1, M}:
        out = Out(ctx, n, K, K, np.float32)
        ctx.norm_rows(out, R.F32, K, ctx.to_device(x[:n]), R.F32, K, ctx.to_device(r[:n]), R.F32, K, None, K,
                      ctx.to_device(g), 1e-6, n, K)
        first = out.get()[0].copy()
        one = first if one is None else one
        np.testing.assert_array_equal(first, one)


@pytest.mark.parametrize("K", [5, 100, 250, 500, 1000, 1500, 2000, 4100, 9000, 20000])
@pytest.mark.parametrize("res_elem", [None, R.F32])
def test_gains_that_carry_large_rows_past_the_largest_float(ctx, K, res_elem):
    """Finite rows give finite results: h * gain leaves the range of 32 bits, y does not."""
    rng = np.random.default_rng(K)
    M = 11
    v = rng.uniform(0.5, 1, (M, K)) * rng.choice([-1, 1], (M, K))
    top = np.array([3e38, 3.4e38, 1e30, 2.0 ** 65, 1.0, 1e37, 3e38, 1e35, 1e25, 3.4e38, 1e-30])
    x = (v * top[:, None]).astype(np.float32)
    r = None if res_elem is None else (x * np.float32(-0.25)).astype(np.float32)
    g = (rng.uniform(1, 2, K) * np.exp2(rng.integers(0, 28, K))).astype(np.float32)
    for eps in (0.0, 1e-6):
        c = Case(ctx, x, R.F32, r, res_elem or 0, g, eps)
        h, g64 = c.h.astype(np.float64), g.astype(np.float64)
        c.y = h * g64 * c.inv
        assert np.isfinite(c.y).all() and (K < 100 or not np.isfinite(c.u).all())
        c.floats(R.F32)
        c.floats(R.BF16)
        c.codes4()
        # the 8-bit codes are those of u times any power of two
        q, sc, s = Out(ctx, M, K, K, np.int8), Out(ctx, 1, M, M, np.float32), c.sums()
        ctx.norm_quant(q, K, sc, *c.rows(s, K))
        far = np.where(top > 1e20, 2.0 ** -64, 1.0)[:, None]
        rq, rs = R.quant_rows((h * far).astype(np.float32) * g)
        np.testing.assert_array_equal(q.get(), rq)
        want = rs.astype(np.float64) / far[:, 0] * c.inv[:, 0]
        assert (np.abs(sc.get()[0] - want) <= Q.NORM_U * want + 2.0 ** -148).all()
        c.check_sum(s)


@pytest.mark.parametrize("K", [5, 250, 1000, 2000, 4100, 20000])
def test_small_gains_leave_large_rows_their_codes(ctx, K):
    """h * gain of ordinary size, with gains next to the smallest normal float: u is that product, to the bit."""
    rng = np.random.default_rng(K)
    M = 6
    x = (rng.standard_normal((M, K)) * np.array([1e37, 1e30, 2.0 ** 70, 1e38 / 8, 1e20, 2.0 ** 66])[:, None]).astype(np.float32)
    g = np.ldexp(rng.uniform(1, 2, K), -125).astype(np.float32)
    for eps in (0.0, 1e-6):
        c = Case(ctx, x, R.F32, None, 0, g, eps)
        c.codes8()
        c.floats(R.F32)


@pytest.mark.parametrize("K", [40, 700, 2000, 20000])
def test_the_largest_eps(ctx, K):
    """mean + eps past the largest float: the root is not."""
    x = np.random.default_rng(K).standard_normal((6, K)).astype(np.float32)
    x *= np.array([1e18, 1e17, 1.0, 0.0, 1e-3, 3e37], np.float32)[:, None] * np.float32(0.2)
    for eps in (np.finfo(np.float32).max, np.float32(1.7e38)):
        c = Case(ctx, x, R.F32, None, 0, None, eps)
        assert (c.y[0] != 0).all()
        c.floats(R.F32)
        c.codes8()


# More rows than the workgroups of one launch take at once, so each goes on to a
# second row or group of rows: lanes of a row 16, 32, 64 (one and two runs), 192, 256
# (one and two), 512, 1024, and rows past those.
@pytest.mark.parametrize("M,K,first", [(32801, 90, 32768), (16391, 250, 16384), (8201, 500, 8192), (8203, 1000, 8192),
                                       (6001, 1025, 2730), (4199, 1541, 2048), (4301, 2049, 2048), (2500, 4099, 1024),
                                       (1101, 8195, 512), (1030, 16385, 512)])
def test_workgroups_of_several_rows(ctx, M, K, first):
    """Rows that are summed again between rows that are not, and the sum in the residual's place."""
    assert M > first
    rng = np.random.default_rng(M + K)
    x, r, g = inputs(M, K, M + K)
    m = np.arange(M)
    kind = rng.integers(0, 8, M)  # most rows are ordinary
    kind[[0, first % M, M - 1]] = 1, 0, 2
    scale = np.select([kind == 1, kind == 2, kind == 3], [1e30, 1e-30, 0.0], 1.0).astype(np.float32)[:, None]
    x, r = x * scale, r * scale
    c = Case(ctx, x, R.F32, r, R.F32, g, 0.0)
    c.codes8()
    c.codes4()
    want = Out(ctx, M, K, K, np.float32)
    ctx.norm_rows(want, R.F32, K, *c.rows())
    c.check_y(want.get(), R.F32)
    # in place
    out = Out(ctx, M, K, K, np.float32)
    ctx.norm_rows(out, R.F32, K, c.dx, R.F32, K, c.dr, R.F32, K, c.dr, K, c.dg, 0.0, M, K)
    np.testing.assert_array_equal(c.dr.download(), c.h)
    np.testing.assert_array_equal(out.get(), want.get())
    assert (want.get()[m[kind == 3]] == 0).all()


@pytest.mark.parametrize("K", [600, 1000, 1024, 2050])
def test_what_of_a_row_does_not_depend_on_the_batch(ctx, K):
    """Sums and 8-bit codes are the same bits in any batch; floats and scales, whose sum may be taken in another
    order (513 to 1024 columns, from 1024 rows on), keep to the same bounds."""
    M = 1100
    x, r, g = inputs(M, K, K)
    seen = []
    for n in (1, 2, 1023, 1024, M):
        c = Case(ctx, x[:n], R.F32, r[:n], R.F32, g)
        q, sc, s = Out(ctx, n, K, K, np.int8), Out(ctx, 1, n, n, np.float32), Out(ctx, n, K, K, np.float32)
        ctx.norm_quant(q, K, sc, *c.rows(s, K))
        c.check_sum(s)
        c.floats(R.F32)
        c.codes4()
        seen.append((q.get(), s.get()))
    for q, s in seen[:-1]:
        np.testing.assert_array_equal(q, seen[-1][0][:len(q)])
        np.testing.assert_array_equal(s, seen[-1][1][:len(s)])


def test_norm_then_products_in_a_graph(gpu_ctx_factory):
    """The run of them together: residual and norm, a product in 8 bits, a norm, a product in 4, captured and replayed."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    rng = np.random.default_rng(4)
    M, K, N = 70, 320, 96
    w1, s1 = c.to_device(rng.integers(-127, 128, (K, K)).astype(np.int8)), c.to_device(np.full(K, 1e-3, np.float32))
    wf = rng.standard_normal((N, K)).astype(np.float32)
    wc, wsc = Q.mx4_quant(wf)
    w2, s2 = c.to_device(Q.mx4_pack(wc)), c.to_device(wsc)
    g = c.to_device((1 + 0.1 * rng.standard_normal(K)).astype(np.float32))
    x, res = c.to_device(np.zeros((M, K), np.float32)), c.to_device(np.zeros((M, K), np.float32))
    start = c.to_device(np.zeros((M, K), np.float32))
    q, sc, h = c.empty((M, K), np.int8), c.empty(M), c.empty((M, K))
    q4, sc4, out = c.empty((M, K // 2), np.uint8), c.empty((M, K // 32), np.uint8), c.empty((M, N))

    def call():
        # the residual is added to in place: it starts from `start`
        c.norm_quant(q, K, sc, x, R.F32, K, start, R.F32, K, res, K, g, 1e-6, M, K)
        c.i8_matmul(h, R.F32, K, q, K, sc, w1, K, s1, None, R.RELU, M, K, K)
        c.norm_mx4(q4, K // 2, sc4, K // 32, h, R.F32, K, res, R.F32, K, res, K, g, 1e-6, M, K)
        c.mx4_matmul(out, R.F32, N, q4, K // 2, sc4, K // 32, w2, K // 2, s2, K // 32, None, R.NONE, M, N, K)

    graph = Captured(c, call)  # none of them takes scratch at these sizes, so none has to run before
    for seed in range(4):
        r = np.random.default_rng(seed)
        x.upload(r.standard_normal((M, K)).astype(np.float32))
        start.upload(r.standard_normal((M, K)).astype(np.float32))
        out.fill(0xFF)
        graph.replay()
        c.synchronize()
        got, gres = out.download(), res.download()
        call()
        c.synchronize()
        np.testing.assert_array_equal(got, out.download())
        np.testing.assert_array_equal(gres, res.download())
        # each call against its definition on what the call before it gave
        hq, _, _, _ = Q.norm(x.download(), start.download(), g.download(), 1e-6)
        np.testing.assert_array_equal(res.download(), hq + h.download())
        y = Q.mx4_values(Q.mx4_unpack(q4.download(), K), sc4.download())
        ref, d = Q.mx4_product(y, Q.mx4_values(wc, wsc), None, R.NONE)
        check(got, R.F32, ref, d)
    graph.close()


def test_refusals(ctx):
    f, q = ctx.empty(4096, np.float32), ctx.empty(4096, np.int8)
    odd = View(f, 2)
    INV, UNS = _lib.E_INVALID, _lib.E_UNSUPPORTED
    rows = dict(d_x=f, x_elem=0, ldx=40, d_res=f, res_elem=0, ldr=40, d_sum=f, ldsum=40, d_gain=f, eps=1e-6, rows=2,
                cols=40)
    wrong = [dict(x_elem=3), dict(x_elem=-1), dict(ldx=39), dict(res_elem=3), dict(ldr=39), dict(ldsum=39), dict(eps=-1.0),
             dict(eps=float("nan")), dict(eps=float("inf")), dict(rows=-1), dict(cols=0), dict(cols=-1), dict(d_x=Null),
             dict(d_x=odd), dict(d_res=odd), dict(d_gain=odd), dict(d_sum=odd), dict(d_res=None),
             dict(d_sum=f, ldsum=41)]
    for fn, out in ((ctx.norm_rows, dict(d_y=f, y_elem=0, ldy=40)), (ctx.norm_quant, dict(d_q=q, ldq=40, d_scale=f)),
                    (ctx.norm_mx4, dict(d_q=q, ldq=20, d_s=q, lds=2))):
        for bad in wrong:
            refused(INV, fn, **{**out, **rows, **bad})
        refused(UNS, fn, **{**out, **rows, "rows": 1 << 31})
    for bad in [dict(y_elem=3), dict(ldy=39), dict(d_y=Null), dict(d_y=odd)]:
        refused(INV, ctx.norm_rows, **{**dict(d_y=f, y_elem=0, ldy=40), **rows, **bad})
    for bad in [dict(ldq=39), dict(d_q=Null), dict(d_scale=Null), dict(d_scale=odd)]:
        refused(INV, ctx.norm_quant, **{**dict(d_q=q, ldq=40, d_scale=f), **rows, **bad})
    for bad in [dict(ldq=19), dict(lds=1), dict(d_q=Null), dict(d_s=Null)]:
        refused(INV, ctx.norm_mx4, **{**dict(d_q=q, ldq=20, d_s=q, lds=2), **rows, **bad})
    ctx.norm_rows(Null, 0, 40, Null, 0, 40, None, 0, 0, None, 0, None, 1e-6, 0, 40)
