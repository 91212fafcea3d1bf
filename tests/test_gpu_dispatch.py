"""Rows to the order of their experts and back, and the gradients of both, against
their definitions in 64 bits."""
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


def choose(rng, M, k, E):
    """Experts of each row: some rows without any, some slots without one or with one that is not there, some twice."""
    idx = rng.integers(0, E, (M, k)).astype(np.int32) if rng.random() < 0.5 or k > E else \
        np.argsort(rng.random((M, E)), axis=1)[:, :k].astype(np.int32)
    if M > 3:
        idx[1] = -1
        idx[2, k // 2:] = -1
        idx[3, 0] = E
        idx[M - 1, k - 1] = 2 ** 31 - 1
        idx[rng.random((M, k)) < 0.05] = -5
    return idx


def values(rng, rows, cols, elem):
    bits = R.to_bits(rng.standard_normal((rows, cols)).astype(np.float32), elem)
    return bits, R.from_bits(bits, elem)


def run_dispatch(ctx, idx, E, bits, elem, pad=0):
    """(rows used, place, start); rows past the last pair must stay as they were."""
    (M, k), D = idx.shape, bits.shape[1]
    z, place = Out(ctx, M * k, D, D + pad, R.np_type(elem)), Out(ctx, M, k, k, np.int32)
    start = Out(ctx, 1, E + 1, E + 1, np.int32)
    ctx.dispatch(z, D + pad, place, start, ctx.to_device(strided(bits, D + pad + 1)), elem, D + pad + 1,
                 ctx.to_device(idx), M, k, E, D)
    got, n = z.get(), start.get()[0]
    left = np.ascontiguousarray(got[n[-1]:]).view(np.uint8)
    assert (left == 0x5A).all()
    return got[:n[-1]], place.get(), n


SIZES = [  # M, k, E, D
    (1, 1, 1, 1), (1, 6, 64, 128), (2, 3, 4, 33), (5, 64, 1024, 7), (40, 8, 8, 130), (257, 2, 8, 512), (300, 1, 100, 64),
    (1000, 4, 60, 96), (700, 3, 1000, 40), (3000, 8, 64, 257), (9001, 2, 256, 33), (70000, 1, 16, 8), (20000, 6, 1024, 16),
    (128, 16, 16, 1000), (129, 16, 17, 1001), (4, 2, 3, 20000), (512, 4, 7, 24), (2048, 1, 2, 10), (2049, 1, 2, 10),
    (256, 4, 5, 12), (205, 5, 1024, 4), (4096, 1, 9, 2), (4097, 1, 9, 2), (1366, 3, 1024, 2), (262200, 4, 5, 2),
    (16, 64, 60, 40), (2, 64, 60, 40), (128, 8, 60, 9), (128, 8, 1024, 9), (3, 2, 4, 4099), (200, 3, 8, 2051),
    (2050, 1, 8, 2051), (2100, 3, 8, 700), (2048, 8, 9, 1024), (2049, 8, 9, 1025),
    (16384, 1, 5, 2), (16385, 1, 1024, 2)]


@pytest.mark.parametrize("M,k,E,D", SIZES)
@pytest.mark.parametrize("elem,pad", [(R.F32, 0), (R.BF16, 3), (R.F16, 8)])
def test_dispatch(ctx, M, k, E, D, elem, pad):
    rng = np.random.default_rng(M * 7 + k + E)
    idx = choose(rng, M, k, E)
    bits, _ = values(rng, M, D, elem)
    z, place, start = run_dispatch(ctx, idx, E, bits, elem, pad)
    rp, rs = Q.places(idx, E)
    np.testing.assert_array_equal(start, rs)
    np.testing.assert_array_equal(place, rp)
    m, j = np.nonzero(rp >= 0)
    want = np.empty((rs[-1], D), bits.dtype)
    want[rp[m, j]] = bits[m]
    np.testing.assert_array_equal(z, want)


@pytest.mark.parametrize("E", [1, 2, 3, 4, 5, 255, 256, 257, 1021, 1022, 1023, 1024])
def test_starts_of_few_pairs(ctx, E):
    """The starts in one launch with the rows, four experts a thread: any number of experts, and none past them written."""
    rng = np.random.default_rng(E)
    for M, k in ((1, 1), (3, 5), (200, 3), (1024, 1)):
        idx = choose(rng, M, k, E)
        idx[0, 0] = E - 1  # the last expert has a pair
        bits = np.zeros((M, 4), np.float32)
        _, place, start = run_dispatch(ctx, idx, E, bits, R.F32)
        rp, rs = Q.places(idx, E)
        np.testing.assert_array_equal(start, rs)
        np.testing.assert_array_equal(place, rp)


def test_dispatch_keeps_the_order_of_one_expert(ctx):
    """All on one expert, all on none, and the same experts over and over: places are in the pairs' order."""
    for M, k, E in ((5000, 2, 40), (300, 3, 40)):
        bits = np.zeros((M, 4), np.float32)
        for idx in (np.full((M, k), E - 1, np.int32), np.full((M, k), -1, np.int32),
                    np.broadcast_to(np.arange(k, dtype=np.int32), (M, k)).copy()):
            z, place, start = run_dispatch(ctx, idx, E, bits, R.F32)
            rp, rs = Q.places(idx, E)
            np.testing.assert_array_equal(place, rp)
            np.testing.assert_array_equal(start, rs)


def test_dispatch_of_nothing(ctx):
    start = ctx.empty(8, np.int32).fill(0xFF)
    ctx.dispatch(Null, 8, Null, start, Null, R.F32, 8, Null, 0, 2, 7, 8)
    assert (start.download() == 0).all()
    # rows without columns have places all the same
    idx = np.array([[2, 0], [0, 2]], np.int32)
    place = ctx.empty((2, 2), np.int32)
    ctx.dispatch(Null, 0, place, start, Null, R.F32, 0, ctx.to_device(idx), 2, 2, 7, 0)
    np.testing.assert_array_equal(place.download(), [[2, 0], [1, 3]])
    np.testing.assert_array_equal(start.download(), [0, 2, 2, 4, 4, 4, 4, 4])
    ctx.dispatch(Null, 0, place.fill(0xFF), None, Null, R.F32, 0, ctx.to_device(idx), 2, 2, 7, 0)
    np.testing.assert_array_equal(place.download(), [[2, 0], [1, 3]])


@pytest.mark.parametrize("M,k,E,N", SIZES)
@pytest.mark.parametrize("z_elem,out_elem,weighted,pad", [(R.F32, R.F32, True, 0), (R.BF16, R.BF16, True, 3),
                                                          (R.F16, R.F32, False, 8), (R.BF16, R.F16, True, 0)])
def test_combine(ctx, M, k, E, N, z_elem, out_elem, weighted, pad):
    rng = np.random.default_rng(M * 7 + k + E)
    place = Q.places(choose(rng, M, k, E), E)[0]
    bits, z = values(rng, M * k, N, z_elem)
    wt = rng.standard_normal((M, k)).astype(np.float32)
    wt[place < 0] = np.nan  # not read
    out = Out(ctx, M, N, N + pad, R.np_type(out_elem))
    ctx.combine(out, out_elem, N + pad, ctx.to_device(strided(bits, N + pad)), z_elem, N + pad, ctx.to_device(place),
                ctx.to_device(wt) if weighted else None, M, k, N)
    check(out.get(), out_elem, *Q.combine(z, place, wt if weighted else None))


@pytest.mark.parametrize("M,k,E,N", SIZES)
@pytest.mark.parametrize("z_elem,out_elem,weighted,pad", [(R.F32, R.F32, True, 0), (R.BF16, R.BF16, True, 3),
                                                          (R.F16, R.F32, False, 8), (R.BF16, R.F16, True, 0),
                                                          (R.F32, R.BF16, True, 1)])
def test_gradients(ctx, M, k, E, N, z_elem, out_elem, weighted, pad):
    rng = np.random.default_rng(M * 7 + k + E)
    place = Q.places(choose(rng, M, k, E), E)[0]
    bits, z = values(rng, M * k, N, z_elem)
    dbits, d = values(rng, M, N, out_elem)
    wt = rng.standard_normal((M, k)).astype(np.float32)
    wt[place < 0] = np.nan
    dp, dw_in = ctx.to_device(place), ctx.to_device(wt) if weighted else None
    dz, dw = Out(ctx, M * k, N, N + pad, R.np_type(z_elem)), Out(ctx, M, k, k, np.float32)
    ctx.combine_grad(dz, N + pad, dw, ctx.to_device(strided(bits, N + pad)), z_elem, N + pad,
                     ctx.to_device(strided(dbits, N + pad)), out_elem, N + pad, dp, dw_in, M, k, N)
    rz, rw, bw = Q.combine_grad(z, place, wt if weighted else None, d)
    used = (place >= 0).sum()
    got = dz.get()
    assert (np.ascontiguousarray(got[used:]).view(np.uint8) == 0x5A).all()
    check(got[:used], z_elem, rz[:used], R.U * np.abs(rz[:used]) + 2.0 ** -148)
    check(dw.get(), R.F32, rw, bw)
    # each of the two alone
    alone = Out(ctx, M * k, N, N + pad, R.np_type(z_elem))
    ctx.combine_grad(alone, N + pad, None, None, z_elem, 0, ctx.to_device(strided(dbits, N + pad)), out_elem, N + pad,
                     dp, dw_in, M, k, N)
    np.testing.assert_array_equal(alone.get(), got)
    again = Out(ctx, M, k, k, np.float32)
    ctx.combine_grad(None, 0, again, ctx.to_device(strided(bits, N + pad)), z_elem, N + pad,
                     ctx.to_device(strided(dbits, N + pad)), out_elem, N + pad, dp, dw_in, M, k, N)
    np.testing.assert_array_equal(again.get(), dw.get())
    # dispatch's: the same sum without weights
    dx = Out(ctx, M, N, N + pad, R.np_type(z_elem))
    ctx.dispatch_grad(dx, z_elem, N + pad, ctx.to_device(strided(bits, N + pad)), N + pad, dp, M, k, N)
    check(dx.get(), z_elem, *Q.combine(z, place, None))


def test_gradients_against_differences(ctx):
    """<dout, f(v + t)> - <dout, f(v)> is the gradient's product with t: each map is linear in each of its inputs."""
    rng = np.random.default_rng(9)
    M, k, E, N = 60, 4, 9, 130
    idx = choose(rng, M, k, E)
    place = Q.places(idx, E)[0]
    dp, z = ctx.to_device(place), rng.standard_normal((M * k, N)).astype(np.float32)
    wt, dout = rng.standard_normal((M, k)).astype(np.float32), rng.standard_normal((M, N)).astype(np.float32)

    def f(z, wt):
        out = ctx.empty((M, N))
        ctx.combine(out, R.F32, N, ctx.to_device(z), R.F32, N, dp, ctx.to_device(wt), M, k, N)
        return (out.download().astype(np.float64) * dout).sum()

    def err(z, wt):  # of f: the bound of its outputs, and their rounding
        y, b = Q.combine(z, place, wt)
        return ((b + R.U * np.abs(y)) * np.abs(dout)).sum()

    dz, dw = ctx.empty((M * k, N)).fill(0), ctx.empty((M, k))
    ctx.combine_grad(dz, N, dw, ctx.to_device(z), R.F32, N, ctx.to_device(dout), R.F32, N, dp, ctx.to_device(wt), M, k,
                     N)
    dz, dw = dz.download().astype(np.float64), dw.download().astype(np.float64)
    for t in range(4):
        v = rng.standard_normal((M * k, N)).astype(np.float32)
        z2 = z + v
        step = z2.astype(np.float64) - z
        want = (dz * step).sum()
        tol = err(z, wt) + err(z2, wt) + 3 * R.U * np.abs(dz * step).sum()
        assert abs(f(z2, wt) - f(z, wt) - want) <= tol
        u = rng.standard_normal((M, k)).astype(np.float32)
        w2 = wt + u
        step = w2.astype(np.float64) - wt
        bound = Q.combine_grad(z, place, wt, dout)[2]
        tol = err(z, wt) + err(z, w2) + (bound * np.abs(step)).sum()
        assert abs(f(z, w2) - f(z, wt) - (dw * step).sum()) <= tol
    # dispatch: <dz, dispatch(x)> = <dispatch_grad(dz), x>
    x, d = rng.standard_normal((M, N)).astype(np.float32), rng.standard_normal((M * k, N)).astype(np.float32)
    rows, _, start = run_dispatch(ctx, idx, E, x, R.F32)
    dx = ctx.empty((M, N))
    ctx.dispatch_grad(dx, R.F32, N, ctx.to_device(d), N, dp, M, k, N)
    ref, bound = Q.combine(d, place, None)
    left = (rows.astype(np.float64) * d[:start[-1]]).sum()
    assert abs(left - (dx.download().astype(np.float64) * x).sum()) <= ((bound + R.U * np.abs(ref)) * np.abs(x)).sum()


def test_places_outside_the_rows_are_skipped(ctx):
    M, k, N = 3, 2, 16
    z, w = np.ones((M * k, N), np.float32), np.ones((M, k), np.float32)
    place = np.array([[0, 6], [-1, 2 ** 31 - 1], [5, -7]], np.int32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.combine(out, R.F32, N, ctx.to_device(z), R.F32, N, ctx.to_device(place), ctx.to_device(w), M, k, N)
    np.testing.assert_array_equal(out.get()[:, 0], [1, 0, 1])
    dz, dw = Out(ctx, M * k, N, N, np.float32), Out(ctx, M, k, k, np.float32)
    ctx.combine_grad(dz, N, dw, ctx.to_device(z), R.F32, N, ctx.to_device(np.ones((M, N), np.float32)), R.F32, N,
                     ctx.to_device(place), ctx.to_device(w), M, k, N)
    np.testing.assert_array_equal(dw.get(), [[N, 0], [0, 0], [N, 0]])
    got = dz.get()
    assert (got[[0, 5]] == 1).all() and (np.ascontiguousarray(got[1:5]).view(np.uint8) == 0x5A).all()


def test_past_32_bit_offsets(ctx):
    """Sorted rows 4.9 GB apart from first to last, there and back."""
    M, k, E, D, ld = 1024, 4, 8, 40, 600000
    rng = np.random.default_rng(5)
    idx = choose(rng, M, k, E)
    bits, x = values(rng, M, D, R.BF16)
    z, place = ctx.empty(M * k * ld, np.uint16), ctx.empty((M, k), np.int32)
    ctx.dispatch(z, ld, place, None, ctx.to_device(bits), R.BF16, D, ctx.to_device(idx), M, k, E, D)
    rp = Q.places(idx, E)[0]
    np.testing.assert_array_equal(place.download(), rp)
    out = ctx.empty((M, D))
    ctx.combine(out, R.F32, D, z, R.BF16, ld, place, None, M, k, D)
    np.testing.assert_array_equal(out.download(), x * (rp >= 0).sum(axis=1)[:, None])  # up to four of the same: exact
    dw = ctx.empty((M, k))
    d = ctx.to_device(bits)
    ctx.combine_grad(z, ld, None, None, R.BF16, 0, d, R.BF16, D, place, None, M, k, D)
    ctx.combine_grad(None, 0, dw, z, R.BF16, ld, d, R.BF16, D, place, None, M, k, D)
    y = (x.astype(np.float64) ** 2).sum(axis=1)[:, None] * (rp >= 0)
    assert (np.abs(dw.download() - y) <= (8 + 12) * R.U * y * 1.01 + R.U * y).all()
    z.free()


def test_not_finite_values_pass_where_they_belong(ctx):
    rng = np.random.default_rng(3)
    M, k, E, N = 50, 3, 6, 40
    place = Q.places(np.argsort(rng.random((M, E)), axis=1)[:, :k].astype(np.int32), E)[0]
    z = rng.standard_normal((M * k, N)).astype(np.float32)
    z[place[7, 1], 3], z[place[9, 0]] = np.nan, np.inf
    wt = rng.random((M, k)).astype(np.float32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.combine(out, R.F32, N, ctx.to_device(z), R.F32, N, ctx.to_device(place), ctx.to_device(wt), M, k, N)
    got = out.get()
    assert np.isnan(got[7, 3]) and np.isinf(got[9]).all() and (~np.isfinite(got)).sum() == N + 1


@pytest.mark.parametrize("elem", [R.F32, R.BF16])
@pytest.mark.parametrize("N", [300, 1000, 1100])
def test_what_of_a_row_does_not_depend_on_the_batch(ctx, N, elem):
    """Sums over slots and dz are the same bits in any batch; the weights' gradients, summed over columns by a wave from
    2048 rows on and by a workgroup below, keep to the same bound."""
    rng = np.random.default_rng(N)
    M, k, few = 2300, 3, 7
    place = np.concatenate([rng.permutation(few * k), few * k + rng.permutation((M - few) * k)]).astype(np.int32)
    place = place.reshape(M, k)  # the first rows' pairs are the first rows of z in every batch
    (bits, z), (dbits, d) = values(rng, M * k, N, elem), values(rng, M, N, elem)
    wt = rng.standard_normal((M, k)).astype(np.float32)
    dev = [ctx.to_device(a) for a in (bits, dbits, wt)]
    seen = []
    for n in (few, 2047, 2048, M):
        p = place[:n].copy()
        p[few:] = np.where(p[few:] < n * k, p[few:], -1)
        dp = ctx.to_device(p)
        outs = [Out(ctx, n, N, N, R.np_type(elem)), Out(ctx, n, N, N, R.np_type(elem)),
                Out(ctx, n * k, N, N, R.np_type(elem)), Out(ctx, n, k, k, np.float32)]
        ctx.combine(outs[0], elem, N, dev[0], elem, N, dp, dev[2], n, k, N)
        ctx.dispatch_grad(outs[1], elem, N, dev[0], N, dp, n, k, N)
        ctx.combine_grad(outs[2], N, outs[3], dev[0], elem, N, dev[1], elem, N, dp, dev[2], n, k, N)
        check(outs[3].get(), R.F32, *Q.combine_grad(z[:n * k], p, wt[:n], d[:n])[1:])
        seen.append([outs[0].get()[:few], outs[1].get()[:few], outs[2].get()[:few * k]])
    for other in seen[:-1]:
        for a, b in zip(other, seen[-1]):
            np.testing.assert_array_equal(a, b)


def test_route_dispatch_products_combine(gpu_ctx_factory):
    """The run of them together: route, rows by expert, a 4-bit product for each expert, and back; then replayed from a
    graph, where the products take all the rows (their starts are the device's)."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    rng = np.random.default_rng(11)
    M, k, E, D, N = 200, 2, 5, 96, 64
    logits, x = c.to_device(rng.standard_normal((M, E)).astype(np.float32)), c.to_device(np.zeros((M, D), np.float32))
    wf = rng.standard_normal((E * N, D)).astype(np.float32)
    wc, ws = Q.mx4_quant(wf)
    dw, dws = c.to_device(Q.mx4_pack(wc)), c.to_device(ws)
    idx, wt, place = c.empty((M, k), np.int32), c.empty((M, k)), c.empty((M, k), np.int32)
    start, rows, z = c.empty(E + 1, np.int32), c.empty((M * k, D)), c.empty((M * k, N))
    out = c.empty((M, N))

    def front():
        c.route(idx, wt, None, logits, R.F32, E, None, None, M, E, k, renorm=True)
        c.dispatch(rows, D, place, start, x, R.F32, D, idx, M, k, E, D)

    def expert(e, r0, n):
        at = lambda a, b: View(a, int(b))  # noqa: E731
        c.mx4_linear(at(z, r0 * N * 4), R.F32, N, at(rows, r0 * D * 4), R.F32, D, at(dw, e * N * D // 2), D // 2,
                     at(dws, e * N * D // 32), D // 32, None, R.NONE, n, N, D)

    def whole():
        front()
        s = start.download().tolist()
        for e in range(E):
            expert(e, s[e], s[e + 1] - s[e])
        c.combine(out, R.F32, N, z, R.F32, N, place, wt, M, k, N)

    rows.fill(0)
    x.upload(rng.standard_normal((M, D)).astype(np.float32))
    whole()
    c.synchronize()
    xv = Q.mx4_values(*Q.mx4_quant(x.download()))
    wv = Q.mx4_values(wc, ws).reshape(E, N, D)
    gi, gw = idx.download(), wt.download()
    y, d = np.zeros((M, N)), np.zeros((M, N))
    for j in range(k):
        for m in range(M):
            v, b = Q.mx4_product(xv[m:m + 1], wv[gi[m, j]], None, R.NONE)
            t = gw[m, j].astype(np.float64)
            y[m] += t * v[0]
            d[m] += np.abs(t) * (b[0] + R.U * np.abs(v[0])) + (k + 1) * R.U * 1.01 * np.abs(t * v[0])
    check(out.download(), R.F32, y, d)

    # the sort and the sum in a graph, beside a product of all sorted rows by one expert
    def captured():
        front()
        expert(2, 0, M * k)
        c.combine(out, R.F32, N, z, R.F32, N, place, wt, M, k, N)

    captured()
    c.synchronize()
    g = Captured(c, captured)
    for seed in range(4):
        r = np.random.default_rng(seed)
        x.upload(r.standard_normal((M, D)).astype(np.float32))
        logits.upload(r.standard_normal((M, E)).astype(np.float32))
        out.fill(0xFF)
        g.replay()
        c.synchronize()
        got, gp = out.download(), place.download()
        np.testing.assert_array_equal(gp, Q.places(idx.download(), E)[0])
        captured()
        c.synchronize()
        np.testing.assert_array_equal(got, out.download())
        assert np.isfinite(got).all()
    g.close()


def test_large_sort_in_a_graph(gpu_ctx_factory):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    M, k, E, D = 9000, 3, 50, 8
    x = np.random.default_rng(0).standard_normal((M, D)).astype(np.float32)
    dx, idx, place, start = c.to_device(x), c.empty((M, k), np.int32), c.empty((M, k), np.int32), c.empty(E + 1, np.int32)
    z = c.empty((M * k, D))
    idx.fill(0)
    seen = []

    def call():
        c.dispatch(z, D, place, start, dx, R.F32, D, idx, M, k, E, D)

    def refused_call():
        with pytest.raises(vdttfs.VdttfsError) as e:
            call()
        seen.append(e.value.code)
        c.norm_rows(z, R.F32, D, dx, R.F32, D, None, 0, 0, None, 0, None, 0.0, M, D)  # the capture goes on

    Captured(c, refused_call).close()
    assert seen == [_lib.E_UNSUPPORTED]
    call()
    c.synchronize()
    g = Captured(c, call)
    for seed in range(4):
        i = np.random.default_rng(seed).integers(-1, E, (M, k)).astype(np.int32)
        idx.upload(i)
        place.fill(0x11)
        start.fill(0x11)
        g.replay()
        c.synchronize()
        rp, rs = Q.places(i, E)
        np.testing.assert_array_equal(place.download(), rp)
        np.testing.assert_array_equal(start.download(), rs)
        call()
        c.synchronize()
        np.testing.assert_array_equal(place.download(), rp)
    g.close()


@pytest.mark.parametrize("M,k,E,D", [(1, 6, 64, 1024), (100, 8, 16, 130), (1200, 3, 9, 77)])
def test_a_training_step_in_a_graph(gpu_ctx_factory, M, k, E, D):
    """There, back and both gradients, replayed between eager calls of the same."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    x, idx, wt, dout = (c.empty(s, t) for s, t in (((M, D), np.float32), ((M, k), np.int32), ((M, k), np.float32),
                                                   ((M, D), np.float32)))
    z, place, start = c.empty((M * k, D)), c.empty((M, k), np.int32), c.empty(E + 1, np.int32)
    out, dz, dw, dx = c.empty((M, D)), c.empty((M * k, D)), c.empty((M, k)), c.empty((M, D))
    results = (z, place, start, out, dz, dw, dx)

    def call():
        c.dispatch(z, D, place, start, x, R.F32, D, idx, M, k, E, D)
        c.combine(out, R.F32, D, z, R.F32, D, place, wt, M, k, D)
        c.combine_grad(dz, D, dw, z, R.F32, D, dout, R.F32, D, place, wt, M, k, D)
        c.dispatch_grad(dx, R.F32, D, dz, D, place, M, k, D)

    idx.fill(0)
    call()
    c.synchronize()
    g = Captured(c, call)
    for seed in range(4):
        rng = np.random.default_rng(seed)
        i = rng.integers(-1, E, (M, k)).astype(np.int32)
        idx.upload(i)
        for a in (x, wt, dout):
            a.upload(rng.standard_normal(a.shape).astype(np.float32))
        seen = []
        for run in (g.replay, call, g.replay):
            for r in results:
                r.fill(0)
            c.synchronize()
            run()
            c.synchronize()
            seen.append([r.download() for r in results])
        for a, b in zip(seen[0] + seen[2], seen[1] + seen[1]):
            np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(seen[0][1], Q.places(i, E)[0])
    g.close()


def test_refusals(ctx):
    f, i = ctx.empty(4096, np.float32), ctx.empty(4096, np.int32)
    odd, INV, UNS = View(f, 2), _lib.E_INVALID, _lib.E_UNSUPPORTED
    d = dict(d_z=f, ldz=8, d_place=i, d_start=i, d_x=f, elem=0, ldx=8, d_idx=i, M=2, top_k=2, n_experts=4, cols=8)
    for bad in [dict(ldz=7), dict(ldx=7), dict(elem=3), dict(elem=-1), dict(M=-1), dict(top_k=0), dict(n_experts=0),
                dict(cols=-1), dict(d_z=Null), dict(d_place=Null), dict(d_x=Null), dict(d_idx=Null), dict(d_z=odd),
                dict(d_place=odd), dict(d_start=odd), dict(d_idx=odd), dict(d_x=odd)]:
        refused(INV, ctx.dispatch, **{**d, **bad})
    for bad in [dict(n_experts=1025), dict(top_k=65), dict(M=1 << 30)]:
        refused(UNS, ctx.dispatch, **{**d, **bad})
    c = dict(d_out=f, out_elem=0, ldo=8, d_z=f, z_elem=0, ldz=8, d_place=i, d_weight=f, M=2, top_k=2, cols=8)
    for bad in [dict(ldz=7), dict(ldo=7), dict(out_elem=3), dict(z_elem=3), dict(M=-1), dict(top_k=0), dict(cols=-1),
                dict(d_out=Null), dict(d_z=Null), dict(d_place=Null), dict(d_weight=odd), dict(d_out=odd)]:
        refused(INV, ctx.combine, **{**c, **bad})
    for bad in [dict(top_k=65), dict(M=1 << 30)]:
        refused(UNS, ctx.combine, **{**c, **bad})
    g = dict(d_dx=f, elem=0, lddx=8, d_dz=f, lddz=8, d_place=i, M=2, top_k=2, cols=8)
    for bad in [dict(lddx=7), dict(lddz=7), dict(elem=3), dict(M=-1), dict(d_dx=Null), dict(d_dz=Null),
                dict(d_place=Null), dict(d_dz=odd)]:
        refused(INV, ctx.dispatch_grad, **{**g, **bad})
    h = dict(d_dz=f, lddz=8, d_dw=f, d_z=f, z_elem=0, ldz=8, d_dout=f, out_elem=0, lddo=8, d_place=i, d_weight=f, M=2,
             top_k=2, cols=8)
    for bad in [dict(lddz=7), dict(ldz=7), dict(lddo=7), dict(z_elem=3), dict(out_elem=3), dict(M=-1), dict(top_k=0),
                dict(d_dz=None, d_dw=None), dict(d_z=None), dict(d_dout=Null), dict(d_place=Null), dict(d_dz=odd),
                dict(d_dw=odd), dict(d_weight=odd)]:
        refused(INV, ctx.combine_grad, **{**h, **bad})
    ctx.combine(Null, 0, 8, Null, 0, 8, Null, None, 0, 2, 8)
    ctx.dispatch_grad(Null, 0, 8, Null, 8, Null, 0, 2, 8)
    ctx.combine_grad(f, 8, f, Null, 0, 8, Null, 0, 8, Null, None, 0, 2, 8)
