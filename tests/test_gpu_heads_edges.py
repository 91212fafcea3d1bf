"""The 8-bit heads where they went, or could go, wrong: rounding that depends on
the batch, choices between infinite values, scores and activations far from zero,
sizes at the ends of their types, empty widths, graphs on other streams."""
import ctypes

import numpy as np
import pytest

import headref as R
import vdttfs
from vdttfs import _lib
from test_gpu_heads import (Out, View, check, codes, ctx, expert_case, refused, run_experts,  # noqa: F401
                            run_route)
from test_gpu_heads_paths import tile_rows
from test_gpu_scratch import Captured

pytestmark = pytest.mark.gpu
FLT_MAX = np.finfo(np.float32).max


# ---- slots of a 16-bit output are summed in 32 bits ----------------------------------
@pytest.mark.parametrize("out_elem", [R.BF16, R.F16])
def test_slots_of_a_large_batch_cancel(ctx, out_elem):
    """Both slots of a row name one expert, and their weights differ by 2^-8: the
    sum is exact to the roundings of 32 bits, whatever the batch."""
    M, E, D, F, N = 8300, 8, 64, 64, 520
    assert M * 2 * N * 4 > 32 << 20
    rng = np.random.default_rng(11)
    weights = expert_case(rng, E, D, F, N, False, True)
    idx = np.repeat(rng.integers(0, E, (M, 1)), 2, axis=1).astype(np.int32)
    wt = np.repeat((0.5 + rng.random((M, 1))).astype(np.float32), 2, axis=1)
    wt[:, 1] *= -np.float32(1 - 2.0 ** -8)
    bits = R.to_bits(rng.standard_normal((M, D)).astype(np.float32), out_elem)
    got = run_experts(ctx, bits, out_elem, D, idx, wt, weights, R.RELU, False, out_elem)
    at = np.unique(np.concatenate([[0, 1, M - 1], rng.integers(0, M, 200)]))
    q, s = R.quant_rows(R.from_bits(bits[at], out_elem))
    y, d, _ = R.experts(q, s, idx[at], wt[at], *weights, R.RELU, False)
    check(got[at], out_elem, y, d)


@pytest.mark.parametrize("elem", [R.BF16, R.F16])
def test_expert_rows_do_not_depend_on_the_batch(ctx, elem):
    """16-bit rows alone, in a small batch and in one of more than 32 MB of slots: the same bits."""
    M, k, E, D, F, N = 2100, 8, 12, 96, 64, 520
    assert M * k * N * 4 > 32 << 20
    rng = np.random.default_rng(12)
    weights = expert_case(rng, E, D, F, N, True, True)
    bits = R.to_bits(rng.standard_normal((M, D)).astype(np.float32), elem)
    idx = np.argsort(rng.random((M, E)), axis=1)[:, :k].astype(np.int32)
    wt = rng.random((M, k)).astype(np.float32)
    large = run_experts(ctx, bits, elem, D, idx, wt, weights, R.SILU, True, elem)
    for n in (1, 5, 60, 400):
        some = run_experts(ctx, bits[:n], elem, D, idx[:n], wt[:n], weights, R.SILU, True, elem)
        np.testing.assert_array_equal(some, large[:n])


# ---- choices between infinite values -------------------------------------------------
def routed(ctx, l, bias, k, score, groups, top_groups, group_top):
    """The choice, checked against the definition; every row of it is told apart or equal."""
    args = (k, score, groups, top_groups, group_top, False, 1.0)
    gi, gw = run_route(ctx, l, R.F32, bias, None, *args)
    ri, rw, decided = R.route(l, bias, None, *args)
    assert decided.all()
    np.testing.assert_array_equal(gi, ri)
    assert (np.abs(gw - rw) <= R.route_bound(l.shape[1]) * rw + 1e-37).all()
    return gi


# experts, slots: the second takes another kernel (more than 256 experts or 8 slots)
KERNELS = [(64, 4), (320, 4), (64, 10)]


@pytest.mark.parametrize("E,k", KERNELS)
@pytest.mark.parametrize("groups", [8, 16])
@pytest.mark.parametrize("top_groups,group_top", [(1, 1), (1, 2), (2, 2), (3, 1)])
def test_groups_of_infinite_value(ctx, E, k, groups, top_groups, group_top):
    """A bias of +inf in one to four groups: the first of them are kept, and no others."""
    per = E // groups
    l = np.tile(np.linspace(-1, 1, E, dtype=np.float32)[::-1], (3, 1))
    for infinite in ([4], [0, 4], [2, 4], [1, 5], [3, 7], [0, 1, 4], [1, 3, 5, 7], [6, 2, 4]):
        bias = np.zeros(E, np.float32)
        for g in infinite:
            bias[g * per + per // 2] = np.inf
        gi = routed(ctx, l, bias, k, 1, groups, top_groups, group_top)
        kept = set(gi[0][gi[0] >= 0] // per)
        assert len(kept) <= top_groups and sorted(infinite)[0] in kept


@pytest.mark.parametrize("E,k", KERNELS)
def test_sums_of_a_group_past_the_largest_float(ctx, E, k):
    """Groups whose best two sum past the largest float, above and below, are still ordered by their sums."""
    per = E // 8
    l = np.zeros((2, E), np.float32)
    big = lambda v: np.float32(v) * FLT_MAX  # noqa: E731
    bias = np.zeros(E, np.float32)
    for g, v in enumerate((0.6, 0.9, 0.7, 1.0, 0.8, 0.3, 0.55, 1.0)):
        bias[g * per:(g + 1) * per] = big(v)
    for top in (1, 2, 3):
        gi = routed(ctx, l, bias, k, 1, 8, top, 2)
        assert set(gi[0][gi[0] >= 0] // per) <= set([3, 7, 1][:top])
    # masked by the lowest value, not by -inf: these experts can be chosen, those of a group of -inf cannot
    bias[:] = -np.inf
    bias[5 * per:6 * per] = -FLT_MAX
    bias[6 * per:7 * per] = -0.75 * FLT_MAX
    for top in (1, 2):
        gi = routed(ctx, l, bias, k, 1, 8, top, 2)
        assert gi[0, 0] == 6 * per
    bias[6 * per:7 * per] = -np.inf
    assert routed(ctx, l, bias, k, 1, 8, 1, 2)[0, 0] == 5 * per


@pytest.mark.parametrize("E,k", KERNELS)
def test_infinity_is_above_the_largest_float(ctx, E, k):
    l = np.zeros((2, E), np.float32)
    bias = np.zeros(E, np.float32)
    bias[[1, 3]], bias[[7, 50]], bias[60] = FLT_MAX, np.inf, FLT_MAX / 2
    gi = routed(ctx, l, bias, k, 1, 1, 1, 1)
    np.testing.assert_array_equal(gi[0, :4], [7, 50, 1, 3])


# ---- routing keeps nothing between calls ------------------------------------------------
def test_route_with_counts_needs_no_earlier_call(gpu_ctx_factory):
    """The first call of a context may be a captured one, and graphs of it may run beside it on other streams."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    E, k, M = 64, 4, 30000
    rng = np.random.default_rng(3)
    sets = []
    for _ in range(3):
        l = c.to_device(rng.standard_normal((M, E)).astype(np.float32))
        sets.append((l, c.empty((M, k), np.int32), c.empty((M, k)), c.empty(E, np.int32)))

    def call(i):
        l, idx, wt, n = sets[i]
        c.route(idx, wt, n, l, R.F32, E, None, None, M, E, k)

    graphs = [Captured(c, lambda i=i: call(i)) for i in range(2)]
    streams = []
    for g in graphs:
        s = ctypes.c_void_p()
        assert g.h.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0
        g.s = s
        streams.append(s)
    for turn in range(4):
        for _, idx, _, n in sets:
            idx.fill(0xFF)
            n.fill(0x7F)
        c.synchronize()
        for g in graphs:
            g.replay()
        call(2)
        c.synchronize()
        for s in streams:
            assert graphs[0].h.hipStreamSynchronize(s) == 0
        for _, idx, _, n in sets:
            got = idx.download()
            assert (got >= 0).all()
            np.testing.assert_array_equal(n.download(), np.bincount(got.ravel(), minlength=E))
    for g, s in zip(graphs, streams):
        g.close()
        assert g.h.hipStreamDestroy(s) == 0


# ---- activations and scores far from zero ---------------------------------------------
@pytest.mark.parametrize("M", [1, 40, 700])
def test_silu_of_any_size(ctx, M):
    """v / (1 + exp(-v)) of products without terms, whose values are their biases.  Bound: the
    hardware's exp2 and reciprocal are within 1 ulp (2 U each), the correction of the
    exponent, the sum and the product round once each (3 U), and U more covers second
    order; a subnormal result is within 2^-149."""
    v = np.concatenate([
        [-80, -87, -87.25, -87.33, -87.34, -87.4, -88, -88.1, -89, -90, -95, -100, -103, -103.9, -104.5, -110, -126,
         -127, -150, -1000, -1e10, -3e38, -FLT_MAX, 0.0, -0.0, 1e-45, -1e-45, 1e-30, -1e-30, 60, 80, 87.4, 88.7, 89, 104,
         200, 1e10, 3e38, FLT_MAX, np.inf, -np.inf, np.nan],
        -np.linspace(55, 112, 400), np.linspace(-30, 30, 301), np.linspace(80, 100, 41)]).astype(np.float32)
    N = len(v)
    out, one = Out(ctx, M, N, N, np.float32), ctx.to_device(np.ones(max(M, N), np.float32))
    null = View(one, 0)
    ctx.i8_matmul(out, R.F32, N, null, 0, one, null, 0, one, ctx.to_device(v), R.SILU, M, N, 0)
    with np.errstate(all="ignore"):
        w = v.astype(np.float64)
        y = w / (1.0 + np.exp(-w))
    assert np.isnan(y[41]) and np.isnan(y[40]) and y[39] == np.inf
    got = out.get().astype(np.float64)
    finite = np.isfinite(y)
    np.testing.assert_array_equal(got[:, ~finite], np.broadcast_to(y[~finite], (M, (~finite).sum())))
    tol = 8 * R.U * np.abs(y[finite]) + 2.0 ** -149
    off = np.abs(got[:, finite] - y[finite]) - tol
    assert (off <= 0).all(), w[finite][off.max(axis=0) > 0]


@pytest.mark.parametrize("E,k", KERNELS)
@pytest.mark.parametrize("score", [0, 1])
def test_neighbouring_logits_have_scores_of_their_own(ctx, E, k, score):
    """Of two logits one last bit apart the larger is chosen, where a last bit of the logit is
    eight of the score's or more: below -8 a score is within 3.5 of its last bits (the
    hardware's exp2 and reciprocal one each, the exponent's correction, the sum and the
    softmax's quotient half a one each)."""
    rng = np.random.default_rng(E)
    M = 3000
    low = -rng.uniform(16, 80, M).astype(np.float32)
    l = np.full((M, E), -100, np.float32)
    if score == 0:
        l[:, 3] = 0.0  # the sum is 1: the others are far below it
    first, second = rng.integers(4, E // 2, M), rng.integers(E // 2, E, M)
    l[np.arange(M), first] = low
    l[np.arange(M), second] = np.nextafter(low, np.float32(0))
    gi, _ = run_route(ctx, l, R.F32, None, None, k, score, 1, 1, 1, False, 1.0)
    at = 1 if score == 0 else 0
    np.testing.assert_array_equal(gi[:, at], second)
    np.testing.assert_array_equal(gi[:, at + 1], first)


# ---- empty widths ----------------------------------------------------------------------
@pytest.mark.parametrize("M,D,F,N,tile", [(2000, 0, 400, 390, 64), (2000, 20, 0, 390, 32), (30, 0, 16, 20, 1),
                                          (2000, 0, 0, 40, 32)])
@pytest.mark.parametrize("gated", [False, True])
def test_experts_of_empty_widths_and_unaligned_weights(ctx, M, D, F, N, tile, gated):
    """Nothing is read of weights that have no terms, so their address does not matter."""
    E, k = 4, 1
    assert tile_rows(M, k, E, D, F, N, gated) == tile
    rng = np.random.default_rng(M + D + F)
    weights = expert_case(rng, E, D, F, N, gated, True)
    w1, s1, b1, w2, s2, b2 = weights
    idx = rng.integers(0, E, (M, k)).astype(np.int32)
    wt = rng.random((M, k)).astype(np.float32)
    x = rng.standard_normal((M, max(D, 1))).astype(np.float32)

    def off(a):  # one byte past its alignment
        return View(ctx.to_device(np.concatenate([np.zeros(1, np.int8), a.ravel(), np.zeros(16, np.int8)])), 1)

    def some(a):
        return ctx.to_device(a if a.size else np.zeros(4, np.float32))

    dev = off(w1), some(s1), some(b1), off(w2), some(s2), some(b2)
    out = Out(ctx, M, N, N, np.float32)
    ctx.experts(out, R.F32, N, ctx.to_device(x), R.F32, max(D, 1), ctx.to_device(idx), ctx.to_device(wt), M, k,
                vdttfs.ExpertWeights(E, D, F, N, R.RELU, gated, *dev))
    q, s = R.quant_rows(x[:, :D])
    y, d, _ = R.experts(q, s, idx, wt, *weights, R.RELU, gated)
    check(out.get(), R.F32, y, d)


def test_a_call_without_scratch_can_be_captured_at_once(gpu_ctx_factory):
    """Few pairs of experts without hidden channels: the biases alone, and no scratch."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    rng = np.random.default_rng(1)
    E, D, N, M, k = 4, 20, 12, 5, 2
    s2, b2 = np.ones((E, N), np.float32), rng.standard_normal((E, N)).astype(np.float32)
    idx, wt = rng.integers(0, E, (M, k)).astype(np.int32), np.ones((M, k), np.float32)
    one = c.empty(64)
    ew = vdttfs.ExpertWeights(E, D, 0, N, R.NONE, False, one, one, None, one, c.to_device(s2), c.to_device(b2))
    x, di, dw, out = c.to_device(np.ones((M, D), np.float32)), c.to_device(idx), c.to_device(wt), c.empty((M, N))
    g = Captured(c, lambda: c.experts(out, R.F32, N, x, R.F32, D, di, dw, M, k, ew))
    for _ in range(3):
        out.fill(0xFF)
        g.replay()
        c.synchronize()
        np.testing.assert_array_equal(out.download(), b2[idx[:, 0]] + b2[idx[:, 1]])
    g.close()


# ---- sizes at the ends of their types ---------------------------------------------------
class Piece:
    """Part of a device array of `n` elements, from element `at` on."""

    def __init__(self, arr, at, n):
        self.ctx, self.ptr = arr.ctx, ctypes.c_void_p(arr.ptr.value + at * arr.dtype.itemsize)
        self.n, self.dtype = n, arr.dtype

    def put(self, values):
        h = np.ascontiguousarray(values, self.dtype)
        assert h.size == self.n
        _lib.check(vdttfs.lib().vdttfs_h2d(self.ctx.handle, self.ptr, ctypes.c_void_p(h.ctypes.data), h.nbytes))

    def get(self):
        h = np.empty(self.n, self.dtype)
        _lib.check(vdttfs.lib().vdttfs_d2h(self.ctx.handle, ctypes.c_void_p(h.ctypes.data), self.ptr, h.nbytes))
        return h


@pytest.mark.parametrize("elem", [R.BF16, R.TIMES])
def test_a_row_of_nearly_2_31_columns(ctx, elem):
    """The last of a thread's columns is past 2^31; 127 columns fewer end inside a thread's eight."""
    cols = (1 << 31) - 1
    x, q, s = ctx.empty(cols, R.np_type(elem)), ctx.empty(cols + 8, np.int8), ctx.empty(1)
    ends = np.arange(3000)
    if elem == R.BF16:
        x.fill(0x3F)  # 0x3F3F: 0.746
        h = R.to_bits(((ends % 255 - 127) / 127).astype(np.float32), elem)
    else:
        x.fill(0x7F)  # past every window
        h = (ends % 70).astype(np.float32)
    for n in (cols, cols - 127):
        Piece(x, 0, 3000).put(h)
        Piece(x, n - 3000, 3000).put(h)
        q.fill(0x5A)
        ctx.quant_rows(x, elem, cols, 1, n, q, cols, s)
        if elem == R.BF16:
            v = R.from_bits(h, elem)
            rq, rs = R.quant_rows(np.concatenate([v, [R.from_bits(np.full(1, 0x3F3F, np.uint16), elem)[0]]])[None])
            rq, filler = rq[0, :3000], rq[0, 3000]
        else:
            rq, rs = R.quant_times(h[None], 64, 0.0)
            rq, filler = rq[0], 0
        np.testing.assert_array_equal(Piece(q, 0, 3000).get(), rq)
        np.testing.assert_array_equal(Piece(q, n - 3000, 3000).get(), rq)
        assert (Piece(q, n, 8).get() == 0x5A).all()
        for at in (3000, n // 2, n - 4000):
            assert (Piece(q, at, 1000).get() == filler).all()
        assert s.download()[0] == rs[0]
    for a in (x, q):
        a.free()


def test_refusals_of_sizes_that_no_launch_serves(ctx):
    f, q, i = ctx.empty(64), ctx.empty(64, np.int8), ctx.empty(64, np.int32)
    for N in (_lib.I8_MAX_N + 1, (1 << 31) - 1):
        refused(_lib.E_UNSUPPORTED, ctx.quant_kernel, f, 1, N, q, 1, f)
        refused(_lib.E_UNSUPPORTED, ctx.i8_matmul, f, R.BF16, N, q, 1, f, q, 1, f, None, 0, 1, N, 1)
        refused(_lib.E_UNSUPPORTED, ctx.i8_linear, f, R.BF16, N, f, 0, 1, q, 1, f, None, 0, 1, N, 1)
        refused(_lib.E_UNSUPPORTED, ctx.experts, f, R.BF16, N, f, 0, 1, i, f, 1, 1,
                vdttfs.ExpertWeights(1, 1, 1, N, 0, False, q, f, None, q, f, None))
    for K in (_lib.I8_MAX_K + 1, (1 << 31) - 1):
        refused(_lib.E_UNSUPPORTED, ctx.experts, f, R.F32, 1, f, 0, K, i, f, 1, 1,
                vdttfs.ExpertWeights(1, K, 0, 1, 0, False, q, f, None, q, f, None))


@pytest.mark.parametrize("K", [1, 16])
def test_matmul_of_more_tiles_than_a_launch(ctx, K):
    """2^30 rows and some, one output each: 2^24 tiles of 64 rows, where a launch has fewer than 2^23."""
    M, a_launch = (1 << 30) + 77, ((1 << 23) - 1) * 64
    q, s, out = ctx.empty((M, K), np.int8), ctx.empty(M), ctx.empty(M, np.uint16)
    q.fill(1), s.fill(0x3F), out.fill(0xFF)
    scale = np.full(1, 0x3F3F3F3F, np.uint32).view(np.float32)[0]
    ends = [0, a_launch - 3, 2 * a_launch - 3, M - 6]
    for n, at in enumerate(ends):
        Piece(q, at * K, 6 * K).put(np.repeat(np.arange(6, dtype=np.int8) - 20 * (n + 1), K))
        Piece(s, at, 6).put(scale * np.arange(1, 7, dtype=np.float32))
    c = ctx.to_device(np.full(1, 1.0, np.float32))
    ctx.i8_matmul(out, R.BF16, 1, q, K, s, ctx.to_device(np.ones((1, K), np.int8)), K, c, None, R.NONE, M, 1, K)
    want = np.full(M, R.to_bits(np.full(1, K * scale, np.float32), R.BF16)[0], np.uint16)
    for n, at in enumerate(ends):
        v = K * (np.arange(6) - 20.0 * (n + 1)) * (scale * np.arange(1, 7, dtype=np.float32))
        want[at:at + 6] = R.to_bits(v.astype(np.float32), R.BF16)
    np.testing.assert_array_equal(out.download(), want)
    for a in (q, s, out):
        a.free()
