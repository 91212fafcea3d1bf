"""Microscaled 4-bit rows: quantisation and products against their definitions in
64 bits, with bounds from the roundings alone (tests/moreref.py)."""
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


def bytes_of(cols):
    return (cols + 1) // 2


def blocks_of(cols):
    return -(-cols // 32)


def quantised(ctx, bits, elem, cols, pad_x=0, pad_q=0, pad_s=0):
    rows = len(bits)
    n, b = bytes_of(cols), blocks_of(cols)
    q, s = Out(ctx, rows, n, n + pad_q, np.uint8), Out(ctx, rows, b, b + pad_s, np.uint8)
    ctx.mx4_quant_rows(ctx.to_device(strided(bits, cols + pad_x)), elem, cols + pad_x, rows, cols, q, n + pad_q, s,
                       b + pad_s)
    return q.get(), s.get()


def check_codes(got, x):
    q, s = got
    c, rs = Q.mx4_quant(x)
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(q, Q.mx4_pack(c))


# ---- quantisation ---------------------------------------------------------------
@pytest.mark.parametrize("elem", [R.F32, R.BF16, R.F16])
@pytest.mark.parametrize("rows,cols,pads", [(1, 1, (0, 0, 0)), (1, 2, (1, 3, 1)), (3, 7, (5, 1, 2)), (5, 31, (0, 0, 0)),
                                            (4, 32, (0, 0, 0)), (2, 33, (3, 5, 1)), (9, 513, (0, 0, 0)),
                                            (300, 100, (12, 14, 0)), (2, 4097, (1, 1, 1)), (70, 1000, (0, 12, 1))])
def test_codes_are_exact(ctx, elem, rows, cols, pads):
    rng = np.random.default_rng(rows * 1000 + cols + elem)
    x = (rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, cols)))).astype(np.float32)
    if rows > 2:
        x[1] = 0
        x[2, :cols // 2] = 0
    bits = R.to_bits(x, elem)
    check_codes(quantised(ctx, bits, elem, cols, *pads), R.from_bits(bits, elem))


def test_every_element_and_every_half_way(ctx):
    """All multiples of 1/16 up to 8 at each of a few scales: ties go to even, the largest do not grow."""
    t = np.arange(-128, 129) / 16
    rows = []
    for e in (-126, -20, 0, 5, 120):
        for lead in (7.9, 6.0, 4.0):
            r = np.zeros((len(t), 32))
            r[:, 0], r[:, 13] = lead, t
            r[:, 31] = -t
            rows.append(np.ldexp(r, e))
    x = np.concatenate(rows).astype(np.float32)
    check_codes(quantised(ctx, x, R.F32, 32), x)


def test_powers_of_two_and_their_neighbours_lead(ctx):
    """The scale is that of the largest value, to its last bit."""
    p = np.ldexp(1.0, np.arange(-149, 128)).astype(np.float32)
    lead = np.concatenate([p, np.nextafter(p, np.float32(0)), np.nextafter(p, np.float32(np.inf))])
    lead = lead[np.isfinite(lead)]
    rng = np.random.default_rng(3)
    x = (rng.uniform(-1, 1, (len(lead), 40)) * lead[:, None].astype(np.float64)).astype(np.float32)
    x[:, 5], x[:, 38] = lead, -lead
    check_codes(quantised(ctx, x, R.F32, 40), x)
    bits = R.to_bits(x, R.BF16)
    check_codes(quantised(ctx, bits, R.BF16, 40), R.from_bits(bits, R.BF16))


def test_subnormals_of_16_bits(ctx):
    bits = np.arange(1, 0x0400, dtype=np.uint16).reshape(-1, 33)  # 31 rows of 33
    check_codes(quantised(ctx, bits, R.F16, 33), R.from_bits(bits, R.F16))
    bits = np.arange(1, 0x0080 * 3 + 1, dtype=np.uint16).reshape(-1, 32)
    check_codes(quantised(ctx, bits, R.BF16, 32), R.from_bits(bits, R.BF16))


@pytest.mark.parametrize("elem", [R.F32, R.BF16, R.F16])
def test_blocks_that_are_not_finite(ctx, elem):
    x = np.ones((6, 100), np.float32)
    x[0, 3], x[1, 99], x[2, 64] = np.nan, np.inf, -np.inf
    x[3, 40], x[3, 41], x[4, 0] = np.nan, np.inf, -0.0
    x[5] = -0.0
    bits = R.to_bits(x, elem)
    q, s = quantised(ctx, bits, elem, 100)
    c, rs = Q.mx4_quant(x)
    assert rs[0, 0] == 255 and rs[1, 3] == 255 and rs[0, 1] != 255
    np.testing.assert_array_equal(s, rs)
    np.testing.assert_array_equal(q, Q.mx4_pack(c))


@pytest.mark.parametrize("T,tfs", [(1, 0.0), (64, 0.0), (64, 32.0), (80, 40.0), (255, 3.5)])
def test_spike_times(gpu_ctx_factory, T, tfs):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=T, tfs=tfs, delta=16))
    rng = np.random.default_rng(T)
    t = np.floor(rng.random((7, 301)) * (T + tfs + 4)).astype(np.float32)
    t[rng.random(t.shape) < 0.3] = 9999.0
    t[0, :4], t[1, :3] = [np.nan, np.inf, -5.0, 1e9], [T + tfs - 0.25, T + tfs, tfs - 0.5]
    t[2] = 9999.0
    check_codes(quantised(c, t, R.TIMES, 301, 2, 1, 3), Q.mx4_times(t, T, tfs))


@pytest.mark.parametrize("c_in,c_out", [(1, 1), (16, 64), (37, 65), (512, 10), (300, 130), (33, 200)])
def test_kernel_is_rows_of_the_transpose(ctx, c_in, c_out):
    w = np.random.default_rng(c_in).standard_normal((c_in, c_out)).astype(np.float32)
    w[:, 0] = 0
    if c_out > 2:
        w[c_in // 2, 2] = np.inf
    n, b = bytes_of(c_in), blocks_of(c_in)
    q, s = Out(ctx, c_out, n, n + 3, np.uint8), Out(ctx, c_out, b, b + 1, np.uint8)
    ctx.mx4_quant_kernel(ctx.to_device(w), c_in, c_out, q, n + 3, s, b + 1)
    check_codes((q.get(), s.get()), np.ascontiguousarray(w.T))


# ---- products -------------------------------------------------------------------
def operand(ctx, rng, rows, cols, pad=0, shift=0, spread=8):
    """Random codes of every kind and random scales: (device codes, device scales, ld, lds, values)."""
    n, b = bytes_of(cols), blocks_of(cols)
    c = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    s = rng.integers(127 - spread, 127, (rows, b)).astype(np.uint8)
    q = Q.mx4_pack(c)
    if cols % 2:
        q[:, -1] |= rng.integers(0, 16, rows).astype(np.uint8) << 4  # not an element
    at = lambda a, ld: View(ctx.to_device(np.concatenate([np.full(shift, 255, np.uint8), strided(a, ld).ravel()])), shift)  # noqa: E731
    return at(q, n + pad), at(s, b + pad), n + pad, b + pad, Q.mx4_values(c, s)


SIZES = [(1, 1, 1), (1, 16, 64), (1, 100, 4096), (2, 33, 15), (4, 64, 127), (5, 129, 1000), (16, 17, 128), (17, 64, 129),
         (31, 300, 513), (64, 64, 256), (65, 127, 300), (129, 257, 385), (300, 10, 77), (256, 512, 512), (7, 1024, 8192),
         (513, 1030, 640), (1100, 257, 300), (1500, 512, 128), (2100, 300, 1024), (1025, 70, 90), (1024, 1024, 400),
         (2000, 2100, 208), (1300, 5000, 288), (900, 700, 1000), (2600, 2600, 1504), (2561, 2500, 1601), (1, 3000, 33),
         (16, 4096, 2048), (13, 555, 7001), (100, 100, 20000)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("elem,kind,bias,pad,shift", [(R.F32, R.NONE, False, 0, 0), (R.F32, R.SILU, True, 3, 1),
                                                      (R.BF16, R.RELU, True, 16, 0), (R.F16, R.SILU, False, 0, 0),
                                                      (R.F16, R.NONE, True, 5, 7)])
def test_matmul(ctx, M, N, K, elem, kind, bias, pad, shift):
    """pad: bytes between rows; shift: bytes by which codes and scales miss their alignment."""
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    q, s, ld, lds, x = operand(ctx, rng, M, K, pad, shift)
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K, pad, shift)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    out = Out(ctx, M, N, N + pad, R.np_type(elem))
    ctx.mx4_matmul(out, elem, N + pad, q, ld, s, lds, w, ldw, ws, ldws, ctx.to_device(b) if bias else None, kind, M, N,
                   K)
    y, d = Q.mx4_product(x, wv, b, kind)
    check(out.get(), elem, y, d)


@pytest.mark.parametrize("M,N,K", [(1, 40, 500), (40, 70, 500), (300, 500, 1024), (600, 700, 2048)])
def test_matmul_of_scales_far_apart(ctx, M, N, K):
    """Scales over 2^60 each: sums keep 32-bit floats' precision of their largest terms."""
    rng = np.random.default_rng(M)
    q, s, ld, lds, x = operand(ctx, rng, M, K, spread=60)
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K, spread=60)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_matmul(out, R.F32, N, q, ld, s, lds, w, ldw, ws, ldws, None, R.NONE, M, N, K)
    check(out.get(), R.F32, *Q.mx4_product(x, wv, None, R.NONE))


@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (40, 70, 300), (200, 300, 1024), (1000, 900, 1024)])
def test_a_nan_block_reaches_its_row_and_its_channel_alone(ctx, M, N, K):
    rng = np.random.default_rng(K)
    c, s = rng.integers(0, 16, (M, K)).astype(np.uint8), np.full((M, blocks_of(K)), 126, np.uint8)
    w, ws = rng.integers(0, 16, (N, K)).astype(np.uint8), np.full((N, blocks_of(K)), 126, np.uint8)
    s[M // 2, -1], ws[N // 3, 0] = 255, 255
    c[M // 2, (blocks_of(K) - 1) * 32:] = 0
    n, b = bytes_of(K), blocks_of(K)
    out = Out(ctx, M, N, N, np.float32)
    dev = [ctx.to_device(a) for a in (Q.mx4_pack(c), s, Q.mx4_pack(w), ws)]
    ctx.mx4_matmul(out, R.F32, N, dev[0], n, dev[1], b, dev[2], n, dev[3], b, None, R.NONE, M, N, K)
    y, d = Q.mx4_product(Q.mx4_values(c, s), Q.mx4_values(w, ws), None, R.NONE)
    assert np.isnan(y[M // 2]).all() and np.isnan(y[:, N // 3]).all() and np.isnan(y).sum() == M + N - 1
    check(out.get(), R.F32, y, d)


@pytest.mark.parametrize("M,N", [(1, 5), (3, 70), (200, 130)])
def test_matmul_of_no_terms_is_the_bias(ctx, M, N):
    b = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_matmul(out, R.F32, N, Null, 0, Null, 0, Null, 0, Null, 0, ctx.to_device(b), R.NONE, M, N, 0)
    np.testing.assert_array_equal(out.get(), np.broadcast_to(b, (M, N)))


@pytest.mark.parametrize("M,N,K", [(3, 70, 700), (40, 70, 160), (300, 333, 500), (200, 300, 1024), (900, 1100, 1280),
                                   (1500, 1300, 1024)])
def test_matmul_of_scales_at_both_ends(ctx, M, N, K):
    """Scales from 2^-127 to 2^127 whose products are near 1: sums of them are exact; elements of 0 under the largest."""
    rng = np.random.default_rng(M + K)
    b = blocks_of(K)
    c, w = rng.integers(0, 16, (M, K)).astype(np.uint8), rng.integers(0, 16, (N, K)).astype(np.uint8)
    a = rng.integers(0, 255, b)
    a[:3] = 0, 254, 127
    s = np.tile(a.astype(np.uint8), (M, 1))
    ws = np.clip(254 - a + rng.integers(-2, 3, (N, b)), 0, 254).astype(np.uint8)
    s[:, 3], ws[:, 3] = 254, 254
    c[:, 96:128] &= 8  # zeros of both signs
    n = bytes_of(K)
    out = Out(ctx, M, N, N, np.float32)
    dev = [ctx.to_device(v) for v in (Q.mx4_pack(c), s, Q.mx4_pack(w), ws)]
    ctx.mx4_matmul(out, R.F32, N, dev[0], n, dev[1], b, dev[2], n, dev[3], b, None, R.NONE, M, N, K)
    # multiples of 2^-4 below 2^18: exact in every order
    np.testing.assert_array_equal(out.get(), Q.mx4_values(c, s) @ Q.mx4_values(w, ws).T)


@pytest.mark.parametrize("M,N,K", [(3, 70, 64), (40, 70, 64), (300, 333, 500), (200, 300, 512)])
def test_matmul_of_sums_below_the_normal_range(ctx, M, N, K):
    rng = np.random.default_rng(M)
    b, n = blocks_of(K), bytes_of(K)
    c, w = rng.integers(0, 16, (M, K)).astype(np.uint8), rng.integers(0, 16, (N, K)).astype(np.uint8)
    s, ws = np.full((M, b), 60, np.uint8), np.full((N, b), 127 - 60 - 10, np.uint8)  # products of 2^-137
    out = Out(ctx, M, N, N, np.float32)
    dev = [ctx.to_device(v) for v in (Q.mx4_pack(c), s, Q.mx4_pack(w), ws)]
    ctx.mx4_matmul(out, R.F32, N, dev[0], n, dev[1], b, dev[2], n, dev[3], b, None, R.NONE, M, N, K)
    np.testing.assert_array_equal(out.get(), Q.mx4_values(c, s) @ Q.mx4_values(w, ws).T)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_of_no_terms_is_the_bias(ctx, M):
    N = 50
    b = np.random.default_rng(1).standard_normal(N).astype(np.float32)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_linear(out, R.F32, N, Null, R.F32, 0, Null, 0, Null, 0, ctx.to_device(b), R.NONE, M, N, 0)
    np.testing.assert_array_equal(out.get(), np.broadcast_to(b, (M, N)))


def operand_at(ctx, rng, rows, cols, off_q, off_s):
    """operand with rows of codes off 16 bytes by off_q and of scales off 4 by off_s, first rows too."""
    c = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    s = rng.integers(120, 127, (rows, blocks_of(cols))).astype(np.uint8)
    ld, lds = -(-bytes_of(cols) // 16) * 16 + off_q, -(-blocks_of(cols) // 4) * 4 + off_s
    at = lambda a, ld, off: View(ctx.to_device(np.concatenate([np.full(off, 255, np.uint8), strided(a, ld).ravel()])), off)  # noqa: E731
    return at(Q.mx4_pack(c), ld, off_q), at(s, lds, off_s), ld, lds, Q.mx4_values(c, s)


@pytest.mark.parametrize("M,N,K", [(2561, 4200, 512), (3329, 3001, 545), (1400, 1500, 3001), (4097, 200, 2050),
                                   (70, 8200, 1025), (513, 769, 4100)])
@pytest.mark.parametrize("off", [(0, 0, 0, 0), (3, 0, 0, 0), (0, 1, 0, 0), (0, 0, 8, 0), (0, 0, 0, 2), (0, 3, 4, 0),
                                 (5, 0, 0, 1), (0, 1, 0, 3), (2, 1, 7, 2)])
def test_large_matmul_at_any_alignment(ctx, M, N, K, off):
    """off: bytes by which codes and scales of the rows, then of the channels, miss 16 and 4."""
    rng = np.random.default_rng(M + N + K)
    q, s, ld, lds, x = operand_at(ctx, rng, M, K, *off[:2])
    w, ws, ldw, ldws, wv = operand_at(ctx, rng, N, K, *off[2:])
    b = rng.standard_normal(N).astype(np.float32)
    out = Out(ctx, M, N, N + 1, np.float32)
    ctx.mx4_matmul(out, R.F32, N + 1, q, ld, s, lds, w, ldw, ws, ldws, ctx.to_device(b), R.NONE, M, N, K)
    check(out.get(), R.F32, *Q.mx4_product(x, wv, b, R.NONE))


def test_matmul_that_copies_in_a_graph(gpu_ctx_factory):
    """Rows off 16 bytes are copied to scratch: a capture before any call is refused, and goes on."""
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    M, N, K = 1200, 1300, 5001
    rng = np.random.default_rng(4)
    n, b = bytes_of(K), blocks_of(K)
    w, ws, ldw, ldws, _ = operand_at(c, rng, N, K, 5, 1)
    q, s, out = c.empty((M, n), np.uint8), c.empty((M, b), np.uint8), c.empty((M, N), np.float32)
    s.fill(127)
    f = c.empty(32)
    seen = []

    def call():
        c.mx4_matmul(out, R.F32, N, q, n, s, b, w, ldw, ws, ldws, None, R.NONE, M, N, K)

    def refused_call():
        with pytest.raises(vdttfs.VdttfsError) as e:
            call()
        seen.append(e.value.code)
        c.mx4_quant_rows(f, R.F32, 32, 1, 32, q, n, s, b)  # the capture goes on

    Captured(c, refused_call).close()
    assert seen == [_lib.E_UNSUPPORTED]
    call()
    c.synchronize()
    g = Captured(c, call)
    for seed in range(4):
        q.upload(np.random.default_rng(seed).integers(0, 256, (M, n)).astype(np.uint8))
        out.fill(0xFF)
        g.replay()
        c.synchronize()
        got = out.download()
        call()
        c.synchronize()
        np.testing.assert_array_equal(got, out.download())
        assert np.isfinite(got).all() and got.any()
    g.close()


def test_matmul_past_32_bit_offsets(ctx):
    """Rows of codes 2.4 GB apart from first to last, and rows of outputs."""
    M, N, K, ld = 8192, 96, 400, 300032
    rng = np.random.default_rng(5)
    x = rng.standard_normal((M, K)).astype(np.float32)
    q, s = ctx.empty(M * ld, np.uint8), ctx.empty(M * 16, np.uint8)
    ctx.mx4_quant_rows(ctx.to_device(x), R.F32, K, M, K, q, ld, s, 16)
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_matmul(out, R.F32, N, q, ld, s, 16, w, ldw, ws, ldws, None, R.NONE, M, N, K)
    check(out.get(), R.F32, *Q.mx4_product(Q.mx4_values(*Q.mx4_quant(x)), wv, None, R.NONE))
    q.free()


def test_matmul_of_rows_longer_than_offsets(ctx):
    """128 rows of codes span 2^31 bytes: ones in the upper half of the rows, twos in the lower."""
    M, K = 1408, 33554432 + 160
    n, b = K // 2, K // 32
    q, s, out = ctx.empty(M * n, np.uint8), ctx.empty(M * b, np.uint8), Out(ctx, M, M, M, np.float32)
    q.fill(0x22)
    _lib.check(_lib.lib().vdttfs_memset(ctx.handle, View(q, M // 2 * n).ptr, 0x44, M // 2 * n))
    s.fill(127)
    ctx.mx4_matmul(out, R.F32, M, q, n, s, b, q, n, s, b, None, R.NONE, M, M, K)
    half = np.where(np.arange(M) < M // 2, 1.0, 2.0)
    np.testing.assert_array_equal(out.get(), np.outer(half, half) * K)  # sums of 32s: exact
    q.free()
    s.free()


@pytest.mark.parametrize("M,N,K", [(1, 70, 333), (3, 70, 333), (16, 70, 333), (20, 70, 333), (150, 70, 333), (1, 4096, 4096),
                                   (5, 1000, 2048), (16, 300, 8192), (700, 600, 512), (33, 40, 1)])
@pytest.mark.parametrize("x_elem", [R.F32, R.BF16, R.F16, R.TIMES])
def test_linear_is_quant_rows_then_matmul(ctx, M, N, K, x_elem):
    ldx = K + 7
    rng = np.random.default_rng(M + K)
    if x_elem == R.TIMES:
        bits = np.floor(rng.random((M, K)) * 70).astype(np.float32)
        bits[rng.random(bits.shape) < 0.4] = 9999
        x = Q.mx4_times(bits, 64, 0.0)
    else:
        x = (rng.standard_normal((M, K)) * 3).astype(np.float32)
        if M > 2:
            x[1, K // 2], x[2] = np.nan, 0  # one row poisoned, one empty; the others stay
        bits = R.to_bits(x, x_elem)
        x = R.from_bits(bits, x_elem)
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K)
    b = rng.standard_normal(N).astype(np.float32)
    out = Out(ctx, M, N, N + 1, np.float32)
    ctx.mx4_linear(out, R.F32, N + 1, ctx.to_device(strided(bits, ldx)), x_elem, ldx, w, ldw, ws, ldws,
                   ctx.to_device(b), R.NONE, M, N, K)
    check(out.get(), R.F32, *Q.mx4_product(Q.mx4_values(*Q.mx4_quant(x)), wv, b, R.NONE))


def test_linear_again_smaller_and_larger(ctx):
    """Scratch of another call's size is neither read nor relied on."""
    rng = np.random.default_rng(2)
    for M, N, K in [(300, 100, 700), (3, 50, 33), (40, 64, 1000), (1, 8, 1), (20, 30, 129), (300, 100, 701)]:
        x = rng.standard_normal((M, K)).astype(np.float32)
        w, ws, ldw, ldws, wv = operand(ctx, rng, N, K)
        out = Out(ctx, M, N, N, np.float32)
        ctx.mx4_linear(out, R.F32, N, ctx.to_device(x), R.F32, K, w, ldw, ws, ldws, None, R.NONE, M, N, K)
        check(out.get(), R.F32, *Q.mx4_product(Q.mx4_values(*Q.mx4_quant(x)), wv, None, R.NONE))


@pytest.mark.parametrize("M,N,K", [(1, 300, 1024), (90, 200, 515), (500, 600, 1024)])
def test_linear_in_a_graph(gpu_ctx_factory, M, N, K):
    c = gpu_ctx_factory(vdttfs.TaskConsts(T=64, delta=16))
    rng = np.random.default_rng(8)
    w, ws, ldw, ldws, _ = operand(c, rng, N, K)
    x, out = c.to_device(np.zeros((M, K), np.float32)), c.empty((M, N), np.float32)

    def call():
        c.mx4_linear(out, R.F32, N, x, R.F32, K, w, ldw, ws, ldws, None, R.SILU, M, N, K)

    call()
    c.synchronize()
    g = Captured(c, call)
    for seed in range(4):
        x.upload(np.random.default_rng(seed).standard_normal((M, K)).astype(np.float32))
        out.fill(0xFF)
        g.replay()
        c.synchronize()
        got = out.download()
        call()
        c.synchronize()
        np.testing.assert_array_equal(got, out.download())
        # a larger call grows the scratch; the graph keeps its own
        big = np.ones((1000, 3000 + 1000 * seed), np.float32)
        bw, bws, bld, blds, _ = operand(c, rng, 20, big.shape[1])
        c.mx4_linear(c.empty((1000, 20)), R.F32, 20, c.to_device(big), R.F32, big.shape[1], bw, bld, bws, blds, None,
                     R.NONE, 1000, 20, big.shape[1])
    g.close()


# ---- refusals -------------------------------------------------------------------
def test_refusals(ctx):
    f, q = ctx.empty(4096, np.float32), ctx.empty(4096, np.uint8)
    odd, two = View(f, 2), View(f, 1)
    INV, UNS = _lib.E_INVALID, _lib.E_UNSUPPORTED
    rows = dict(d_x=f, elem=0, ldx=40, rows=2, cols=40, d_q=q, ldq=20, d_s=q, lds=2)
    for bad in [dict(elem=4), dict(elem=-1), dict(ldx=39), dict(rows=-1), dict(cols=-1), dict(ldq=19), dict(lds=1),
                dict(d_x=Null), dict(d_q=Null), dict(d_s=Null), dict(d_x=odd), dict(d_x=two, elem=1)]:
        refused(INV, ctx.mx4_quant_rows, **{**rows, **bad})
    refused(UNS, ctx.mx4_quant_rows, **{**rows, "rows": 1 << 31})
    kern = dict(d_kernel=f, C_in=40, C_out=4, d_w=q, ldw=20, d_ws=q, ldws=2)
    for bad in [dict(C_in=-1), dict(C_out=-1), dict(ldw=19), dict(ldws=1), dict(d_kernel=Null), dict(d_w=Null),
                dict(d_ws=Null), dict(d_kernel=odd)]:
        refused(INV, ctx.mx4_quant_kernel, **{**kern, **bad})
    refused(UNS, ctx.mx4_quant_kernel, **{**kern, "C_out": _lib.I8_MAX_N + 1})
    good = dict(d_out=f, out_elem=0, ldo=8, d_q=q, ldq=20, d_s=q, lds=2, d_w=q, ldw=20, d_ws=q, ldws=2, d_bias=None,
                act=0, M=2, N=8, K=40)
    for bad in [dict(out_elem=3), dict(out_elem=-1), dict(ldo=7), dict(ldq=19), dict(lds=1), dict(ldw=19), dict(ldws=1),
                dict(act=3), dict(act=-1), dict(M=-1), dict(N=-1), dict(K=-1), dict(d_out=Null), dict(d_q=Null),
                dict(d_s=Null), dict(d_w=Null), dict(d_ws=Null), dict(d_out=odd), dict(d_bias=odd),
                dict(out_elem=2, d_out=two)]:
        refused(INV, ctx.mx4_matmul, **{**good, **bad})
    refused(UNS, ctx.mx4_matmul, **{**good, "M": 1 << 31})
    refused(UNS, ctx.mx4_matmul, **{**good, "N": _lib.I8_MAX_N + 1, "ldo": 1 << 30})
    lin = {k: v for k, v in good.items() if k not in ("d_q", "ldq", "d_s", "lds")}
    lin.update(d_x=f, x_elem=0, ldx=40)
    for bad in [dict(x_elem=4), dict(ldx=39), dict(d_x=Null), dict(d_x=odd), dict(ldo=7), dict(d_w=Null), dict(act=3)]:
        refused(INV, ctx.mx4_linear, **{**lin, **bad})


def test_empty_calls_do_nothing(ctx):
    ctx.mx4_quant_rows(Null, 0, 8, 0, 8, Null, 4, Null, 1)
    ctx.mx4_quant_rows(Null, 0, 8, 3, 0, Null, 4, Null, 1)
    ctx.mx4_quant_kernel(Null, 0, 8, Null, 4, Null, 1)
    ctx.mx4_matmul(Null, 0, 8, Null, 8, Null, 1, Null, 8, Null, 1, None, 0, 0, 8, 16)
    ctx.mx4_linear(Null, 0, 8, Null, 0, 16, Null, 8, Null, 1, None, 0, 3, 0, 16)
