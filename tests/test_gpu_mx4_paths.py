"""Every kernel of the microscaled 4-bit products, each asserted by the library's
own rule to be the one that a size takes, past the first turns of its loops.

Scales are 2^-2, 2^-1 and 1: products of elements are then multiples of 2^-6 and
sums of up to 7281 of them stay below 2^18, so every order of additions is exact in
32 bits, and a code or a scale out of place shows."""
import ctypes as C

import numpy as np
import pytest

import headref as R
import moreref as Q
import vdttfs
from test_gpu_heads import Out, View, ctx, strided  # noqa: F401

pytestmark = pytest.mark.gpu

FEW, TILE32, TILE64, LDS32, LDS64, LDS128, LDS256 = range(7)
MOST = 2 ** 24 // (36 * 64)  # terms whose sum is exact


class Args(C.Structure):
    _fields_ = [("A", C.c_void_p), ("lda", C.c_int64), ("sa", C.c_void_p), ("ldsa", C.c_int64), ("B", C.c_void_p),
                ("ldb", C.c_int64), ("sb", C.c_void_p), ("ldsb", C.c_int64), ("bias", C.c_void_p), ("out", C.c_void_p),
                ("ldo", C.c_int64), ("M", C.c_int64), ("N", C.c_int), ("K", C.c_int), ("act", C.c_int),
                ("out_elem", C.c_int)]


class Plan(C.Structure):
    _fields_ = [("path", C.c_int), ("a", C.c_bool), ("sa", C.c_bool), ("b", C.c_bool), ("sb", C.c_bool)]


def plan(q, ld, s, lds, w, ldw, ws, ldws, M, N, K):
    """(kernel, which of rows, their scales, channels, their scales are copied first)."""
    f = vdttfs.lib()["_ZN6vdttfs8mx4_planERKNS_7Mx4ArgsE"]
    f.argtypes, f.restype = [C.c_void_p], Plan
    a = Args(q.ptr, ld, s.ptr, lds, w.ptr, ldw, ws.ptr, ldws, None, None, N, M, N, K, R.NONE, R.F32)
    p = f(C.byref(a))
    return p.path, (p.a, p.sa, p.b, p.sb)


def operand(ctx, rng, rows, cols, off_q=0, off_s=0):
    """Rows of codes off 16 bytes by off_q and of scales off 4 by off_s, first rows too, and their values."""
    c = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    s = rng.integers(125, 128, (rows, -(-cols // 32))).astype(np.uint8)
    q = Q.mx4_pack(c)
    if cols % 2:
        q[:, -1] |= rng.integers(0, 16, rows).astype(np.uint8) << 4  # not an element
    ld, lds = -(-q.shape[1] // 16) * 16 + off_q, -(-s.shape[1] // 4) * 4 + off_s
    at = lambda a, ld, off: View(ctx.to_device(np.concatenate([np.full(off, 255, np.uint8), strided(a, ld).ravel()])), off)  # noqa: E731
    return at(q, ld, off_q), at(s, lds, off_s), ld, lds, Q.mx4_values(c, s).astype(np.float32)


# K: a multiple of 256 or not, odd and even numbers of steps of 256, spans of four steps that are whole and not
CASES = [
    (16, 700, 5000, FEW), (9, 300, 511, FEW), (130, 200, 7000, FEW), (1, 4000, 4096, FEW),
    (40, 500, 77, TILE32), (300, 333, 511, TILE32), (900, 1100, 257, TILE64), (1100, 900, 500, TILE64),
    (200, 300, 512, LDS32), (200, 300, 1000, LDS32), (300, 700, 1024, LDS32), (301, 701, 2305, LDS32),
    (250, 1000, 3333, LDS32),
    (900, 1100, 512, LDS64), (900, 1100, 770, LDS64), (901, 1101, 1280, LDS64), (899, 1099, 1793, LDS64),
    (1500, 1300, 512, LDS128), (1401, 1501, 1025, LDS128), (1400, 1500, 2304, LDS128), (1601, 1299, 4097, LDS128),
    (1500, 1300, 6100, LDS128),
    (3329, 3001, 512, LDS256), (3329, 3001, 768, LDS256), (3329, 3001, 1313, LDS256), (3400, 3329, 1536, LDS256),
    (2561, 4200, 1801, LDS256), (3329, 3001, 2049, LDS256), (3329, 3001, 2304, LDS256), (3329, 3001, 4097, LDS256),
    (2561, 4097, 5120, LDS256)]


@pytest.mark.parametrize("M,N,K,path", CASES)
def test_every_kernel_past_its_first_turns(ctx, M, N, K, path):  # noqa: F811
    assert K <= MOST
    rng = np.random.default_rng(M * 3 + N + K)
    q, s, ld, lds, x = operand(ctx, rng, M, K)
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K)
    assert plan(q, ld, s, lds, w, ldw, ws, ldws, M, N, K) == (path, (False,) * 4)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_matmul(out, R.F32, N, q, ld, s, lds, w, ldw, ws, ldws, None, R.NONE, M, N, K)
    np.testing.assert_array_equal(out.get(), x @ wv.T)


@pytest.mark.parametrize("M,N,K,path", [(3329, 3001, 1313, LDS256), (3329, 3001, 2049, LDS256), (3400, 3329, 2304, LDS256),
                                        (1601, 1999, 2050, LDS128), (899, 1099, 6401, LDS64)])
@pytest.mark.parametrize("off", [(3, 0, 0, 0), (0, 0, 8, 0), (0, 1, 0, 3), (5, 0, 0, 1), (2, 1, 7, 2)])
def test_copied_operands(ctx, M, N, K, path, off):  # noqa: F811
    """off: bytes by which codes and scales of the rows, then of the channels, miss 16 and 4; scales go to LDS in
    fours in the large tiles alone."""
    rng = np.random.default_rng(M + N + K)
    q, s, ld, lds, x = operand(ctx, rng, M, K, *off[:2])
    w, ws, ldw, ldws, wv = operand(ctx, rng, N, K, *off[2:])
    copied = (off[0] > 0, off[1] > 0 and path >= LDS128, off[2] > 0, off[3] > 0 and path >= LDS128)
    both = copied[0] and copied[2]
    assert float(M) * N * K >= (6e9 if both else 3e9)
    assert plan(q, ld, s, lds, w, ldw, ws, ldws, M, N, K) == (path, copied)
    out = Out(ctx, M, N, N, np.float32)
    ctx.mx4_matmul(out, R.F32, N, q, ld, s, lds, w, ldw, ws, ldws, None, R.NONE, M, N, K)
    np.testing.assert_array_equal(out.get(), x @ wv.T)
