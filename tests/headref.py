"""The 8-bit heads from their definitions, in 64 bits with numpy, and how far a
correct 32-bit evaluation may be from them.

What the definition rounds is rounded here too (scales and quotients of a
quantisation, to 32 bits); everything else is in 64.  Bounds: U = 2^-24 is the
rounding of one 32-bit operation; an output adds the rounding of its own type
(2^-24, 2^-8 or 2^-11 of its value for 24, 8 and 11 significant bits, and half
of its smallest subnormal).
"""
import numpy as np

U = 2.0 ** -24
F32, BF16, F16, TIMES = 0, 1, 2, 3
NONE, RELU, SILU = 0, 1, 2
OUT_U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
OUT_TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def to_bits(x, elem):
    """float32 values as the element type's bits, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if elem == BF16:
        u = x.view(np.uint32)
        r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(x), np.uint16(0x7FC0), r)
    if elem == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    return x


def from_bits(b, elem):
    if elem == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32)
    if elem == F16:
        return b.view(np.float16).astype(np.float32)
    return b


def np_type(elem):
    return np.uint16 if elem in (BF16, F16) else np.float32


def quant_rows(x):
    """Codes and scales of float rows: the definition's own 32-bit divisions."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(axis=1, initial=np.float32(0))
        s = (a / np.float32(127)).astype(np.float32)
        s = np.where(np.isfinite(a), s, np.float32(np.nan)).astype(np.float32)
        ok = np.isfinite(a) & (s != 0)
        q = np.rint(x / np.where(ok, s, np.float32(1))[:, None])
    q = np.where(ok[:, None], np.clip(np.nan_to_num(q), -127, 127), 0)
    return q.astype(np.int8), s


def quant_times(t, T, tfs):
    t = np.asarray(t, np.float32)
    with np.errstate(all="ignore"):
        b = np.floor((t - np.float32(tfs)).astype(np.float64))
    b = np.where(b < 0, 0, b)
    hit = (t < 9999.0) & (b < T)
    L = min(T, 127)
    q = np.rint(((T - np.where(hit, b, 0)) * L).astype(np.float32) / np.float32(T))
    return np.where(hit, q, 0).astype(np.int8), np.full(len(t), np.float32(1) / np.float32(L), np.float32)


def act(v, kind):
    if kind == RELU:
        return np.where(v < 0, 0.0, v)
    if kind == SILU:
        with np.errstate(over="ignore", invalid="ignore"):
            return v / (1.0 + np.exp(-v))
    return v


def act_bound(v, d, kind):
    """Error of act at v off by d: |silu'| < 1.1, and its exp (2 roundings), sum and quotient."""
    if kind == SILU:
        return 1.1 * d + 5 * U * np.abs(act(v, SILU)) + 1e-37
    return d


def product(q, s, w, c, b, kind):
    """(values, bound) before the output's rounding: the sum is exact, its
    conversion, the two scales and the bias round once each."""
    acc = q.astype(np.float64) @ w.astype(np.float64).T
    with np.errstate(invalid="ignore"):
        v = acc * s.astype(np.float64)[:, None] * c.astype(np.float64)
        d = 3.01 * U * np.abs(v) + 2.0 ** -148
        if b is not None:
            v = v + b.astype(np.float64)
            d = d + U * np.abs(v) * 1.01
        return act(v, kind), act_bound(v, d, kind)


def out_bound(y, d, elem):
    return d * (1 + OUT_U[elem]) + OUT_U[elem] * np.abs(y) + OUT_TINY[elem]


def scores(l, kind, ok):
    l = np.where(ok, l.astype(np.float64), -np.inf)
    with np.errstate(all="ignore"):
        if kind == 1:
            p = 1.0 / (1.0 + np.exp(-l))
        else:
            m = l.max(axis=1, keepdims=True)
            e = np.where(l == m, 1.0, np.exp(l - m))
            e = np.where(ok, e, 0.0)
            p = e / e.sum(axis=1, keepdims=True)
    return np.where(ok, p, 0.0)


def route(l, bias, rows, k, kind, groups, top_groups, group_top, renorm, scale):
    """(idx, weight, decided, p, c): `decided` marks rows whose order of values
    is told apart by more than 1e-5 of them, or by nothing at all (equal inputs)."""
    M, E = l.shape
    l = np.asarray(l, np.float32)
    ok = (l > -np.inf) & (np.ones(M, bool) if rows is None else rows != 0)[:, None]
    p = scores(l, kind, ok)
    with np.errstate(invalid="ignore"):
        c = p + (0.0 if bias is None else bias.astype(np.float64))
        c = np.where(ok & (c > -np.inf), c, -np.inf)

    def settled(v, first, last):
        """Ranks first..last told apart from the one after them."""
        v = -np.sort(-v, axis=1)[:, first:last + 2]
        with np.errstate(invalid="ignore"):
            gap = v[:, :-1] - v[:, 1:]
            near = (gap > 0) & (gap < 1e-5 * np.maximum(np.abs(v[:, :-1]), 1e-30)) & np.isfinite(v[:, 1:])
        return ~near.any(axis=1)

    decided = np.ones(M, bool)
    if groups > 1:
        s = -np.sort(-c.reshape(M, groups, -1), axis=2)[:, :, :group_top]
        v = np.where(s > -np.inf, s, 0.0).sum(axis=2)
        v = np.where(s[:, :, 0] > -np.inf, v, -np.inf)
        decided &= settled(v, top_groups - 1, top_groups - 1)  # which groups, not their order
        best = np.argsort(-v, axis=1, kind="stable")[:, :top_groups]
        keep = np.zeros((M, groups), bool)
        np.put_along_axis(keep, best, True, axis=1)
        c = np.where(np.repeat(keep, E // groups, axis=1), c, -np.inf)
    decided &= settled(c, 0, k - 1)
    idx = np.argsort(-c, axis=1, kind="stable")[:, :k]
    there = np.take_along_axis(c, idx, axis=1) > -np.inf
    w = np.where(there, np.take_along_axis(p, idx, axis=1), 0.0)
    if renorm:
        t = w.sum(axis=1, keepdims=True)
        w = np.where(t > 0, w / np.where(t > 0, t, 1.0), 0.0)
    return np.where(there, idx, -1).astype(np.int32), w * scale, decided


# exp: 2 roundings of its value and the rounding of l - max (at most 64 U of
# the result for |l - max| < 64); sums of E <= 1024 in any order; three
# quotients and products
def route_bound(E):
    return (2 + 64 + E / 16 + 6 + 6) * U


def experts(q, s, idx, wt, w1, s1, b1, w2, s2, b2, kind, gated):
    """(values, bound) before the output's rounding.  A value of the hidden row
    whose quotient lies within its own error of a rounding boundary may take
    either code: those places add one step of their code times their weight."""
    M, k = idx.shape
    E, H, _ = w1.shape
    F = H // 2 if gated else H
    N = w2.shape[1]
    y, d = np.zeros((M, N)), np.zeros((M, N))
    mag = np.zeros((M, N))
    for e in range(E):
        row, slot = np.nonzero(idx == e)
        if not len(row):
            continue
        if gated:
            g, dg = product(q[row], s[row], w1[e][:F], s1[e][:F], None if b1 is None else b1[e][:F], kind)
            u, du = product(q[row], s[row], w1[e][F:], s1[e][F:], None if b1 is None else b1[e][F:], NONE)
            h, dh = g * u, np.abs(g) * du + np.abs(u) * dg + dg * du + U * np.abs(g * u)
        else:
            h, dh = product(q[row], s[row], w1[e], s1[e], None if b1 is None else b1[e], kind)
        a = np.abs(h).max(axis=1, initial=0)
        ds = dh.max(axis=1, initial=0) / 127 + U * a / 127
        hs = (a / 127).astype(np.float32).astype(np.float64)
        t = h / np.where(hs > 0, hs, 1)[:, None]
        dt = (dh + np.abs(t) * ds[:, None]) / np.where(hs > 0, hs, 1)[:, None] + 2 * U * np.abs(t)
        hq = np.clip(np.rint(t), -127, 127)
        either = (np.abs(np.abs(t - np.floor(t)) - 0.5) <= dt).astype(np.float64)
        w, c = w2[e].astype(np.float64), s2[e].astype(np.float64)
        z = (hq @ w.T) * hs[:, None] * c
        dz = (either @ np.abs(w).T) * hs[:, None] * c + np.abs(hq @ w.T) * ds[:, None] * c + 4 * U * np.abs(z)
        if b2 is not None:
            z = z + b2[e]
            dz = dz + U * np.abs(z)
        ww = wt[row, slot].astype(np.float64)[:, None]
        np.add.at(y, row, ww * z)
        np.add.at(d, row, np.abs(ww) * dz)
        np.add.at(mag, row, np.abs(ww * z))
    return y, d * 1.01 + (k + 1) * U * mag, mag
