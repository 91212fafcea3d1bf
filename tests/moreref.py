"""The heads' other operators from their definitions, in 64 bits with numpy, and
how far a correct 32-bit evaluation may be from them (see headref for U and the
rounding of outputs)."""
import numpy as np

from headref import NONE, U, act, act_bound  # noqa: F401

BLOCK = 32
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


# ---- microscaled rows -----------------------------------------------------------
def in_blocks(x):
    """[rows][cols] as [rows][blocks][32], zeros behind the last."""
    rows, cols = x.shape
    out = np.zeros((rows, -(-cols // BLOCK), BLOCK), x.dtype)
    out.reshape(rows, -1)[:, :cols] = x
    return out


def mx4_round(t):
    """Element codes of values, 64 bits, half to even, no further than 6."""
    a = np.abs(t)
    i = np.where(a < 2, np.rint(a * 2), np.where(a < 4, np.rint(a) + 2, np.rint(a / 2) + 4))
    return (np.minimum(i, 7) + np.where(np.signbit(t), 8, 0)).astype(np.uint8)


def mx4_quant(x):
    """Element codes [rows][cols] and scale bytes [rows][blocks] of float rows."""
    x = np.asarray(x, np.float64)
    b = in_blocks(x)
    with np.errstate(all="ignore"):
        a = np.abs(b).max(axis=2)
        bad = ~np.isfinite(a)
        X = np.clip(np.frexp(np.where(bad | (a == 0), 1.0, a))[1] - 1 - 2, -127, 127)
        X = np.where(a == 0, -127, X)
        c = mx4_round(np.where(bad[:, :, None], 0.0, b) * np.exp2(-X.astype(np.float64))[:, :, None])
    c = np.where(bad[:, :, None], 0, c).reshape(len(x), -1)[:, :x.shape[1]]
    return c.astype(np.uint8), np.where(bad, 255, X + 127).astype(np.uint8)


def mx4_pack(c):
    """Codes two a byte, the first in the low half."""
    if c.shape[1] % 2:
        c = np.concatenate([c, np.zeros((len(c), 1), np.uint8)], axis=1)
    return (c[:, 0::2] | c[:, 1::2] << 4).astype(np.uint8)


def mx4_unpack(q, cols):
    return np.stack([q & 15, q >> 4], axis=2).reshape(len(q), -1)[:, :cols]


def mx4_values(c, s):
    """What codes and scale bytes stand for."""
    v = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return (in_blocks(E2M1[c]) * v[:, :, None]).reshape(len(c), -1)[:, :c.shape[1]]


def mx4_times(t, T, tfs):
    """The value of a spike time: its linear encoding's pixel, in 32 bits."""
    t = np.asarray(t, np.float32)
    with np.errstate(all="ignore"):
        b = np.floor((t - np.float32(tfs)).astype(np.float64))
    b = np.where(b < 0, 0, b)
    hit = (t < 9999.0) & (b < T)
    return np.where(hit, (T - np.where(hit, b, 0)).astype(np.float32) / np.float32(T), np.float32(0))


def mx4_product(x, w, b, kind):
    """(values, bound) of decoded operands.  A block's sum is exact; what is left are
    the additions over blocks and over the parts of a split sum, at most 16, each
    within 2 U (a truncation) of the magnitudes so far."""
    n = -(-x.shape[1] // BLOCK) + 16
    with np.errstate(invalid="ignore", over="ignore"):
        v = x @ w.T
        d = 2 * U * n * (np.abs(x) @ np.abs(w).T) + 2.0 ** -148
        if b is not None:
            v = v + b.astype(np.float64)
            d = d + U * np.abs(v) * 1.01
        return act(v, kind), act_bound(v, d, kind)


# ---- norms ------------------------------------------------------------------------
# A row's squares are added in at most 64 roundings one after another (32 of a
# lane, six levels of a wave, sixteen waves), half of which the root keeps; the
# mean, eps, the root, its reciprocal and the product round once each, as does a
# square.
NORM_U = (64 / 2 + 8) * U


def norm(x, res, gain, eps):
    """(h, u, root, y): h and u are 32-bit floats by definition, root and y in 64."""
    with np.errstate(all="ignore"):
        h = x.astype(np.float32) if res is None else x.astype(np.float32) + res.astype(np.float32)
        u = h if gain is None else h * gain.astype(np.float32)
        mean = (h.astype(np.float64) ** 2).mean(axis=1, keepdims=True)
        root = np.sqrt(mean + np.float64(np.float32(eps)))
        inv = np.where(root > 0, 1.0 / np.where(root > 0, root, 1.0), 0.0)
        inv = np.where(np.isnan(root), np.nan, inv)
        return h, u, inv, u.astype(np.float64) * inv


# ---- rows by expert -----------------------------------------------------------------
def places(idx, E):
    """(place [M][k], start [E + 1]) of the stable order by expert."""
    e = idx.reshape(-1)
    on = (e >= 0) & (e < E)
    order = np.argsort(np.where(on, e, E), kind="stable")[:on.sum()]
    place = np.full(e.size, -1, np.int32)
    place[order] = np.arange(order.size)
    start = np.concatenate([[0], np.cumsum(np.bincount(e[on], minlength=E))]).astype(np.int32)
    return place.reshape(idx.shape), start


def combine(z, place, wt):
    """(values, bound): the products and the sum in the order of the slots, one rounding each."""
    M, k = place.shape
    y, mag = np.zeros((M, z.shape[1])), np.zeros((M, z.shape[1]))
    for j in range(k):
        on = place[:, j] >= 0
        w = np.ones(on.sum()) if wt is None else wt[on, j].astype(np.float64)
        t = w[:, None] * z[place[on, j]].astype(np.float64)
        y[on] += t
        mag[on] += np.abs(t)
    return y, (k + 1) * U * 1.01 * mag + 2.0 ** -148


def combine_grad(z, place, wt, dout):
    """(dz, dw, bound of dw): a lane adds up to 8 (cols / 512 + 1) terms, 12 levels add lanes and waves."""
    M, k = place.shape
    d = dout.astype(np.float64)
    dz, dw, mag = np.zeros(z.shape), np.zeros((M, k)), np.zeros((M, k))
    for j in range(k):
        on = place[:, j] >= 0
        at = place[on, j]
        dz[at] = d[on] if wt is None else wt[on, j].astype(np.float64)[:, None] * d[on]
        t = d[on] * z[at].astype(np.float64)
        dw[on, j], mag[on, j] = t.sum(axis=1), np.abs(t).sum(axis=1)
    return dz, dw, (8 * (z.shape[1] / 512 + 1) + 12) * U * 1.01 * mag + 2.0 ** -148
