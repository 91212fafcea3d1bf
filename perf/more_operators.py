"""More operators of a head over a spiking trunk, as timed cases.

Three groups, with the calls of one case as a program makes them:

* ``mm`` and ``lin``: products of microscaled rows in 4 bits.  A block of 32
  neighbours of a row has a power of two as its scale and elements of the type
  e2m1.  ``mm`` takes activations in such blocks (``mx4_matmul``), ``lin`` floats
  or a spike map that the call quantises (``mx4_linear``).
* ``norm``: rows plus a residual, over their root mean square, as floats
  (``norm_rows``), or as codes for the product behind them: in 8 bits with a scale
  a row (``norm_quant``, then ``i8_matmul``), or in microscaled 4 bits
  (``norm_mx4``, then ``mx4_matmul``).
* ``moe`` and ``moe_grad``: rows to the order of their experts (``dispatch``) and
  the experts' results back, weighted and summed (``combine``); and the gradients
  of both (``combine_grad``, ``dispatch_grad``).

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is true, with the calls of this framework.  ``exact`` computes them in 64
bits from their definitions:

* block scale 2^X, X = floor(log2 max|x|) - 2 within [-127, 127]; elements x / 2^X
  rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6, half to even; of spike
  times, x = (T - bin) / T;
* product: y = act(sum(x w) + b);
* norm: h = x + r, u = h g, y = u / sqrt(mean(h^2) + eps); in 8 bits the codes of a
  row are those of u, and its scale max|u| / 127 over the root;
* dispatch: the pairs (row, slot) in the order of their experts, pairs of one
  expert in their own order; start of each expert, place of each pair, -1 where
  the slot has no expert; rows past the last pair stay as they are;
* combine: out = sum over slots of weight * z[place].
"""
from __future__ import annotations

import ctypes
import math
import os
import sys

import torch

own = False

ELEM = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16), "times": (3, torch.float32)}
ACT = {"none": 0, "relu": 1, "silu": 2}
NO_SPIKE = 9999.0


# ---- the cases ---------------------------------------------------------------
def listed():
    return [
        # one sample through a 4096 -> 4096 layer with 4-bit weights: latency
        {"name": "lin_row1", "op": "lin", "M": 1, "N": 4096, "K": 4096, "in": "bf16", "out": "bf16", "act": "none",
         "bias": False, "pad": 0},
        # a caller's own odd sizes and row strides
        {"name": "mm_ragged", "op": "mm", "M": 333, "N": 1111, "K": 1003, "out": "f32", "act": "relu", "bias": True,
         "pad": 3},
        # a large batch of the 4096 -> 4096 layer: the rate of the matrix units
        {"name": "mm_large", "op": "mm", "M": 8192, "N": 4096, "K": 4096, "out": "bf16", "act": "none", "bias": True,
         "pad": 0},
        # the same from floats
        {"name": "lin_large", "op": "lin", "M": 8192, "N": 4096, "K": 4096, "in": "bf16", "out": "bf16", "act": "none",
         "bias": False, "pad": 0},
        # one sample's features added to the residual and normalised: latency
        {"name": "norm_row1", "op": "norm", "M": 1, "K": 4096, "in": "bf16", "res": "bf16", "gain": True, "pad": 0,
         "out": "bf16", "N": 0, "eps": 1e-6},
        # a ragged batch, the residual in 32 bits, floats out
        {"name": "norm_ragged", "op": "norm", "M": 999, "K": 1001, "in": "f16", "res": "f32", "gain": True, "pad": 7,
         "out": "f16", "N": 0, "eps": 1e-5},
        # the largest batch of wide rows
        {"name": "norm_large", "op": "norm", "M": 16384, "K": 4096, "in": "bf16", "res": "bf16", "gain": True,
         "pad": 0, "out": "bf16", "N": 0, "eps": 1e-6},
        # normalised rows as the 8-bit codes that a router over 64 experts reads
        {"name": "norm_router", "op": "norm", "M": 8192, "K": 2048, "in": "bf16", "res": "bf16", "gain": True,
         "pad": 0, "out": "i8", "N": 64, "eps": 1e-6},
        # one sample to its six experts and back: latency
        {"name": "moe_row1", "op": "moe", "M": 1, "k": 6, "E": 64, "D": 1024, "N": 1024, "in": "bf16", "empty": 0},
        # a large batch to eight experts a row and back, some of the rows padding
        {"name": "moe_large", "op": "moe", "M": 16384, "k": 8, "E": 64, "D": 2048, "N": 2048, "in": "bf16",
         "empty": 5},
        # the gradients of a ragged batch in 32 bits
        {"name": "grad_ragged", "op": "moe_grad", "M": 777, "k": 3, "E": 10, "D": 501, "N": 333, "in": "f32",
         "empty": 3},
        # the gradients of the large batch
        {"name": "grad_large", "op": "moe_grad", "M": 16384, "k": 8, "E": 64, "D": 2048, "N": 2048, "in": "bf16",
         "empty": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["mm", "mm", "lin", "lin", "lin", "norm", "norm", "norm", "moe", "moe", "moe_grad", "moe_grad"])
    if op in ("mm", "lin"):
        c = {"op": op, "M": _log_int(rng, 1, 8192), "N": _log_int(rng, 10, 8192), "K": _log_int(rng, 16, 8192),
             "out": rng.choice(["f32", "bf16", "f16"]), "act": rng.choice(["none", "relu", "silu"]),
             "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 3, 16])}
        if rng.random() < 0.5:  # sizes of layers are often whole multiples
            c["N"], c["K"] = -(-c["N"] // 64) * 64, -(-c["K"] // 64) * 64
        c["M"] = max(1, min(c["M"], 2 ** 37 // (c["N"] * c["K"])))
        if op == "lin":
            c["in"] = rng.choice(["f32", "bf16", "f16", "times"])
            if c["in"] == "times":
                c["T"] = rng.choice([16, 32, 64, 80])
        return c
    if op == "norm":
        c = {"op": op, "M": _log_int(rng, 1, 16384), "K": _log_int(rng, 16, 8192),
             "in": rng.choice(["f32", "bf16", "f16"]), "res": rng.choice(["none", "f32", "bf16", "f16"]),
             "gain": rng.random() < 0.7, "pad": rng.choice([0, 0, 5, 16]),
             "out": rng.choice(["f32", "bf16", "f16", "i8", "i8", "mx4", "mx4"]), "N": 0,
             "eps": rng.choice([1e-6, 1e-5])}
        if rng.random() < 0.5:
            c["K"] = -(-c["K"] // 64) * 64
        c["M"] = max(1, min(c["M"], 2 ** 25 // c["K"]))
        if c["out"] in ("i8", "mx4"):
            c["N"] = _log_int(rng, 10, 512)
        return c
    c = {"op": op, "M": _log_int(rng, 1, 16384), "k": rng.randint(1, 8), "E": _log_int(rng, 8, 256),
         "D": _log_int(rng, 32, 4096), "N": _log_int(rng, 32, 4096), "in": rng.choice(["f32", "bf16", "f16"]),
         "empty": rng.choice([0, 2, 7])}
    if rng.random() < 0.5:
        c["D"], c["N"] = (-(-c[x] // 64) * 64 for x in "DN")
    c["M"] = max(1, min(c["M"], 2 ** 26 // (c["k"] * (c["D"] + c["N"]))))
    return c


# ---- inputs --------------------------------------------------------------------
class _Buf:
    """A torch tensor as the device buffer that the library's calls take."""

    def __init__(self, t):
        self.t, self.ptr, self.size = t, ctypes.c_void_p(t.data_ptr()), t.numel()


class _State:
    pass


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _new(dtype, *shape):
    return _Buf(torch.zeros(shape, dtype=dtype, device="cuda"))


def _floats(g, rows, cols, ld, dtype):
    """Activations: Gaussian, rows of different magnitude, one column in 61 eight times as large."""
    out = torch.zeros((rows, ld), dtype=dtype, device="cuda")
    x = _randn(g, rows, cols) * torch.exp(0.7 * _randn(g, rows, 1))
    x[:, 7::61] *= 8
    out[:, :cols] = x.to(dtype)
    return out


def _times(g, rows, cols, ld, T):
    """A spike map: whole times inside the window in half of the places, none in the others."""
    out = torch.full((rows, ld), NO_SPIKE, device="cuda")
    t = torch.floor(T * _rand(g, rows, cols))
    out[:, :cols] = torch.where(_rand(g, rows, cols) < 0.5, t, torch.full_like(t, NO_SPIKE))
    return out


def _code_bytes(K):
    return (K + 1) // 2


def _blocks(K):
    return (K + 31) // 32


def _pack(v):
    """Elements (their values over the block's scale), two a byte, the first in the low half."""
    a = v.abs()
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    c = c + 8 * (v < 0).to(torch.uint8)
    if c.shape[1] % 2:
        c = torch.nn.functional.pad(c, (0, 1))
    return c[:, 0::2] + 16 * c[:, 1::2]


def _mx_rows(g, rows, cols, pad, scale):
    """Rows of a microscaled matrix as a program holds them: codes and scales, each with a stride of its own."""
    v, e = _quant(_randn(g, rows, cols) * torch.exp(0.7 * _randn(g, rows, 1)) * scale)
    n, b = _code_bytes(cols), _blocks(cols)
    q = torch.zeros((rows, n + pad), dtype=torch.uint8, device="cuda")
    s = torch.zeros((rows, b + pad), dtype=torch.uint8, device="cuda")
    q[:, :n], s[:, :b] = _pack(v), (e + 127).to(torch.uint8)
    return _Buf(q), _Buf(s)


def _choose(g, M, E, k, empty):
    """The experts of each row, as routing leaves them: distinct, some asked for more often, largest weight first."""
    wt, idx = torch.sort(torch.softmax(_randn(g, M, E) + 0.5 * _randn(g, 1, E), 1), dim=1, descending=True)
    wt, idx = wt[:, :k], idx[:, :k].to(torch.int32)
    if empty:  # padding rows have none, and some rows fewer than k
        wt = torch.where(_rand(g, M, 1) * empty < 0.2, torch.zeros_like(wt), wt)
        wt[1::7, k // 2:] = 0
        idx = torch.where(wt > 0, idx, torch.full_like(idx, -1))
    return idx.contiguous(), (wt / wt.sum(1, keepdim=True).clamp_min(1e-20)).contiguous()


def prepare(case, seed):
    g, s = _gen(seed), _State()
    s.case, op = case, case["op"]
    if op in ("mm", "lin"):
        M, N, K, pad = case["M"], case["N"], case["K"], case["pad"]
        if op == "mm":
            s.q, s.s = _mx_rows(g, M, K, pad, 1.0)
        else:
            s.ldx = K + pad
            s.x = _Buf(_times(g, M, K, s.ldx, case["T"]) if case["in"] == "times"
                       else _floats(g, M, K, s.ldx, ELEM[case["in"]][1]))
        s.w, s.ws = _mx_rows(g, N, K, pad, 1 / math.sqrt(K))
        s.bias = _Buf(0.3 * _randn(g, N)) if case["bias"] else None
        s.out = _new(ELEM[case["out"]][1], M, N)
    elif op == "norm":
        M, K, N, out, s.ld = case["M"], case["K"], case["N"], case["out"], case["K"] + case["pad"]
        s.x = _Buf(_floats(g, M, K, s.ld, ELEM[case["in"]][1]))
        s.res = s.sum = None
        if case["res"] != "none":
            s.res = _Buf(_floats(g, M, K, s.ld, ELEM[case["res"]][1]))
            s.sum = _new(ELEM[case["res"]][1], M, K)
        s.gain = _Buf(1 + 0.2 * _randn(g, K)) if case["gain"] else None
        if out in ELEM:
            s.y = _new(ELEM[out][1], M, K)
            return s
        if out == "i8":
            s.q, s.s, s.out = _new(torch.int8, M, K), _new(torch.float32, M), _new(torch.float32, M, N)
            w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int32)
            s.w, s.ws = _Buf(w.to(torch.int8)), _Buf((0.5 + _rand(g, N)) / (74 * math.sqrt(K)))
        else:
            s.q, s.s = _new(torch.uint8, M, _code_bytes(K)), _new(torch.uint8, M, _blocks(K))
            s.w, s.ws = _mx_rows(g, N, K, 0, 1 / math.sqrt(K))
            s.out = _new(torch.bfloat16, M, N)
    else:
        M, k, E, D, N, dtype = case["M"], case["k"], case["E"], case["D"], case["N"], ELEM[case["in"]][1]
        idx, wt = _choose(g, M, E, k, case["empty"])
        s.idx, s.wt = _Buf(idx), _Buf(wt)
        s.z = _Buf(_randn(g, M * k, N).to(dtype))
        if op == "moe":
            s.x = _Buf(_floats(g, M, D, D, dtype))
            s.place, s.start = _new(torch.int32, M, k), _new(torch.int32, E + 1)
            s.sorted, s.out = _new(dtype, M * k, D), _new(dtype, M, N)
        else:  # the forward's places, the gradient of its output and of the sorted rows
            s.place = _Buf(_places(idx, E)[0].contiguous())
            s.dout, s.dsorted = _Buf(_randn(g, M, N).to(dtype)), _Buf(_randn(g, M * k, D).to(dtype))
            s.dz, s.dwt, s.dx = _new(dtype, M * k, N), _new(torch.float32, M, k), _new(dtype, M, D)
    return s


# ---- one pass ------------------------------------------------------------------
_contexts = {}


def _context(T):
    """The program's context for a window of T steps (spike maps only depend on it)."""
    if T not in _contexts:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vd-ttfs_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import vdttfs
        _contexts[T] = vdttfs.Context(vdttfs.TaskConsts(T=T, delta=16))
    return _contexts[T]


def _run_own(s):
    case, op = s.case, s.case["op"]
    ctx = _context(case.get("T", 64))
    if op == "mm":
        ctx.mx4_matmul(s.out, ELEM[case["out"]][0], case["N"], s.q, s.q.t.shape[1], s.s, s.s.t.shape[1], s.w,
                       s.w.t.shape[1], s.ws, s.ws.t.shape[1], s.bias, ACT[case["act"]], case["M"], case["N"],
                       case["K"])
        return s.out.t
    if op == "lin":
        ctx.mx4_linear(s.out, ELEM[case["out"]][0], case["N"], s.x, ELEM[case["in"]][0], s.ldx, s.w, s.w.t.shape[1],
                       s.ws, s.ws.t.shape[1], s.bias, ACT[case["act"]], case["M"], case["N"], case["K"])
        return s.out.t
    if op == "norm":
        M, K, N, out = case["M"], case["K"], case["N"], case["out"]
        rows = (s.x, ELEM[case["in"]][0], s.ld, s.res, ELEM[case["res"]][0] if s.res else 0, s.ld, s.sum, K, s.gain,
                case["eps"], M, K)
        if out in ELEM:
            ctx.norm_rows(s.y, ELEM[out][0], K, *rows)
            return _answer(s, y=s.y.t)
        q = s.q.t.shape[1]
        if out == "i8":
            ctx.norm_quant(s.q, q, s.s, *rows)
            ctx.i8_matmul(s.out, 0, N, s.q, q, s.s, s.w, K, s.ws, None, 0, M, N, K)
        else:
            b = s.s.t.shape[1]
            ctx.norm_mx4(s.q, q, s.s, b, *rows)
            ctx.mx4_matmul(s.out, 1, N, s.q, q, s.s, b, s.w, s.w.t.shape[1], s.ws, s.ws.t.shape[1], None, 0, M, N, K)
        return _answer(s, out=s.out.t)
    M, k, D, N, elem = case["M"], case["k"], case["D"], case["N"], ELEM[case["in"]][0]
    if op == "moe":
        ctx.dispatch(s.sorted, D, s.place, s.start, s.x, elem, D, s.idx, M, k, case["E"], D)
        ctx.combine(s.out, elem, N, s.z, elem, N, s.place, s.wt, M, k, N)
        return {"sorted": s.sorted.t, "place": s.place.t, "start": s.start.t, "out": s.out.t}
    ctx.combine_grad(s.dz, N, s.dwt, s.z, elem, N, s.dout, elem, N, s.place, s.wt, M, k, N)
    ctx.dispatch_grad(s.dx, elem, D, s.dsorted, D, s.place, M, k, D)
    return {"dz": s.dz.t, "dweight": s.dwt.t, "dx": s.dx.t}


def _answer(s, **out):
    return {**out, "sum": s.sum.t} if s.sum is not None else out


def _act(v, act):
    return torch.clamp_min(v, 0) if act == "relu" else v / (1 + torch.exp(-v)) if act == "silu" else v


def _in_blocks(x):
    """[rows][K] as [rows][blocks][32], zeros behind the last element."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)


def _round_elements(t):
    """To the nearest element, half to even, no further than the largest; |t| is below 8."""
    a = t.abs()
    r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    return torch.copysign(torch.clamp_max(r, 6), t)


def _scaled(x, e):
    """x * 2^e by the power's own bits (exp2 and pow of a GPU may miss it by the last one), |e| <= 127."""
    return x * ((e.long() + 1023) << 52).view(torch.float64).to(x.dtype)


def _quant(x):
    """Elements over their scale [rows][K] and the scales' exponents [rows][blocks] of 32-bit rows."""
    b = _in_blocks(x)
    a = b.abs().amax(2)
    e = torch.frexp(a)[1] - 3
    e = torch.where(a > 0, e.clamp(-127, 127), -127)
    t = _scaled(b, -e[:, :, None])
    return _round_elements(t).view(x.shape[0], -1)[:, :x.shape[1]], e


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(q, s, K):
    """What codes and scales stand for, [rows][K] in 32 bits."""
    q, s = q[:, :_code_bytes(K)], s[:, :_blocks(K)]
    pairs = torch.stack((q & 15, q >> 4), 2).view(q.shape[0], -1)
    v = torch.tensor(_E2M1, device=q.device)[pairs.int()][:, :K]
    return _scaled(_in_blocks(v), (s.int() - 127)[:, :, None]).view(q.shape[0], -1)[:, :K]


def _product(x, w, bias, act):
    y = x @ w.t()
    return _act(y if bias is None else y + bias.t, act)


def _plain_lin(s, case):
    K = case["K"]
    if case["op"] == "mm":
        x = _values(s.q.t, s.s.t, K)
    else:
        x = s.x.t[:, :K]
        if case["in"] == "times":
            x = torch.where(x < case["T"], case["T"] - torch.floor(x), 0) / case["T"]
        v, e = _quant(x.float())
        x = _scaled(_in_blocks(v), e[:, :, None]).view(x.shape[0], -1)[:, :K]
    return _product(x, _values(s.w.t, s.ws.t, K), s.bias, case["act"]).to(ELEM[case["out"]][1])


def _plain_norm(s, case):
    K, out = case["K"], case["out"]
    h = s.x.t[:, :K].float()
    if s.res is not None:
        h = h + s.res.t[:, :K].float()
        s.sum.t.copy_(h)
    root = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + case["eps"])
    u = h if s.gain is None else h * s.gain.t
    if out == "i8":
        a = u.abs().amax(1, keepdim=True)
        sc = a / torch.full_like(a, 127)
        q = torch.where(sc > 0, torch.round(u / sc), 0).clamp(-127, 127)
        return _answer(s, out=(q @ s.w.t.float().t()) * (sc * root) * s.ws.t)
    y = u * root
    if out in ELEM:
        return _answer(s, y=y.to(ELEM[out][1]))
    v, e = _quant(y)
    x = _scaled(_in_blocks(v), e[:, :, None]).view(v.shape[0], -1)[:, :K]
    return _answer(s, out=(x @ _values(s.w.t, s.ws.t, K).t()).to(torch.bfloat16))


def _places(idx, E):
    """Places of the pairs, the pairs in sorted order, the experts' starts."""
    e = idx.reshape(-1)
    e = torch.where((e >= 0) & (e < E), e, E)
    order = torch.sort(e, stable=True)[1]
    place = torch.empty_like(e)
    place[order] = torch.arange(e.numel(), dtype=torch.int32, device=e.device)
    count = torch.zeros(E + 1, dtype=torch.int32, device=e.device)
    count.scatter_add_(0, e.long(), torch.ones_like(e))
    start = (torch.cumsum(count, 0) - count).to(torch.int32)
    return torch.where(e < E, place, -1).view(idx.shape), order, start


def _plain_moe(s, case):
    M, k, dtype = case["M"], case["k"], ELEM[case["in"]][1]
    place, order, start = _places(s.idx.t, case["E"])
    there = torch.arange(M * k, device=place.device) < start[-1]
    rows = torch.where(there[:, None], s.x.t[order // k], 0)
    z = s.z.t[place.clamp_min(0).reshape(-1)].float().view(M, k, -1)
    w = torch.where(place >= 0, s.wt.t, 0)
    return {"sorted": rows, "place": place, "start": start, "out": (z * w[:, :, None]).sum(1).to(dtype)}


def _plain_grad(s, case):
    M, k, dtype = case["M"], case["k"], ELEM[case["in"]][1]
    on, at = s.place.t >= 0, s.place.t.clamp_min(0).reshape(-1).long()
    d = s.dout.t.float()
    dw = torch.where(on, (s.z.t[at].float().view(M, k, -1) * d[:, None]).sum(2), 0)
    pair = torch.full((M * k + 1,), -1, dtype=torch.long, device=at.device)  # the last place takes pairs without one
    pair[torch.where(on.reshape(-1), at, M * k)] = torch.arange(M * k, device=at.device)
    pair = pair[:-1]
    dz = torch.where(pair[:, None] >= 0, d[pair.clamp_min(0) // k] * s.wt.t.reshape(-1)[pair.clamp_min(0)][:, None], 0)
    dx = torch.where(on[:, :, None], s.dsorted.t[at].float().view(M, k, -1), 0).sum(1)
    return {"dz": dz.to(dtype), "dweight": dw, "dx": dx.to(dtype)}


def _run_plain(s):
    case, op = s.case, s.case["op"]
    if op in ("mm", "lin"):
        return _plain_lin(s, case)
    return {"norm": _plain_norm, "moe": _plain_moe, "moe_grad": _plain_grad}[op](s, case)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------
def _two64(e):
    """2^e for whole e, by table."""
    return torch.tensor([2.0 ** i for i in range(-260, 261)], dtype=torch.float64, device=e.device)[e.long() + 260]


def _element64(t):
    """Rounded to the type's step at each value: a half below 2, half of its binade's lower end above."""
    e = torch.clamp_min(torch.frexp(t)[1] - 1, 0) - 1  # frexp(0) is 0
    return (torch.round(t * _two64(-e)) * _two64(e)).clamp(-6, 6)


def _codes64(x):
    """What the codes of x stand for, by definition."""
    rows, K = x.shape
    parts = [x[:, i::32] for i in range(32)]
    a = torch.zeros((rows, _blocks(K)), dtype=torch.float64, device=x.device)
    for p in parts:
        a[:, :p.shape[1]] = torch.maximum(a[:, :p.shape[1]], p.abs())
    X = torch.floor(torch.log2(a.clamp_min(2.0 ** -200))).to(torch.int32)
    X = X + (_two64(X + 1) <= a).to(torch.int32) - (_two64(X) > a).to(torch.int32)
    X = torch.clamp(X - 2, -127, 127)
    scale = _two64(X).repeat_interleave(32, 1)[:, :K]
    return _element64(x / scale) * scale


def _decode64(q, s, K):
    c = torch.empty((q.shape[0], 2 * _code_bytes(K)), dtype=torch.int32, device=q.device)
    b = q[:, :_code_bytes(K)].int()
    c[:, 0::2], c[:, 1::2] = b % 16, b // 16
    m, e, sign = c % 2, c // 2 % 4, 1 - 2 * (c // 8)
    v = torch.where(e > 0, 1 + m.double() / 2, m.double() / 2)
    v = (sign * v * _two64(torch.clamp_min(e, 1) - 1))[:, :K]
    return v * _two64(s[:, :_blocks(K)].int() - 127).repeat_interleave(32, 1)[:, :K]


def _act64(v, act):
    return v.clamp(min=0) if act == "relu" else v * torch.sigmoid(v) if act == "silu" else v


def _exact_norm(s, case):
    K, out = case["K"], case["out"]
    h = s.x.t[:, :K].double()
    if s.res is not None:
        h = h + s.res.t[:, :K].double()
    root = torch.rsqrt(h.square().sum(1, keepdim=True) / K + case["eps"])
    u = h if s.gain is None else h * s.gain.t.double()
    more = {} if s.res is None else {"sum": h}
    if out in ELEM:
        return {"y": u * root, **more}
    if out == "i8":  # the sums and products before the codes are the definition's own 32-bit ones
        u = h.float() if s.gain is None else h.float() * s.gain.t
        sc = (u.double().abs().max(dim=1, keepdim=True)[0] / 127).float().double()
        q = torch.round((u.double() / sc).float().double()).clamp(-127, 127)
        return {"out": torch.mm(q, s.w.t.double().t().contiguous()) * sc * root * s.ws.t.double(), **more}
    return {"out": torch.mm(_codes64(u * root), _decode64(s.w.t, s.ws.t, K).t().contiguous()), **more}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("mm", "lin"):
        K = case["K"]
        if op == "mm":
            x = _decode64(s.q.t, s.s.t, K)
        else:
            x = s.x.t[:, :K].double()
            if case["in"] == "times":
                b = torch.floor(x)
                x = (torch.where(b < case["T"], case["T"] - b, torch.zeros_like(b)) / case["T"]).float().double()
            x = _codes64(x)
        y = torch.mm(x, _decode64(s.w.t, s.ws.t, K).t().contiguous())
        return _act64(y if s.bias is None else y + s.bias.t.double(), case["act"])
    if op == "norm":
        return _exact_norm(s, case)
    M, k, N = case["M"], case["k"], case["N"]
    if op == "moe":
        D, E = case["D"], case["E"]
        place = torch.full((M * k,), -1, dtype=torch.int32, device="cuda")
        rows = torch.zeros((M * k, D), dtype=torch.float64, device="cuda")
        out = torch.zeros((M, N), dtype=torch.float64, device="cuda")
        start, at = [], 0
        for e in range(E):
            start.append(at)
            row, slot = torch.nonzero(s.idx.t == e, as_tuple=True)  # in the order of pairs
            n = row.numel()
            place[row * k + slot] = torch.arange(at, at + n, dtype=torch.int32, device="cuda")
            rows[at:at + n] = s.x.t[row].double()
            out.index_add_(0, row, s.z.t[at:at + n].double() * s.wt.t[row, slot].double()[:, None])
            at += n
        start = torch.tensor(start + [at], dtype=torch.int32, device="cuda")
        return {"sorted": rows, "place": place.view(M, k), "start": start, "out": out}
    dz = torch.zeros((M * k, N), dtype=torch.float64, device="cuda")
    dw = torch.zeros((M, k), dtype=torch.float64, device="cuda")
    dx = torch.zeros((M, case["D"]), dtype=torch.float64, device="cuda")
    for j in range(k):
        row = torch.nonzero(s.place.t[:, j] >= 0)[:, 0]
        at = s.place.t[row, j].long()
        dz[at] = s.dout.t[row].double() * s.wt.t[row, j].double()[:, None]
        dw[row, j] = (s.dout.t[row].double() * s.z.t[at].double()).sum(1)
        dx[row] += s.dsorted.t[at].double()
    return {"dz": dz, "dweight": dw, "dx": dx}


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "times": 4}
    op, M = case["op"], case["M"]

    def codes(K, out="mx4"):
        return K + 4 if out == "i8" else _code_bytes(K) + _blocks(K)

    if op in ("mm", "lin"):
        N, K = case["N"], case["K"]
        row = codes(K) if op == "mm" else K * size[case["in"]]
        return {"bytes": M * row + N * (codes(K) + (4 if case["bias"] else 0)) + M * N * size[case["out"]],
                "flops": 2 * M * N * K}
    if op == "norm":
        K, N, out = case["K"], case["N"], case["out"]
        n = M * K * (size[case["in"]] + (0 if case["res"] == "none" else 2 * size[case["res"]]))
        n += 4 * K if case["gain"] else 0
        if N:  # codes in between are not counted
            return {"bytes": n + N * codes(K, out) + M * N * (4 if out == "i8" else 2), "flops": 2 * M * N * K}
        return {"bytes": n + M * K * size[out], "flops": 6 * M * K}
    k, D, N, one = case["k"], case["D"], case["N"], size[case["in"]]
    pairs = M * k * (0.8 if case["empty"] else 1)  # those with an expert, about
    if op == "moe":
        return {"bytes": one * (M * D + pairs * D + pairs * N + M * N) + 12 * M * k + 4 * case["E"],
                "flops": 2 * pairs * N}
    return {"bytes": one * (pairs * (2 * N + D) + M * (N + D)) + 12 * M * k, "flops": pairs * (3 * N + D)}
