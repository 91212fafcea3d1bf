"""The operators of a dense or conditional head over a spiking trunk, as timed cases.

Four operators: the product of 8-bit codes with a scale for each row and each
output channel (``i8_matmul``), the same with the rows quantised in the call
from floats or from a spike map (``i8_linear``), routing of rows to experts
(``route``) and the experts' products (``experts``).  ``run`` computes them
with elementary torch operations in 32 bits, or, where ``own`` is true, with
the calls of this framework.  ``exact`` computes them in 64 bits from their
definitions:

* codes of a row x: s = max|x| / 127 held in 32 bits, q = the 32-bit quotient
  x / s rounded to the nearest whole number (half to even);
* codes of spike times: T - bin (bin = floor(t) within a window of T <= 127
  steps, 0 without a spike), s = 1 / T;
* product: y = act(sum(q w) * s * c + b);
* routing: scores p by softmax or sigmoid over the experts whose logit is
  above -inf, chosen by p + bias (inside the best groups, if any) largest
  first and ties to the lowest index, -1 where none is left; weights p,
  renormalised to sum to one if asked for, times a factor;
* experts: h = act(u) or act(gate) * up of the first product, h quantised by
  row, the second product, and the sum over a row's experts by weight.
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
        # one row through a 4096 -> 4096 layer (the size of the FC sweep): the latency of a single sample
        {"name": "mm_row1", "op": "mm", "M": 1, "N": 4096, "K": 4096, "out": "bf16", "act": "none", "bias": False,
         "pad": 0},
        # a caller's own odd sizes and row strides
        {"name": "mm_ragged", "op": "mm", "M": 333, "N": 1111, "K": 1003, "out": "f32", "act": "relu", "bias": True,
         "pad": 5},
        # a large batch of the same layer: the rate of the matrix units
        {"name": "mm_large", "op": "mm", "M": 8192, "N": 4096, "K": 4096, "out": "bf16", "act": "none", "bias": True,
         "pad": 0},
        # the dense twin of VGG-16's first FC layer over the spike map of a batch of 256
        {"name": "lin_spikes_b256", "op": "lin", "M": 256, "N": 512, "K": 512, "in": "times", "out": "f32",
         "act": "relu", "bias": True, "pad": 0, "T": 64},
        # a few samples in flight
        {"name": "lin_rows5", "op": "lin", "M": 5, "N": 4096, "K": 4096, "in": "f16", "out": "f16", "act": "silu",
         "bias": True, "pad": 0},
        # the largest batch in floats
        {"name": "lin_large", "op": "lin", "M": 8192, "N": 4096, "K": 4096, "in": "bf16", "out": "bf16", "act": "none",
         "bias": False, "pad": 0},
        # one sample routed: launch latency
        {"name": "route_row1", "op": "route", "M": 1, "E": 64, "k": 6, "in": "f32", "score": "softmax", "groups": 1,
         "top_groups": 1, "group_top": 1, "bias": False, "renorm": True, "scale": 1.0, "masked": False},
        # a ragged batch with padding rows and experts out of reach
        {"name": "route_ragged", "op": "route", "M": 1999, "E": 60, "k": 4, "in": "f16", "score": "softmax",
         "groups": 1, "top_groups": 1, "group_top": 1, "bias": True, "renorm": False, "scale": 2.5, "masked": True},
        # many rows, balanced by a bias and limited to half of the groups
        {"name": "route_large", "op": "route", "M": 65536, "E": 256, "k": 8, "in": "bf16", "score": "sigmoid",
         "groups": 8, "top_groups": 4, "group_top": 2, "bias": True, "renorm": True, "scale": 2.5, "masked": True},
        # one sample through its six experts
        {"name": "exp_row1", "op": "exp", "M": 1, "k": 6, "E": 64, "D": 1024, "F": 512, "N": 1024, "in": "bf16",
         "out": "bf16", "act": "silu", "gated": True, "bias": False, "empty": 0},
        # a class head of eight experts over VGG-16's 512 features, from their spike map, batch 256
        {"name": "exp_spikes_b256", "op": "exp", "M": 256, "k": 2, "E": 8, "D": 512, "F": 512, "N": 10, "in": "times",
         "out": "f32", "act": "relu", "gated": False, "bias": True, "empty": 3, "T": 64},
        # a wide expert layer on a large batch, some of the rows padding
        {"name": "exp_large", "op": "exp", "M": 8192, "k": 8, "E": 64, "D": 2048, "F": 1024, "N": 2048, "in": "bf16",
         "out": "bf16", "act": "silu", "gated": True, "bias": False, "empty": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["mm", "mm", "lin", "lin", "lin", "route", "route", "exp", "exp", "exp"])
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
    if op == "route":
        per = rng.choice([1, 4, 6, 8, 16, 32])  # experts in a group
        groups = 1 if per == 1 else rng.choice([g for g in (2, 4, 8) if g * per <= 256])
        E = _log_int(rng, 4, 256) if per == 1 else groups * per
        top = rng.randint(1, groups)
        return {"op": op, "M": _log_int(rng, 1, 65536), "E": E, "k": rng.randint(1, min(8, top * (E // groups))),
                "in": rng.choice(["f32", "bf16", "f16"]), "score": rng.choice(["softmax", "sigmoid"]),
                "groups": groups, "top_groups": top, "group_top": min(2, E // groups) if rng.random() < 0.5 else 1,
                "bias": rng.random() < 0.6, "renorm": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]),
                "masked": rng.random() < 0.5}
    c = {"op": op, "M": _log_int(rng, 1, 8192), "k": rng.randint(1, 8), "E": _log_int(rng, 8, 128),
         "D": _log_int(rng, 64, 2048), "F": _log_int(rng, 32, 2048), "N": _log_int(rng, 10, 2048),
         "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "act": rng.choice(["relu", "silu"]),
         "gated": rng.random() < 0.5, "bias": rng.random() < 0.5, "empty": rng.choice([0, 2, 7])}
    if rng.random() < 0.5:
        c["D"], c["F"], c["N"] = (-(-c[x] // 64) * 64 for x in "DFN")
    c["in"] = c["out"]
    if c["out"] == "f32":
        # h is quantised again, so its last bit can be another code: up to 1040
        # terms of code products every order of a 32-bit sum gives the same h
        c.update(D=min(c["D"], 1024), act="relu", **{"in": rng.choice(["f32", "times"])})
        if c["in"] == "times":
            c["T"] = rng.choice([16, 32, 64, 80])
    both = c["F"] * (c["D"] * (2 if c["gated"] else 1) + c["N"])
    c["E"] = max(8, min(c["E"], 2 ** 29 // both))
    c["M"] = max(1, min(c["M"], 2 ** 38 // (both * c["k"])))
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


def _codes(g, rows, cols, ld):
    """Codes of Gaussian rows, the largest of a row near the end of the range."""
    out = torch.zeros((rows, ld), dtype=torch.int8, device="cuda")
    out[:, :cols] = (_randn(g, rows, cols) * (127 / 4)).round().clamp(-127, 127).to(torch.int8)
    return out


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


def _inputs(case, g, cols, ld):
    if case["in"] == "times":
        return _times(g, case["M"], cols, ld, case["T"])
    return _floats(g, case["M"], cols, ld, ELEM[case["in"]][1])


def _choice64(case, logits, bias):
    """Scores and choice values in 64 bits; -inf where an expert cannot be chosen."""
    l = logits.double()
    p = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l)
    p = torch.nan_to_num(p)  # a row without an expert
    c = p if bias is None else p + bias.double()
    return p, torch.where(l > -math.inf, c, torch.full_like(c, -math.inf))


def _groups64(case, c):
    """The group values, and the choice values inside the groups that are kept."""
    M, E = c.shape
    v = torch.sort(c.view(M, case["groups"], -1), dim=2, descending=True)[0][:, :, :case["group_top"]]
    any_ = v[:, :, :1] > -math.inf
    v = torch.where(v > -math.inf, v, torch.zeros_like(v)).sum(2, keepdim=True)
    v = torch.where(any_, v, torch.full_like(v, -math.inf))[:, :, 0]
    best = torch.sort(v, dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
    keep = torch.zeros_like(v, dtype=torch.bool).scatter_(1, best, True)
    keep = keep[:, :, None].expand(-1, -1, E // case["groups"]).reshape(M, E)
    return v, torch.where(keep, c, torch.full_like(c, -math.inf))


def _undecided(case, logits, bias):
    """Rows where the choice hangs on the last bits of 32: unequal neighbours within 1e-5."""
    def near(v, n):
        v = torch.sort(v, dim=1, descending=True)[0][:, :n + 1]
        gap = v[:, :-1] - v[:, 1:]
        return ((gap > 0) & (gap < 1e-5 * v[:, :-1].abs())).any(1)

    _, c = _choice64(case, logits, bias)
    bad = torch.zeros(c.shape[0], dtype=torch.bool, device=c.device)
    if case["groups"] > 1:
        v, kept = _groups64(case, c)
        bad, c = near(v, case["groups"]), kept
    return bad | near(c, case["k"])


def _logits(case, g, bias):
    """Router logits; with "masked", an expert in 17 of some rows at -inf, and rows with none left."""
    M, E, dtype = case["M"], case["E"], ELEM[case["in"]][1]

    def some():
        l = 1.5 * _randn(g, M, E)
        if case["masked"]:
            l = torch.where(_rand(g, M, E) < 1 / 17, torch.full_like(l, -math.inf), l)
            l = torch.where(_rand(g, M, 1) < 1 / 50, torch.full_like(l, -math.inf), l)
        return l.to(dtype)

    l = some()
    for _ in range(4):
        l = torch.where(_undecided(case, l, bias)[:, None], some(), l)
    return l.contiguous()


def prepare(case, seed):
    g, s = _gen(seed), _State()
    s.case, op = case, case["op"]
    if op in ("mm", "lin"):
        M, N, K = case["M"], case["N"], case["K"]
        ld = K + case["pad"]
        if op == "mm":
            s.x = _Buf(_codes(g, M, K, ld))
            s.row_scale = _Buf((torch.exp(0.7 * _randn(g, M)) * (4 / 127)).contiguous())
        else:
            s.x = _Buf(_inputs(case, g, K, ld))
        s.w = _Buf(_codes(g, N, K, ld))
        s.ch_scale = _Buf((0.5 + _rand(g, N)) * (4 / 127 / math.sqrt(K)))
        s.bias = _Buf(0.3 * _randn(g, N)) if case["bias"] else None
        s.ld, s.out = ld, _new(ELEM[case["out"]][1], M, N)
    elif op == "route":
        M, E, k = case["M"], case["E"], case["k"]
        s.bias = _Buf(0.05 * _randn(g, E) / (1 if case["score"] == "sigmoid" else E)) if case["bias"] else None
        s.x = _Buf(_logits(case, g, None if s.bias is None else s.bias.t))
        # 0 where a row is padding
        s.rows = _Buf((_rand(g, M) > 0.03).to(torch.uint8)) if case["masked"] else None
        s.idx, s.wt, s.count = _new(torch.int32, M, k), _new(torch.float32, M, k), _new(torch.int32, E)
    else:
        M, k, E, D, F, N = (case[x] for x in ("M", "k", "E", "D", "F", "N"))
        H = 2 * F if case["gated"] else F
        s.x = _Buf(_inputs(case, g, D, D))
        # the experts of a row, as routing leaves them: distinct, some asked for more often, largest weight first
        l = _randn(g, M, E) + 0.5 * _randn(g, 1, E)
        wt, idx = torch.sort(torch.softmax(l, 1), dim=1, descending=True)
        wt, idx = wt[:, :k], idx[:, :k].to(torch.int32)
        if case["empty"]:  # padding rows have none, and some rows fewer than k
            wt = torch.where(_rand(g, M, 1) * case["empty"] < 0.2, torch.zeros_like(wt), wt)
            wt[1::7, k // 2:] = 0
            idx = torch.where(wt > 0, idx, torch.full_like(idx, -1))
        s.wt, s.idx = _Buf((wt / wt.sum(1, keepdim=True).clamp_min(1e-20)).contiguous()), _Buf(idx.contiguous())
        s.w1, s.w2 = _Buf(_codes(g, E * H, D, D)), _Buf(_codes(g, E * N, F, F))
        s.s1 = _Buf((0.5 + _rand(g, E, H)) * (4 / 127 / math.sqrt(D)))
        s.s2 = _Buf((0.5 + _rand(g, E, N)) * (4 / 127 / math.sqrt(F)))
        s.b1 = _Buf(0.3 * _randn(g, E, H)) if case["bias"] else None
        s.b2 = _Buf(0.3 * _randn(g, E, N)) if case["bias"] else None
        s.out = _new(ELEM[case["out"]][1], M, N)
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
        _contexts[T] = vdttfs, vdttfs.Context(vdttfs.TaskConsts(T=T, delta=16))
    return _contexts[T]


def _run_own(s):
    case, op = s.case, s.case["op"]
    vdttfs, ctx = _context(case.get("T", 64))
    if op == "mm":
        ctx.i8_matmul(s.out, ELEM[case["out"]][0], case["N"], s.x, s.ld, s.row_scale, s.w, s.ld, s.ch_scale, s.bias,
                      ACT[case["act"]], case["M"], case["N"], case["K"])
        return s.out.t
    if op == "lin":
        ctx.i8_linear(s.out, ELEM[case["out"]][0], case["N"], s.x, ELEM[case["in"]][0], s.ld, s.w, s.ld, s.ch_scale,
                      s.bias, ACT[case["act"]], case["M"], case["N"], case["K"])
        return s.out.t
    if op == "route":
        ctx.route(s.idx, s.wt, s.count, s.x, ELEM[case["in"]][0], case["E"], s.bias, s.rows, case["M"], case["E"],
                  case["k"], score=0 if case["score"] == "softmax" else 1, groups=case["groups"],
                  top_groups=case["top_groups"], group_top=case["group_top"], renorm=case["renorm"],
                  scale=case["scale"])
        return {"idx": s.idx.t, "weight": s.wt.t, "count": s.count.t}
    ctx.experts(s.out, ELEM[case["out"]][0], case["N"], s.x, ELEM[case["in"]][0], case["D"], s.idx, s.wt, case["M"],
                case["k"], vdttfs.ExpertWeights(case["E"], case["D"], case["F"], case["N"], ACT[case["act"]],
                                                case["gated"], s.w1, s.s1, s.b1, s.w2, s.s2, s.b2))
    return s.out.t


def _act(v, act):
    return torch.clamp_min(v, 0) if act == "relu" else v / (1 + torch.exp(-v)) if act == "silu" else v


def _quant(x):
    """Codes (as floats) and scales of the last axis of x, in 32 bits."""
    a = x.abs().amax(-1, keepdim=True)
    s = a / torch.full_like(a, 127)
    return torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-127, 127), s


def _quant_times(t, T):
    return torch.where(t < T, T - torch.floor(t), torch.zeros_like(t)), torch.full_like(t[:, :1], 1 / T)


def _quant_in(case, x):
    return _quant_times(x, case["T"]) if case["in"] == "times" else _quant(x.float())


def _run_plain(s):
    case, op = s.case, s.case["op"]
    if op in ("mm", "lin"):
        K = case["K"]
        if op == "mm":
            q, sc = s.x.t[:, :K].float(), s.row_scale.t[:, None]
        else:
            q, sc = _quant_in(case, s.x.t[:, :K])
        y = (q @ s.w.t[:, :K].float().t()) * sc * s.ch_scale.t
        if s.bias is not None:
            y = y + s.bias.t
        return _act(y, case["act"]).to(ELEM[case["out"]][1])
    if op == "route":
        return _route_plain(s, case)
    return _experts_plain(s, case)


def _route_plain(s, case):
    M, E, k, none = case["M"], case["E"], case["k"], -math.inf
    l = s.x.t.float()
    ok = l > none
    if s.rows is not None:
        ok = ok & (s.rows.t != 0)[:, None]
    l = torch.where(ok, l, none)
    if case["score"] == "softmax":
        p = torch.exp(torch.where(ok, l - l.amax(1, keepdim=True), none))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-l))
    c = p if s.bias is None else p + s.bias.t
    c = torch.where(ok, c, none)
    if case["groups"] > 1:
        v = torch.sort(c.view(M, case["groups"], -1), dim=2, descending=True)[0][:, :, :case["group_top"]]
        v = torch.where((v[:, :, 0] > none), torch.where(v > none, v, 0).sum(2), none)
        best = torch.sort(v, dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        keep = torch.zeros(v.shape, dtype=torch.bool, device=v.device).scatter_(1, best, True)
        c = torch.where(keep.repeat_interleave(E // case["groups"], 1), c, none)
    v, idx = torch.sort(c, dim=1, descending=True, stable=True)
    v, idx = v[:, :k], idx[:, :k]
    w = torch.where(v > none, p.gather(1, idx), 0)
    if case["renorm"]:
        t = w.sum(1, keepdim=True)
        w = torch.where(t > 0, w / t, 0)
    count = torch.zeros(E, dtype=torch.int32, device=l.device)
    count.scatter_add_(0, idx.reshape(-1), (v > none).reshape(-1).to(torch.int32))
    return {"idx": torch.where(v > none, idx, -1).to(torch.int32), "weight": w * case["scale"], "count": count}


def _experts_plain(s, case):
    """The pairs (row, expert) padded to the busiest expert's number, as two batched products."""
    M, k, E, D, F, N = (case[x] for x in ("M", "k", "E", "D", "F", "N"))
    q, sc = _quant_in(case, s.x.t)
    pair = torch.nonzero(s.idx.t.reshape(-1) >= 0)[:, 0]
    e = s.idx.t.reshape(-1)[pair].long()
    y = torch.zeros((M * k, N), device=q.device)
    if pair.numel():
        e, order = torch.sort(e, stable=True)
        pair = pair[order]
        count = torch.bincount(e, minlength=E)
        at = torch.arange(e.numel(), device=q.device) - (torch.cumsum(count, 0) - count)[e]
        most = int(count.max())
        xq, xs = torch.zeros((E, most, D), device=q.device), torch.zeros((E, most, 1), device=q.device)
        xq[e, at], xs[e, at] = q[pair // k], sc[pair // k]
        u = torch.bmm(xq, s.w1.t.float().view(E, -1, D).transpose(1, 2)) * xs * s.s1.t[:, None]
        if s.b1 is not None:
            u = u + s.b1.t[:, None]
        h = _act(u[:, :, :F], case["act"]) * u[:, :, F:] if case["gated"] else _act(u, case["act"])
        hq, hs = _quant(h)
        z = torch.bmm(hq, s.w2.t.float().view(E, N, F).transpose(1, 2)) * hs * s.s2.t[:, None]
        if s.b2 is not None:
            z = z + s.b2.t[:, None]
        y[pair] = z[e, at]
    y = (y.view(M, k, N) * s.wt.t[:, :, None]).sum(1)
    return y.to(ELEM[case["out"]][1])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------
def _codes64(case, x):
    """Codes and scales by definition: the scale and the quotient are rounded to 32 bits, nothing else."""
    if case.get("in") == "times":
        T = case["T"]
        b = torch.floor(x.double())
        return torch.where(b < T, T - b, torch.zeros_like(b)), torch.full((x.shape[0], 1), 1 / T, device=x.device,
                                                                          dtype=torch.float64)
    x = x.double()
    s = (x.abs().max(dim=1, keepdim=True)[0] / 127).float().double()
    q = torch.round((x / s).float().double())
    return torch.clamp(torch.where(s == 0, torch.zeros_like(q), q), -127, 127), s


def _act64(v, act):
    return v.clamp(min=0) if act == "relu" else v * torch.sigmoid(v) if act == "silu" else v


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("mm", "lin"):
        x, w = s.x.t[:, :case["K"]], s.w.t[:, :case["K"]].double()
        q, sc = (x.double(), s.row_scale.t.double()[:, None]) if op == "mm" else _codes64(case, x)
        y = torch.mm(q, w.t().contiguous()).mul_(sc).mul_(s.ch_scale.t.double())
        return _act64(y if s.bias is None else y + s.bias.t.double(), case["act"])
    if op == "route":
        l = s.x.t if s.rows is None else s.x.t.masked_fill((s.rows.t == 0)[:, None], -math.inf)
        p, c = _choice64(case, l, None if s.bias is None else s.bias.t)
        if case["groups"] > 1:
            c = _groups64(case, c)[1]
        v, idx = (x[:, :case["k"]] for x in torch.sort(c, dim=1, descending=True, stable=True))
        w = torch.gather(p, 1, idx).masked_fill(v == -math.inf, 0)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
        idx = idx.masked_fill(v == -math.inf, -1)
        count = torch.stack([(idx == e).sum() for e in range(case["E"])])
        return {"idx": idx, "weight": w * case["scale"], "count": count}
    F, y = case["F"], torch.zeros((case["M"], case["N"]), dtype=torch.float64, device="cuda")
    q, sc = _codes64(case, s.x.t)
    w1, w2 = s.w1.t.view(case["E"], -1, case["D"]), s.w2.t.view(case["E"], case["N"], F)
    for e in range(case["E"]):
        row, slot = torch.nonzero(s.idx.t == e, as_tuple=True)
        if not row.numel():
            continue
        u = torch.mm(q[row], w1[e].double().t().contiguous()) * sc[row] * s.s1.t[e].double()
        u = u if s.b1 is None else u + s.b1.t[e].double()
        h = _act64(u[:, :F], case["act"]) * u[:, F:] if case["gated"] else _act64(u, case["act"])
        hq, hs = _codes64({}, h)
        z = torch.mm(hq, w2[e].double().t().contiguous()) * hs * s.s2.t[e].double()
        z = z if s.b2 is None else z + s.b2.t[e].double()
        y.index_add_(0, row, z * s.wt.t[row, slot].double()[:, None])
    return y


# ---- what a pass cannot do without ----------------------------------------------
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "times": 4}
    op, M = case["op"], case["M"]
    if op in ("mm", "lin"):
        N, K = case["N"], case["K"]
        row = K + 4 if op == "mm" else K * size[case["in"]]
        return {"bytes": M * row + N * (K + 4 + (4 if case["bias"] else 0)) + M * N * size[case["out"]],
                "flops": 2 * M * N * K}
    if op == "route":
        E, k = case["E"], case["k"]
        return {"bytes": M * (E * size[case["in"]] + 8 * k + (1 if case["masked"] else 0)) + 4 * E +
                (4 * E if case["bias"] else 0), "flops": 10 * M * E}
    k, E, D, F, N = (case[x] for x in ("k", "E", "D", "F", "N"))
    H = 2 * F if case["gated"] else F
    used = E * (1 - (1 - min(1, k / E)) ** M)  # experts that some row asks for, if all were asked for alike
    one = H * (D + 4) + N * (F + 4) + (4 * (H + N) if case["bias"] else 0)
    return {"bytes": M * (D * size[case["in"]] + 8 * k + N * size[case["out"]]) + used * one,
            "flops": 2 * M * k * (H * D + N * F)}
