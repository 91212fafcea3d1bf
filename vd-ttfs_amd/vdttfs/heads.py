"""A conditional head on a spiking trunk, in 8-bit integers.

The trunk's last spike map is its activation already: a product in 8-bit codes
(``Context.i8_linear``) projects it, a potential readout over the experts
(``Context.fc_vmem``) gives the router's logits, ``Context.route`` picks each
sample's experts, and ``Context.experts`` applies them.  Everything runs on the
context's stream, after the trunk's forward, without a copy or a wait.

    python -m vdttfs.heads          # VGG-16's 512 features, 16 experts, 2 a sample
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .core import (ACT_NONE, ACT_RELU, ELEM_F32, ELEM_TIMES, LAYER_FC, SCORE_SIGMOID, Context, DeviceArray,
                   ExpertWeights, Net)


class DevicePtr:
    """A device address that something else owns, as the calls take it."""

    def __init__(self, ptr, owner=None):
        self.ptr = ptr if isinstance(ptr, C.c_void_p) else C.c_void_p(ptr)
        self.owner = owner


class QuantizedKernel:
    """An FC kernel of the weights blob, float [C_in][C_out], as codes
    [C_out][ld] and channel scales on the device; rows start on 16 bytes."""

    def __init__(self, ctx: Context, kernel: np.ndarray):
        k = np.ascontiguousarray(kernel, np.float32)
        self.c_in, self.c_out = k.shape
        self.ld = (self.c_in + 15) // 16 * 16
        self.w, self.scale = ctx.empty((self.c_out, self.ld), np.int8), ctx.empty(self.c_out)
        d = ctx.to_device(k)
        ctx.quant_kernel(d, self.c_in, self.c_out, self.w, self.ld, self.scale)
        ctx.synchronize()
        d.free()


class ExpertHead:
    """Projection, router and experts over a spike map of `features` neurons.

    project [features][width] and its bias; router [features][experts] and its
    bias, read out as membrane potentials under the decay table `alpha`
    (T + 1 floats); w1 [experts][width][hidden], w2 [experts][hidden][classes]
    and their biases: host floats in the FC layout of the weights blob.
    `balance` is added to a sample's scores where experts are chosen, and not to
    their weights.  Shapes that do not go together raise ValueError."""

    def __init__(self, ctx: Context, B: int, project, project_bias, router, router_bias, alpha, w1, b1, w2, b2,
                 top_k: int = 2, balance=None):
        self.ctx, self.B, self.top_k = ctx, B, top_k
        # the kernels read these sizes, whatever the arrays hold
        if any(len(np.shape(a)) != n for a, n in ((project, 2), (w1, 3), (w2, 3))):
            raise ValueError("project has two dimensions, w1 and w2 have three")
        self.features, self.width = np.shape(project)
        self.n_experts, _, self.hidden = np.shape(w1)
        self.classes = np.shape(w2)[2]
        F, W, E, H, N = self.features, self.width, self.n_experts, self.hidden, self.classes
        for name, a, shape in (("project_bias", project_bias, (W,)), ("router", router, (F, E)),
                               ("router_bias", router_bias, (E,)), ("alpha", alpha, (ctx.consts.T + 1,)),
                               ("w1", w1, (E, W, H)), ("b1", b1, (E, H)), ("w2", w2, (E, H, N)), ("b2", b2, (E, N)),
                               ("balance", balance, (E,))):
            if (a is not None or name != "balance") and np.shape(a) != shape:
                raise ValueError(f"{name} has shape {np.shape(a)}, not {shape}")
        if B < 1 or not 1 <= top_k <= E:
            raise ValueError(f"a batch of {B} and {top_k} of {E} experts")
        self.project = QuantizedKernel(ctx, project)
        f32 = lambda a: ctx.to_device(np.ascontiguousarray(a, np.float32))  # noqa: E731
        self.project_bias, self.router, self.router_bias, self.alpha = map(
            f32, (project_bias, router, router_bias, alpha))
        self.balance = f32(balance) if balance is not None else None
        self._codes = [self._experts(w1), self._experts(w2)]
        self._bias = [f32(b1), f32(b2)]
        (q1, s1), (q2, s2) = self._codes
        self.weights = ExpertWeights(self.n_experts, self.width, self.hidden, self.classes, ACT_RELU, False, q1, s1,
                                     self._bias[0], q2, s2, self._bias[1])
        self.x, self.logits = ctx.empty((B, self.width)), ctx.empty((B, self.n_experts))
        self.idx, self.weight = ctx.empty((B, top_k), np.int32), ctx.empty((B, top_k))
        self.count = ctx.empty(self.n_experts, np.int32)
        self.out, self.pred = ctx.empty((B, self.classes)), ctx.empty(B, np.int32)

    def _experts(self, w: np.ndarray) -> tuple:
        """Codes [E][C_out][C_in] and scales [E][C_out] of float kernels [E][C_in][C_out]."""
        E, c_in, c_out = w.shape
        q, s = self.ctx.empty((E, c_out, c_in), np.int8), self.ctx.empty((E, c_out))
        d = self.ctx.to_device(np.ascontiguousarray(w, np.float32))
        for e in range(E):
            self.ctx.quant_kernel(DevicePtr(d.ptr.value + 4 * e * c_in * c_out), c_in, c_out,
                                  DevicePtr(q.ptr.value + e * c_in * c_out), c_in, DevicePtr(s.ptr.value + 4 * e * c_out))
        self.ctx.synchronize()
        d.free()
        return q, s

    def forward(self, d_times) -> DeviceArray:
        """Class values [B][classes] from a spike map [B][features] (anything with its address in .ptr)."""
        ctx, B, p = self.ctx, self.B, self.project
        ctx.i8_linear(self.x, ELEM_F32, self.width, d_times, ELEM_TIMES, self.features, p.w, p.ld, p.scale,
                      self.project_bias, ACT_RELU, B, self.width, self.features)
        ctx.fc_vmem(d_times, self.logits, self.router, self.router_bias, self.alpha, B, self.features, self.n_experts)
        ctx.route(self.idx, self.weight, self.count, self.logits, ELEM_F32, self.n_experts, self.balance, None, B,
                  self.n_experts, self.top_k, score=SCORE_SIGMOID, renorm=True)
        ctx.experts(self.out, ELEM_F32, self.classes, self.x, ELEM_F32, self.width, self.idx, self.weight, B,
                    self.top_k, self.weights)
        ctx.readout(self.out, B, self.classes, True, self.pred)
        return self.out


def head_of(ctx: Context, net: Net, n_experts=16, top_k=2, width=256, hidden=128, classes=10, seed=11):
    """A randomly initialised head over the last spiking FC layer of `net`, and
    that layer's map, which the network's forward fills."""
    from . import models
    from .core import build_luts_host
    at = max(i for i, l in enumerate(net.layers) if l.kind == LAYER_FC)
    F = net.layers[at].C_out
    ptr, _ = net.layer_output_ptr(at)
    k = lambda i, *shape: models.kaiming(seed, i, shape, shape[-2])  # noqa: E731
    # potentials of spikes: the decay of the map's layer, as its next layer reads it
    alpha, _ = build_luts_host(ctx.consts, net.layers[at].tc_fire, net.layers[at].td, 16.0, 0.0)
    head = ExpertHead(ctx, net.B, k(0, F, width), np.zeros(width), k(1, F, n_experts), np.zeros(n_experts), alpha,
                      k(2, n_experts, width, hidden), np.zeros((n_experts, hidden)),
                      k(3, n_experts, hidden, classes), np.zeros((n_experts, classes)), top_k,
                      balance=np.zeros(n_experts))
    return head, DevicePtr(ptr, net)


def main(B: int = 256):
    from . import models
    w = models.vgg16()
    with Context(w.consts) as ctx:
        net = Net(ctx, w.layers, B, w.img_elems, tc_in=w.tc_in, td_in=w.td_in, readout=w.readout)
        head, spikes = head_of(ctx, net)
        img = ctx.to_device(models.images_for(w, B))
        for _ in range(3):
            net.forward(img)
            head.forward(spikes)
        ctx.synchronize()
        ctx.timer_begin()
        for _ in range(20):
            head.forward(spikes)
        us = ctx.timer_end() / 20 * 1e3
        print(f"head of {head.n_experts} experts over {head.features} features, batch {B}: {us:.1f} us a forward, "
              f"rows of each expert {head.count.download().tolist()}")
        net.close()


if __name__ == "__main__":
    main()
