"""The conditional head on VGG-16's last spike map: each of its calls against its
definition on what the call before it gave, and the whole of it run again for
the same bits."""
import numpy as np
import pytest

import headref as R
import vdttfs
from vdttfs import heads, models

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1, 5, 64])
def test_head_over_vgg16(gpu_ctx_factory, B):
    w = models.vgg16()
    ctx = gpu_ctx_factory(w.consts)
    net = vdttfs.Net(ctx, w.layers, B, w.img_elems, vdttfs.ENCODE_LINEAR, w.tc_in, w.td_in, w.readout)
    head, spikes = heads.head_of(ctx, net, n_experts=12, top_k=3, width=200, hidden=96)
    img = ctx.to_device(models.images_for(w, B))
    net.forward(img)
    head.forward(spikes)
    ctx.synchronize()
    at = max(i for i, l in enumerate(w.layers) if l.kind == vdttfs.LAYER_FC)
    times = net.layer_output(at).reshape(B, -1)
    assert (times < 9999).any()

    # the weights' codes are those of the float kernels
    F, W, E, H, N = head.features, head.width, head.n_experts, head.hidden, head.classes
    k = lambda i, *shape: models.kaiming(11, i, shape, shape[-2])  # noqa: E731
    pq, ps = R.quant_rows(np.ascontiguousarray(k(0, F, W).T))
    np.testing.assert_array_equal(head.project.w.download()[:, :F], pq)
    np.testing.assert_array_equal(head.project.scale.download(), ps)
    e1 = [R.quant_rows(np.ascontiguousarray(m.T)) for m in k(2, E, W, H)]
    e2 = [R.quant_rows(np.ascontiguousarray(m.T)) for m in k(3, E, H, N)]

    # projection of the spike map
    q, s = R.quant_times(times, w.consts.T, w.consts.tfs)
    y, d = R.product(q, s, pq, ps, np.zeros(W, np.float32), R.RELU)
    x = head.x.download()
    assert (np.abs(x - y) <= R.out_bound(y, d, R.F32)).all()

    # routing of the potentials
    logits, idx, wt = head.logits.download(), head.idx.download(), head.weight.download()
    ri, rw, decided = R.route(logits, np.zeros(E, np.float32), None, 3, 1, 1, 1, 1, True, 1.0)
    np.testing.assert_array_equal(idx[decided], ri[decided])
    assert (np.abs(wt - rw) <= R.route_bound(E) * rw + 1e-37)[decided].all()
    np.testing.assert_array_equal(head.count.download(), np.bincount(idx[idx >= 0], minlength=E))

    # experts of what was routed
    q, s = R.quant_rows(x)
    y, d, _ = R.experts(q, s, idx, wt, np.stack([a for a, _ in e1]), np.stack([b for _, b in e1]),
                        np.zeros((E, H), np.float32), np.stack([a for a, _ in e2]), np.stack([b for _, b in e2]),
                        np.zeros((E, N), np.float32), R.RELU, False)
    out = head.out.download()
    assert (np.abs(out - y) <= R.out_bound(y, d, R.F32)).all()
    np.testing.assert_array_equal(head.pred.download(), out.argmax(axis=1))

    # and again: the same bits
    net.forward(img)
    head.forward(spikes)
    ctx.synchronize()
    np.testing.assert_array_equal(head.out.download(), out)
    np.testing.assert_array_equal(head.idx.download(), idx)
    net.close()
