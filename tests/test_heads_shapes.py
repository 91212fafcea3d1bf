"""An expert head refuses arrays whose shapes do not go together, before it touches the device."""
import types

import numpy as np
import pytest

import vdttfs
from vdttfs import heads

F, W, E, H, N, T = 12, 6, 4, 5, 3, 16
GOOD = dict(project=(F, W), project_bias=(W,), router=(F, E), router_bias=(E,), alpha=(T + 1,), w1=(E, W, H),
            b1=(E, H), w2=(E, H, N), b2=(E, N), balance=(E,))


class Reached(Exception):
    pass


def made(**other):
    def empty(*a):
        raise Reached

    ctx = types.SimpleNamespace(consts=vdttfs.TaskConsts(T=T), empty=empty)
    arrays = {k: np.zeros(v, np.float32) for k, v in GOOD.items()}
    B, top_k = other.pop("B", 2), other.pop("top_k", 2)
    arrays.update({k: None if v is None else np.zeros(v, np.float32) for k, v in other.items()})
    return heads.ExpertHead(ctx, B, top_k=top_k, **arrays)


def test_right_shapes_reach_the_device():
    for other in ({}, {"balance": None}, {"top_k": E}):
        with pytest.raises(Reached):
            made(**other)


@pytest.mark.parametrize("name", sorted(GOOD))
def test_wrong_shapes_are_refused(name):
    shape = GOOD[name]
    for i in range(len(shape)):
        for d in (-1, 1):
            bad = shape[:i] + (shape[i] + d,) + shape[i + 1:]
            with pytest.raises(ValueError):
                made(**{name: bad})
    with pytest.raises(ValueError):
        made(**{name: shape + (1,)})


def test_other_refusals():
    for other in ({"top_k": 0}, {"top_k": E + 1}, {"B": 0}, {"b1": None}, {"alpha": None}):
        with pytest.raises(ValueError):
            made(**other)
