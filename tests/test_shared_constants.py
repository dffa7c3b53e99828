"""Entries of one model that share their device constants (Simulator(share=...)), without a GPU: each entry's rotations read
its own table, whichever entry came first, and the layers of a model one copy of it."""
import numpy as np
import pytest

from cormorant_amd import models
from cormorant_amd.dtype import AP_FIXED_16_8
from cormorant_amd.graph import TensorInfo
from cormorant_amd.simulate import Simulator

SHAPE = models.LlamaShape(layers=2, batch=2, d=128, heads=2, kv=1, hd=64, ff=128, vocab=256, ctx=64)


def tables(g):
    every = [getattr(x, "table", None) for sn in g.nodes for x in (sn, getattr(sn, "rope_q", None))]
    return [t for t in every if isinstance(t, TensorInfo)]


def entries():
    w = models.smollm2_weights(SHAPE, 3)
    decode, _, exps = models.smollm2_decode(SHAPE, seed=3, weights=w, runtime_pos=True)
    unfused, _, _ = models.smollm2_decode(SHAPE, seed=3, weights=w, runtime_pos=True, fused_attention=False)
    paged = [models.smollm2_paged(SHAPE, 4, 2, 8, 16, n, exps, w) for n in (3, 6, 4)]
    return [decode, unfused] + paged


def constants():
    """A simulator's constants alone (the units need a GPU)."""
    import torch
    sim = object.__new__(Simulator)
    sim.device, sim._dtype, sim._weights = torch.device("cpu"), AP_FIXED_16_8, {}
    return sim


@pytest.mark.parametrize("order", [(0, 2, 3), (2, 0, 1), (3, 2, 4), (4, 3, 1, 2, 0)])
def test_rope_tables(order):
    every, sim = entries(), constants()
    for i in order:
        ts = tables(every[i])
        assert len(ts) >= SHAPE.layers
        for t in ts:
            np.testing.assert_array_equal(sim._get(t, {}).numpy(), t.data)


def test_one_copy_for_the_layers():
    for g in entries():
        sim = constants()
        assert len({sim._get(t, {}).data_ptr() for t in tables(g)}) == len(sim._weights) == 1
