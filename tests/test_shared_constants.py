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
    sim.device, sim._dtype, sim._weights, sim._images, sim._constants = torch.device("cpu"), AP_FIXED_16_8, {}, {}, {}
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


def test_outputs_by_name_are_kept():
    """A graph output described by a tensor of its own: forward_raw keeps the graph's outputs whatever ``keep`` holds, so a
    paged node's rows of that name are not the layers' shared buffer."""
    import torch
    from cormorant_amd.graph import Graph
    w = models.smollm2_weights(SHAPE, 3)
    exps = models.smollm2_decode(SHAPE, seed=3, weights=w)[2]
    g = models.smollm2_paged(SHAPE, 4, 2, 8, 16, 3, exps, w)
    preps = [sn for sn in g.nodes if type(sn).__name__ == "PagedPrepNode"]
    t = preps[0].output
    own = TensorInfo(t.onnx_name, list(t.shape), exp=t.exp)
    sim = object.__new__(Simulator)
    sim.device, sim._private, sim._keep, sim._shared, sim._passing = torch.device("cpu"), None, set(), {}, []
    sim._graph = Graph(g.nodes, input_tensors=g.input_tensors, output_tensors=g.output_tensors + [own])
    rows = [sim._paged_rows(sn) for sn in preps]
    assert sim._passing == [preps[1].output.onnx_name] and rows[0].data_ptr() != rows[1].data_ptr()


def embedding(rows, seed):
    from cormorant_amd.host_ops import LlmEmbedNode
    table = np.random.default_rng(seed).standard_normal((rows, 8)).astype(np.float32)
    return LlmEmbedNode([TensorInfo("ids", [2], exp=0, kind="i32")], TensorInfo("h0", [2, 8], exp=15, kind="i32"), table=table)


def test_embeddings_of_entries_that_come_and_go(monkeypatch):
    """Entries share one dict of images that outlives their graphs: a node made where a dropped entry's was (the same id)
    reads its own table, and equal tables are one copy."""
    import torch
    from cormorant_amd import simulate, units
    read = []
    monkeypatch.setattr(units, "embed_rows", lambda img, ids, out, rows, d: read.append(img.numpy()))
    images = {}

    def run(node):
        sim = constants()
        sim._images = images
        sim._embed(node, {"ids": torch.zeros(2, dtype=torch.int32)})
        np.testing.assert_array_equal(read.pop(), node.image())

    monkeypatch.setattr(simulate, "id", lambda node: 7, raising=False)     # each node where the one before it was
    for rows, seed in ((9, 0), (6, 1), (9, 0), (9, 2), (6, 1)):
        run(embedding(rows, seed))
    assert len(images) == 3
