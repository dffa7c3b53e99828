"""Columns of tensors that other nodes write again, on the CPU: which buffers a pass may reuse."""
import pytest

from cormorant_amd import models
from cormorant_amd.graph import ColumnsNode, PagedAttentionNode, ReshapeNode, TensorInfo

SHAPE = models.LlamaShape(layers=2, batch=2, d=128, heads=2, kv=1, hd=64, ff=128, vocab=256, ctx=64)


@pytest.fixture(scope="module")
def small():
    w = models.smollm2_weights(SHAPE, 3)
    return w, models.smollm2_decode(SHAPE, seed=3, weights=w)[2]


def viewed(small, kind, weights8=True):
    """The serving entry whose attention rows pass a view of themselves, which the o projection reads: (graph, the views)."""
    g = models.smollm2_paged(SHAPE, 6, 2, 8, 16, 3, small[1], small[0], weights8=weights8)
    views, nodes = [], []
    for i, sn in enumerate(g.nodes):
        nodes.append(sn)
        if isinstance(sn, PagedAttentionNode):
            om = sn.output
            c = TensorInfo(om.onnx_name + ".view", list(om.shape), exp=om.exp)
            nodes.append(ColumnsNode([om], c, first=0) if kind == "columns" else ReshapeNode([om], c))
            reader = g.nodes[i + 1]
            reader.inputs = [c if t is om else t for t in reader.inputs]
            views.append(c)
    g.nodes = nodes
    return g, views


def names(g):
    from cormorant_amd import simulate
    sim = object.__new__(simulate.Simulator)
    sim._graph, sim._private = g, None
    return sim._step_private()


@pytest.mark.parametrize("kind", ["columns", "reshape"])
def test_viewed_rows_are_not_shared(small, kind):
    """A paged node's rows that a view shows behind the next node are not in the buffer that the layers write in turn."""
    plain = models.smollm2_paged(SHAPE, 6, 2, 8, 16, 3, small[1], small[0], weights8=True)
    assert "l0.om" in names(plain) and "l0.qr" in names(plain)
    private = names(viewed(small, kind)[0])
    assert "l0.om" not in private and "l1.om" not in private and "l0.qr" in private
