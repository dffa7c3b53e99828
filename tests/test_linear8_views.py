"""The 8-bit nodes in the Simulator, on the CPU: which buffers a pass may reuse, which weights share an image, what of their
rows' codes a caller may change, and which tensors they refuse."""
import numpy as np
import pytest
import torch

from cormorant_amd import models
from cormorant_amd.graph import (ColumnsNode, GatedLinear8Node, Graph, Linear8Node, MatmulNode, PagedAttentionNode, ReshapeNode,
                                 SchedulerError, SelectRowNode, TensorInfo)
from cormorant_amd.numeric import encode_matmul_weights

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


def test_a_bias_of_any_bytes_is_its_own_weight(monkeypatch):
    """A weight without a bias and the same weight with one are two images, whatever the bias holds."""
    from cormorant_amd import linear8, simulate
    monkeypatch.setattr(linear8, "Weight8", lambda *a: ("w", a[2] is None))
    images, x = {}, TensorInfo("x", [3, 40], exp=9)
    w = TensorInfo("w", [40, 1], data=np.linspace(-1, 1, 40)[:, None])
    for raw in (int.from_bytes(b"none", "little"), 0, -1):
        nodes = [Linear8Node([x, w], TensorInfo("y", [3, 1], exp=0), bias=b) for b in (None, [float(raw)])]
        assert int(nodes[1].bias_raw[0]) == raw
        for node, alone in zip(nodes, (True, False)):
            sim = object.__new__(simulate.Simulator)
            sim.device, sim._images, sim._constants = torch.device("cpu"), images, {}
            assert sim._weight8(node) == ("w", alone)
    assert len(images) == 4


def test_the_count_of_quantised_rows_is_not_the_callers():
    """Where the codes' maxima lie depends on how many rows were quantised: a Rows8's count is quant_rows' alone."""
    from cormorant_amd import linear8
    rows = linear8.Rows8(100, 64, "cpu")
    assert (rows.n, rows.cap) == (0, 100)
    with pytest.raises(AttributeError):
        rows.n = 16
    assert rows.n == 0


def written_again(kind):
    """Columns of rows that a later node of the pass writes: (graph, feeds, the columns)."""
    n, d = 4, 16
    h, x = TensorInfo("h", [n, d], exp=8), TensorInfo("x", [1, d], exp=8, state=True)
    rows, rng = TensorInfo("n", [], kind="host"), np.random.default_rng(2)
    c, y = TensorInfo("c", [1, 8], exp=8), TensorInfo("y", [1, d], exp=8, state=True)
    r = x if kind == "state" else TensorInfo("r", [1, d], exp=8)
    nodes = [ColumnsNode([r], c, first=8), SelectRowNode([h, rows], y)]
    if kind == "reshape":
        nodes.insert(0, ReshapeNode([x], r))
    y.onnx_name = "x"                                # the state, written in place
    f = {"h": rng.integers(-99, 99, (n, d)) / 256, "n": np.array(3.0), "x": rng.integers(-99, 99, (1, d)) / 256}
    return Graph(nodes, input_tensors=[h, rows, x], output_tensors=[c]), f, c


@pytest.mark.parametrize("kind", ["state", "reshape"])
def test_columns_of_a_state_are_of_their_time(kind):
    """The dispatch's columns of a state's buffer are a copy: a node that writes the state leaves them."""
    from cormorant_amd import simulate
    g, f, c = written_again(kind)
    sim = object.__new__(simulate.Simulator)
    sim._graph, sim._products, sim._weights = g, None, {}
    raw = {"x": torch.arange(16, dtype=torch.int16).view(1, 16)}
    for sn in g.nodes[:-1]:
        sim._dispatch(sn, raw)
    raw["x"].zero_()
    np.testing.assert_array_equal(raw[c.onnx_name].numpy(), [list(range(8, 16))])


def test_columns_of_a_product_are_a_view():
    from cormorant_amd import simulate
    x, p, c = TensorInfo("x", [3, 16], exp=8), TensorInfo("p", [3, 24], exp=8), TensorInfo("c", [3, 8], exp=8)
    g = Graph([Linear8Node([x, TensorInfo("w", [16, 24], data=np.ones((16, 24)))], p), ColumnsNode([p], c, first=16)])
    sim = object.__new__(simulate.Simulator)
    sim._graph, sim._products = g, None
    raw = {"p": torch.zeros(72, dtype=torch.int16)}
    sim._dispatch(g.nodes[1], raw)
    raw["p"][16] = 5
    assert int(raw["c"][0, 0]) == 5


NOT_ROWS = {"group-major": dict(group_layout=(3, 8)), "axis 1": dict(chexp=np.arange(24)), "state": dict(state=True)}


@pytest.mark.parametrize("how", NOT_ROWS)
@pytest.mark.parametrize("where", ["x", "y", "residual"])
@pytest.mark.parametrize("node", ["linear", "gate", "columns"])
def test_tensors_that_are_not_rows_are_refused(node, where, how):
    """Group-major caches and exponents of axis 1 anywhere, states as outputs; a state may be read."""
    kw = {at: NOT_ROWS[how] if at == where else {} for at in ("x", "y", "residual")}
    if where == "residual" and node != "linear":
        pytest.skip("no residual")
    x, w = TensorInfo("x", [4, 24], exp=8, **kw["x"]), TensorInfo("w", [24, 24], data=np.eye(24))
    wide = where == "residual"
    y = TensorInfo("y", [4, 24], exp=8, kind="i32" if wide else "i16", **kw["y"])
    h = [TensorInfo("h", [4, 24], exp=8, kind="i32", **kw["residual"])] if wide else []
    make = {"linear": lambda: Linear8Node([x, w] + h, y, delta_exp=8 if wide else None), "gate": lambda: GatedLinear8Node([x, w, w], y),
            "columns": lambda: ColumnsNode([x], y)}[node]
    if how == "state" and where != "y":
        make()
    else:
        with pytest.raises(SchedulerError):
            make()


def test_a_weight_that_a_matmul_has_encoded():
    """The values of a weight of both widths: its int16 lanes at their exponents, not the lanes over 2^8; raw lanes are refused."""
    from cormorant_amd.dtype import AP_FIXED_16_8
    from cormorant_amd.linear8 import quantise_weight
    rng = np.random.default_rng(3)
    x, y = TensorInfo("x", [2, 24], exp=rng.integers(8, 10, 24)), TensorInfo("y", [2, 16], exp=rng.integers(9, 12, 16))
    values = rng.standard_normal((24, 16)) * 0.05
    w = TensorInfo("w", [24, 16], data=values.copy())
    encode_matmul_weights([MatmulNode([x, w], y)], AP_FIXED_16_8)
    x8 = TensorInfo("x8", [2, 24], exp=9)
    lanes = np.asarray(w.data, np.float64) * 2.0 ** 8 / 2.0 ** np.asarray(w.wexp, np.float64)
    assert np.abs(lanes - values).max() <= 2.0 ** -(np.asarray(w.wexp).min() + 1.0) and (w.wexp != 8).any()
    for node in (Linear8Node([x8, w], y), Linear8Node([x8, TensorInfo("v", [24, 16], data=lanes)], y)):
        codes, mult = quantise_weight(lanes, 9, np.asarray(y.exp))
        np.testing.assert_array_equal(node.codes, codes)
        np.testing.assert_array_equal(node.mult, mult)
    gate = GatedLinear8Node([x8, w, TensorInfo("u", [24, 16], data=values)], TensorInfo("m", [2, 16], exp=9))
    np.testing.assert_array_equal(gate.gate_codes, quantise_weight(lanes, 9, 8)[0])
    with pytest.raises(SchedulerError):
        Linear8Node([x8, TensorInfo("r", [24, 16], data=np.ones((24, 16), np.int16), raw=True)], y)
