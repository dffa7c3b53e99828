"""The 8-bit linear layers' nodes on the CPU: the serving entry with 8-bit weights by the oracle's forward pass, the
front end's nodes for its op list, the nodes' refusals, and weights shared by what they hold."""
import numpy as np
import pytest

from cormorant_amd import linear8, models
from cormorant_amd.frontend import build_graph
from cormorant_amd.graph import ColumnsNode, GatedLinear8Node, Linear8Node, SchedulerError, TensorInfo
from oracle import graph_sim as og
from oracle import linear8 as O

SHAPE = models.LlamaShape(layers=2, batch=2, d=128, heads=2, kv=1, hd=64, ff=128, vocab=256, ctx=64)
T = TensorInfo


@pytest.fixture(scope="module")
def small():
    w = models.smollm2_weights(SHAPE, 3)
    return w, models.smollm2_decode(SHAPE, seed=3, weights=w)[2]


def feeds(ids, new, kv, table):
    return {"ids": np.asarray(ids, np.float64), "q_start": np.concatenate([[0], np.cumsum(new)]).astype(np.float64),
            "kv_len": np.asarray(kv, np.float64), "table": np.asarray(table, np.float64)}


def entry(small, tokens, batch, **kw):
    return models.smollm2_paged(SHAPE, tokens, batch, 8, 16, 3, small[1], small[0], weights8=True, **kw)


def test_packed_rows_are_the_sequences_alone(small):
    """A row's codes are its own: two packed prompts give the rows of each alone, and the same pages."""
    rng = np.random.default_rng(5)
    ids, table = rng.integers(0, SHAPE.vocab, 30), np.array([[3, 1, 6], [0, 7, 2]])
    g = entry(small, 30, 2)
    st, alone = ({t.onnx_name: np.zeros(t.shape) for t in g.state_tensors} for _ in range(2))
    both = og.forward(g, feeds(ids, [18, 11], [18, 11], table), states=st)["l1.h"]
    first = og.forward(entry(small, 18, 1), feeds(ids[:18], [18], [18], table[:1]), states=alone)["l1.h"]
    second = og.forward(entry(small, 11, 1), feeds(ids[18:29], [11], [11], table[1:]), states=alone)["l1.h"]
    np.testing.assert_array_equal(both[:29], np.concatenate([first, second]))
    for nm in st:
        np.testing.assert_array_equal(st[nm], alone[nm])


def test_a_layer_keeps_its_nodes(small):
    """Eight-bit layers in place of every MatMul: one projection for q, k, v, the residuals and the gate in them."""
    kinds = [type(n).__name__ for n in entry(small, 4, 2, with_head=True).nodes]
    assert "MatmulNode" not in kinds and "ResAddRoNode" not in kinds and "SiluMulRoNode" not in kinds
    assert kinds.count("Linear8Node") == 3 * SHAPE.layers + 1 and kinds.count("GatedLinear8Node") == SHAPE.layers
    assert kinds.count("ColumnsNode") == 3 * SHAPE.layers


@pytest.mark.parametrize("with_head", [False, True])
def test_front_end_builds_the_same_nodes(small, with_head):
    kw = dict(int8=True, window=7, with_head=with_head)
    g = entry(small, 4, 2, **kw)
    ops, tensors, ins, outs = entry(small, 4, 2, as_ops=True, **kw)
    f = build_graph(ops, tensors, ins, outs)
    assert [type(n).__name__ for n in f.nodes] == [type(n).__name__ for n in g.nodes]
    fd = feeds(np.random.default_rng(6).integers(0, SHAPE.vocab, 4), [1, 3], [1, 3], [[0, 1, 2], [3, 4, 5]])
    np.testing.assert_array_equal(og.forward(f, fd)[outs[0]], og.forward(g, fd)[outs[0]])


def test_a_node_is_its_products():
    """Linear8Node's residual form is its int16 form and LlmResAdd's sum; the gate its two products and LlmSiluMul's rule."""
    rng = np.random.default_rng(1)
    k, m, x, h = 40, 24, rng.integers(-2000, 2000, (3, 40)), rng.integers(-2 ** 18, 2 ** 18, (3, 24))
    w, wu = (T(n, [k, m], data=rng.standard_normal((k, m)) * 0.05) for n in "wu")
    xt, ht = T("x", [3, k], exp=9), T("h", [3, m], exp=15, kind="i32")
    plain = Linear8Node([xt, w], T("o", [3, m], exp=11), bias=np.linspace(-1, 1, m))
    onto = Linear8Node([xt, w, ht], T("y", [3, m], exp=15, kind="i32"), bias=np.linspace(-1, 1, m), delta_exp=11)
    assert onto.shift == 4 and (onto.bias_raw == np.rint(np.linspace(-1, 1, m) * 2048)).all()
    o = O.linear(x, plain.codes, plain.mult, plain.bias_raw).astype(np.int64)
    np.testing.assert_array_equal(O.linear(x, onto.codes, onto.mult, onto.bias_raw, h, onto.shift), h + (o << 4))
    # |value error| of a row: codes off by half a step of k terms each (x's and w's), and the output's rounding
    real, step_x, step_w = x / 512.0 @ w.data + np.linspace(-1, 1, m), np.abs(x).max(1) / 512.0 / 254, np.abs(w.data).max(0) / 254
    bound = (step_x[:, None] * 1.002 * np.abs(w.data).sum(0) + np.abs(x).sum(1)[:, None] / 512.0 * step_w
             + 1.002 * k * step_x[:, None] * step_w) * (1 + 2.0 ** -17) + 2.0 ** -12 + 2.0 ** -17 * np.abs(real) + 2.0 ** -12
    assert (np.abs(o / 2048.0 - real) <= bound).all()
    g = GatedLinear8Node([xt, w, wu], T("y", [3, m], exp=10), gate_exp=12, up_exp=11)
    assert (g.gate_shift, g.out_shift) == (2, 21)
    np.testing.assert_array_equal(g.gate_codes, plain.codes)


BAD = {
    "no data": lambda x, w, y, h: Linear8Node([x, T("w", [40, 24])], y),
    "k": lambda x, w, y, h: Linear8Node([x, T("w", [39, 24], data=np.ones((39, 24)))], y),
    "m": lambda x, w, y, h: Linear8Node([x, w], T("y", [3, 23], exp=11)),
    "rows": lambda x, w, y, h: Linear8Node([x, w], T("y", [2, 24], exp=11)),
    "x kind": lambda x, w, y, h: Linear8Node([T("x", [3, 40], exp=9, kind="i32"), w], y),
    "x exponents": lambda x, w, y, h: Linear8Node([T("x", [3, 40], exp=np.arange(40)), w], y),
    "y kind": lambda x, w, y, h: Linear8Node([x, w], h),
    "no delta": lambda x, w, y, h: Linear8Node([x, w, h], T("z", [3, 24], exp=15, kind="i32")),
    "delta": lambda x, w, y, h: Linear8Node([x, w, h], T("z", [3, 24], exp=15, kind="i32"), delta_exp=16),
    "far delta": lambda x, w, y, h: Linear8Node([x, w, h], T("z", [3, 24], exp=15, kind="i32"), delta_exp=-2),
    "residual exponent": lambda x, w, y, h: Linear8Node([x, w, h], T("z", [3, 24], exp=14, kind="i32"), delta_exp=9),
    "bias": lambda x, w, y, h: Linear8Node([x, w], y, bias=np.ones(23)),
    "large bias": lambda x, w, y, h: Linear8Node([x, w], y, bias=np.full(24, 2.0 ** 21)),
    "gate sizes": lambda x, w, y, h: GatedLinear8Node([x, w, T("u", [40, 23], data=np.ones((40, 23)))], y),
    "gate exponent": lambda x, w, y, h: GatedLinear8Node([x, w, w], y, gate_exp=15),
    "gelu exponent": lambda x, w, y, h: GatedLinear8Node([x, w, w], y, act="gelu", gate_exp=9),
    "act": lambda x, w, y, h: GatedLinear8Node([x, w, w], y, act="tanh"),
    "y exponents": lambda x, w, y, h: GatedLinear8Node([x, w, w], T("y", [3, 24], exp=np.arange(24))),
    "columns": lambda x, w, y, h: ColumnsNode([x], T("c", [3, 16], exp=9), first=32),
    "column words": lambda x, w, y, h: ColumnsNode([x], T("c", [3, 16], exp=9), first=4),
    "column exponents": lambda x, w, y, h: ColumnsNode([x], T("c", [3, 16], exp=10), first=8),
}


@pytest.mark.parametrize("case", BAD)
def test_refusals(case):
    x, y, h = T("x", [3, 40], exp=9), T("y", [3, 24], exp=11), T("h", [3, 24], exp=15, kind="i32")
    w = T("w", [40, 24], data=np.random.default_rng(0).standard_normal((40, 24)) * 0.05)
    Linear8Node([x, w], y)
    with pytest.raises(SchedulerError):
        BAD[case](x, w, y, h)


def test_weights_are_found_by_what_they_hold(monkeypatch):
    """Simulators that share images hold one copy of equal weights and their own of others, whichever node came first."""
    import torch
    from cormorant_amd import simulate
    made = []
    monkeypatch.setattr(linear8, "Weight8", lambda *a: made.append(a) or ("w", len(made)))
    monkeypatch.setattr(linear8, "GatedWeight8", lambda *a, **k: made.append(a) or ("g", len(made)))
    monkeypatch.setattr(simulate, "id", lambda node: 7, raising=False)      # each node where the one before it was
    images = {}

    def image(node):
        sim = object.__new__(simulate.Simulator)
        sim.device, sim._images, sim._constants = torch.device("cpu"), images, {}
        return sim._weight8(node)
    x, rng = T("x", [3, 40], exp=9), np.random.default_rng(0)
    a, b = (T("w", [40, 24], data=rng.standard_normal((40, 24))) for _ in range(2))
    lin = lambda w, e=3, bias=None: Linear8Node([x, w], T("y", [3, 24], exp=e), bias=bias)      # noqa: E731
    gate = lambda w, u, e=3: GatedLinear8Node([x, w, u], T("y", [3, 24], exp=e), gate_exp=4, up_exp=4)      # noqa: E731
    nodes = [lin(a), lin(b), lin(a, 4), lin(a, 3, np.ones(24)), lin(a, 3, np.zeros(24)), gate(a, b), gate(b, a), gate(a, b, 4)]
    first = [image(n) for n in nodes]
    assert len(set(first)) == len(nodes) == len(made) == len(images)
    assert [image(n) for n in reversed([lin(a), lin(b), lin(a, 4), lin(a, 3, np.ones(24)), lin(a, 3, np.zeros(24)), gate(a, b),
                                        gate(b, a), gate(a, b, 4)])] == first[::-1]
