"""The serving entry with 8-bit weights on the GPU (Simulator) against the oracle's forward pass, every tensor and
every pool bit for bit; the nodes alone; a captured pass replayed."""
import numpy as np
import pytest

from cormorant_amd import models
from cormorant_amd.graph import ColumnsNode, GatedLinear8Node, Graph, Linear8Node, TensorInfo
from oracle import graph_sim as og

pytestmark = pytest.mark.gpu

SHAPE = models.LlamaShape(layers=2, batch=2, d=192, heads=3, kv=1, hd=64, ff=128, vocab=512, ctx=64)
T = TensorInfo


@pytest.fixture(scope="module")
def torch_gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def model():
    w = models.smollm2_weights(SHAPE, 3)
    return models.smollm2_decode(SHAPE, seed=3, weights=w)[2], w


def feeds(ids, new, kv, table):
    return {"ids": np.asarray(ids, np.float64), "q_start": np.concatenate([[0], np.cumsum(new)]).astype(np.float64),
            "kv_len": np.asarray(kv, np.float64), "table": np.asarray(table, np.float64)}


def same(got, want, what):
    for name, v in got.items():
        np.testing.assert_array_equal(v, np.asarray(want[name]).reshape(v.shape), err_msg=f"{what}: {name}")


@pytest.mark.parametrize("int8", [False, True])
def test_serving_steps(torch_gpu, model, int8):
    """Packed prompts, a chunk beside decode tokens, decode steps with the head, over one set of pools and weights."""
    from cormorant_amd.simulate import Simulator
    mk = lambda n, head: models.smollm2_paged(SHAPE, n, 3, 10, 16, 3, *model, int8=int8, with_head=head, weights8=True)  # noqa: E731
    many, few = mk(40, False), mk(3, True)
    sim = Simulator(many)
    sim_few = Simulator(few, share=sim)
    st = {t.onnx_name: np.zeros(t.shape) for t in many.state_tensors}
    ref = {k: v.copy() for k, v in st.items()}
    table, rng, lens = np.array([[4, 0, 9], [1, 7, 2], [5, 3, 8]]), np.random.default_rng(8), np.zeros(3, int)
    for step, new in enumerate(((25, 0, 12), (1, 13, 0), (1, 1, 1), (1, 0, 1))):
        lens += new
        g, s = (many, sim) if max(new) > 1 else (few, sim_few)
        n = int(g.input_tensors[0].shape[0])
        f = feeds(rng.integers(0, SHAPE.vocab, n), new, lens, table)
        same(s._forward_pass(f, states=st), og.forward(g, f, states=ref), f"step {step}")
        for nm in st:
            np.testing.assert_array_equal(st[nm], ref[nm], err_msg=f"step {step}: {nm}")


@pytest.mark.parametrize("n", [1, 20, 70])
@pytest.mark.parametrize("act,fg", [("silu", 11), ("gelu", 8), ("gelu_tanh", 8)])
def test_layer_forms(torch_gpu, n, act, fg):
    """A gate and the down projection onto the residual, columns of its input projection, leading dimensions, a bias,
    exponents a column."""
    from cormorant_amd.simulate import Simulator
    rng = np.random.default_rng([n, fg])
    d, ff = 48, 72
    w = lambda nm, k, m: T(nm, [k, m], data=rng.standard_normal((k, m)) * 0.1)      # noqa: E731
    x, h = T("x", [2, n, d], exp=9), T("h", [2, n, d], exp=15, kind="i32")
    p, c = T("p", [2, n, 2 * d], exp=np.repeat([10, 9], d)), T("c", [2, n, d], exp=9)
    y, z = T("y", [2, n, ff], exp=9), T("z", [2, n, d], exp=15, kind="i32")
    nodes = [Linear8Node([x, w("wp", d, 2 * d)], p, bias=rng.standard_normal(2 * d)), ColumnsNode([p], c, first=d),
             GatedLinear8Node([c, w("wg", d, ff), w("wu", d, ff)], y, act=act, gate_exp=fg, up_exp=10),
             Linear8Node([y, w("wd", ff, d), h], z, delta_exp=12, bias=rng.standard_normal(d))]
    g = Graph(nodes, input_tensors=[x, h], output_tensors=[z])
    f = {"x": np.rint(rng.standard_normal((2, n, d)) * 600) / 512, "h": np.rint(rng.standard_normal((2, n, d)) * 2 ** 16) / 2 ** 15}
    want = og.forward(g, f)
    same(Simulator(g)._forward_pass(f), want, "layer")
    np.testing.assert_array_equal(nodes[2].reference([want["c"], None, None]), want["y"])


@pytest.mark.parametrize("reader", ["out", "reshape", "add", "relu", "matmul", "transpose", "silumul"])
def test_readers_of_columns(torch_gpu, reader):
    """Columns of a projection into nodes that read whole tensors, or out of the graph: as if they were a copy."""
    from cormorant_amd.graph import MatmulNode, OP_ADD, OP_RELU, ReshapeNode, ScheduledNode
    from cormorant_amd.rowops_nodes import SiluMulRoNode, TransposeRoNode
    from cormorant_amd.simulate import Simulator
    rng = np.random.default_rng(len(reader))
    n, d = 24, 32
    x, p = T("x", [n, d], exp=8), T("p", [n, 3 * d], exp=8)
    c, c2, y = T("c", [n, d], exp=8), T("c2", [n, d], exp=8), T("y", [n, d], exp=8)
    nodes = [Linear8Node([x, T("w", [d, 3 * d], data=rng.standard_normal((d, 3 * d)) * 0.2)], p), ColumnsNode([p], c, first=d),
             ColumnsNode([p], c2, first=2 * d)]
    if reader == "out":
        y = c
    elif reader == "reshape":
        y = T("y", [n // 2, 2 * d], exp=8)
        nodes += [ReshapeNode([c], y)]
    elif reader == "add":
        nodes += [ScheduledNode([c, c2], y, OP_ADD)]
    elif reader == "relu":
        nodes += [ScheduledNode([c], y, OP_RELU)]
    elif reader == "matmul":
        nodes += [MatmulNode([c, T("v", [d, d], data=rng.standard_normal((d, d)) * 0.2)], y)]
    elif reader == "transpose":
        y = T("y", [d, n], exp=8)
        nodes += [TransposeRoNode([c], y, perm=(1, 0))]
    else:
        nodes += [SiluMulRoNode([c, c2], y)]
    g = Graph(nodes, input_tensors=[x], output_tensors=[y, c])
    f = {"x": np.rint(rng.standard_normal((n, d)) * 300) / 256}
    same(Simulator(g)._forward_pass(f), og.forward(g, f), reader)


def test_captured_pass_replayed(torch_gpu, model):
    """forward_raw captured once, replayed as the lengths grow with eager passes between, every replay as the oracle."""
    from cormorant_amd.simulate import Simulator
    torch = torch_gpu
    g = models.smollm2_paged(SHAPE, 2, 2, 8, 16, 3, *model, with_head=True, weights8=True)
    sim, name = Simulator(g), g.output_tensors[0].onnx_name
    table, rng = np.array([[6, 2, 0], [3, 5, 1]]), np.random.default_rng(4)
    ref = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    fs = [feeds(rng.integers(0, SHAPE.vocab, 2), [1, 1], [n, n + 14], table) for n in range(1, 5)]
    dev = {nm: sim._to_device(sim._tensor(nm), v) for nm, v in fs[0].items()}
    pools = {nm: torch.zeros(v.shape, dtype=torch.int32, device="cuda") for nm, v in ref.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                    # the images, the workspace: a pass before the capture
        sim.forward_raw({**dev, **{k: v.clone() for k, v in pools.items()}}, keep=[name])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sim.forward_raw({**dev, **pools}, keep=[name])[name]
    for f in fs:
        for nm, v in f.items():
            dev[nm].copy_(sim._to_device(sim._tensor(nm), v))
        graph.replay()
        torch.cuda.synchronize()
        want = og.forward(g, f, states=ref)
        np.testing.assert_array_equal(sim._to_values(sim._tensor(name), out), np.asarray(want[name]).reshape(2, -1))
        for nm in ref:
            np.testing.assert_array_equal(pools[nm].cpu().numpy().astype(np.float64), ref[nm].reshape(pools[nm].shape))
        sim.forward_raw({**{k: sim._to_device(sim._tensor(k), v) for k, v in f.items()},
                         **{k: v.clone() for k, v in pools.items()}}, keep=[name])
