"""The paged serving entry on the GPU (Simulator) against the oracle's forward pass, every tensor and
every pool bit for bit: packed prompts, a chunk beside decode tokens, decode steps; both caches; per-head
norms with interleaved and partial rotations; a captured pass replayed as the batch moves on."""
import numpy as np
import pytest

from cormorant_amd import models
from cormorant_amd.graph import Graph, PagedAttentionNode, TensorInfo, paged_pool, softmax_regs
from cormorant_amd.rowops_nodes import PagedPrepNode
from oracle import graph_sim as og

pytestmark = pytest.mark.gpu

SHAPE = models.LlamaShape(layers=2, batch=2, d=192, heads=3, kv=1, hd=64, ff=128, vocab=512, ctx=64)


@pytest.fixture(scope="module")
def torch_gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def feeds(ids, new, kv, table):
    return {"ids": np.asarray(ids, np.float64), "q_start": np.concatenate([[0], np.cumsum(new)]).astype(np.float64),
            "kv_len": np.asarray(kv, np.float64), "table": np.asarray(table, np.float64)}


def same(got, want, what):
    for name, v in got.items():
        np.testing.assert_array_equal(v, np.asarray(want[name]).reshape(v.shape), err_msg=f"{what}: {name}")


@pytest.mark.parametrize("int8,window", [(False, 0), (True, 0), (False, 9)])
def test_serving_steps(torch_gpu, int8, window):
    """Prompts of 21 and 1 tokens, then a chunk of 13 beside a decode token, then decode steps across a
    page's end, with a third sequence that waits (no tokens) and rows behind the last sequence."""
    from cormorant_amd.simulate import Simulator
    w = models.smollm2_weights(SHAPE, 3)
    exps = models.smollm2_decode(SHAPE, seed=3, weights=w)[2]
    mk = lambda T, head: models.smollm2_paged(SHAPE, T, 3, 10, 16, 3, exps, w, int8=int8, window=window,   # noqa: E731
                                              with_head=head)
    many, few = mk(24, False), mk(3, True)
    sim = Simulator(many)
    sim_few = Simulator(few, share=sim)
    st = {t.onnx_name: np.zeros(t.shape) for t in many.state_tensors}
    ref = {k: v.copy() for k, v in st.items()}
    table = np.array([[4, 0, 9], [1, 7, 2], [5, 3, 8]])
    rng = np.random.default_rng(8)
    lens = np.zeros(3, int)
    for step, new in enumerate(((21, 0, 1), (1, 13, 0), (0, 0, 0), (1, 1, 1), (1, 0, 1), (1, 1, 0))):
        lens += new
        g, s = (many, sim) if max(new) > 1 else (few, sim_few)
        T = int(g.input_tensors[0].shape[0])
        print(f"step {step}: new {new} lengths {lens}", flush=True)
        f = feeds(rng.integers(0, SHAPE.vocab, T), new, lens, table)
        got, want = s._forward_pass(f, states=st), og.forward(g, f, states=ref)
        same(got, want, f"step {step}")
        for nm in st:
            np.testing.assert_array_equal(st[nm], ref[nm], err_msg=f"step {step}: {nm}")


def test_lean_pass(torch_gpu):
    """A pass whose caller reads the output alone (the layers' rows in one buffer): h and the pools as in a
    pass that keeps every tensor, padded rows among them; a kept row tensor is its layer's own."""
    from cormorant_amd.simulate import Simulator
    w = models.smollm2_weights(SHAPE, 3)
    exps = models.smollm2_decode(SHAPE, seed=3, weights=w)[2]
    g = models.smollm2_paged(SHAPE, 30, 2, 8, 16, 3, exps, w)
    sim = Simulator(g)
    f = feeds(np.random.default_rng(1).integers(0, SHAPE.vocab, 30), [18, 9], [18, 9], [[3, 1, 6], [0, 7, 2]])
    every = sim._forward_pass(f)
    dev = {nm: sim._to_device(sim._tensor(nm), v) for nm, v in {**f, **sim.initial_states()}.items()}
    raw = sim.forward_raw(dict(dev), keep=["l1.h", "l0.om"])
    assert "l0.om" in raw and not {"l0.qr", "l1.qr", "l1.om"} & set(raw)
    for nm in ("l1.h", "l0.om", "l0.pool", "l1.pool"):
        np.testing.assert_array_equal(sim._to_values(sim._tensor(nm), raw[nm]), every[nm])


def layer(T, B, H, KV, HD, rotary, interleaved, norm, int8, page=16, max_pages=4, pages=11):
    """A prep and the attention of its rows as a graph."""
    fq, fk, fv = 11, 10, 9
    rng = np.random.default_rng(HD + rotary)
    t = [TensorInfo(n, [T, w * HD], exp=e) for n, w, e in (("q", H, fq), ("k", KV, fk), ("v", KV, fv))]
    pool = paged_pool("pool", pages, page, KV, HD, int8)
    step = [TensorInfo("q_start", [B + 1], exp=0, kind="i32"), TensorInfo("kv_len", [B], exp=0, kind="i32"),
            TensorInfo("table", [B, max_pages], exp=0, kind="i32")]
    qr, o = TensorInfo("qr", [T, H * HD], exp=11), TensorInfo("o", [T, H * HD], exp=14 + fv - 8)
    cos, sin = models.rope_half_tables(1e4, rotary, max_pages * page)
    gam = [1 + 0.1 * rng.standard_normal(HD) for _ in range(2)] if norm else [None, None]
    geo = dict(heads=H, kv_heads=KV, head_dim=HD, page=page, int8=int8, f_v=fv)
    cm, cfg = softmax_regs(11 + fk - 8, HD ** -0.5, 14)
    nodes = [PagedPrepNode(t + [pool] + step, qr, f_k=fk, cos=cos, sin=sin, interleaved=interleaved, gamma_q=gam[0],
                           gamma_k=gam[1], eps=1e-5, **geo),
             PagedAttentionNode([qr, pool] + step, o, cm=cm, cfg=cfg, **geo)]
    return Graph(nodes, input_tensors=t + step, output_tensors=[o])


@pytest.mark.parametrize("hd,rotary,interleaved,norm,int8", [
    (64, 64, True, False, False), (64, 32, False, True, True), (128, 128, False, True, False), (128, 64, True, True, True),
])
def test_layer_forms(torch_gpu, hd, rotary, interleaved, norm, int8):
    from cormorant_amd.simulate import Simulator
    g = layer(40, 3, 4, 2, hd, rotary, interleaved, norm, int8)
    rng = np.random.default_rng(9)
    f = {n: np.rint(rng.standard_normal((40, w * hd)) * 400) / 2.0 ** e for n, w, e in (("q", 4, 11), ("k", 2, 10),
                                                                                       ("v", 2, 9))}
    f.update({k: v for k, v in feeds([], [30, 1, 7], [30, 1, 7], rng.permutation(11)[:9].reshape(3, 3)).items()
              if k != "ids"})
    f["table"] = np.concatenate([f["table"], -np.ones((3, 1))], axis=1)
    st, ref = ({"pool": np.zeros(g.state_tensors[0].shape)} for _ in range(2))
    got, want = Simulator(g)._forward_pass(f, states=st), og.forward(g, f, states=ref)
    same(got, want, "layer")
    np.testing.assert_array_equal(st["pool"], ref["pool"])
    assert (got["o"][38:] == 0).all() and (got["o"][:38] != 0).any()


def test_captured_pass_replayed(torch_gpu):
    """forward_raw of a decode graph captured once: replays as the lengths grow, eager passes between
    them, every replay's rows and pools equal to the oracle's."""
    from cormorant_amd.simulate import Simulator
    torch = torch_gpu
    w = models.smollm2_weights(SHAPE, 3)
    exps = models.smollm2_decode(SHAPE, seed=3, weights=w)[2]
    g = models.smollm2_paged(SHAPE, 2, 2, 8, 16, 3, exps, w, with_head=True)
    sim = Simulator(g)
    name = g.output_tensors[0].onnx_name
    table = np.array([[6, 2, 0], [3, 5, 1]])
    rng = np.random.default_rng(4)
    ref = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    fs = [feeds(rng.integers(0, SHAPE.vocab, 2), [1, 1], [n, n + 14], table) for n in range(1, 6)]
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
    for i, f in enumerate(fs):
        for nm, v in f.items():
            dev[nm].copy_(sim._to_device(sim._tensor(nm), v))
        print(f"replay {i}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        want = og.forward(g, f, states=ref)
        np.testing.assert_array_equal(sim._to_values(sim._tensor(name), out), np.asarray(want[name]).reshape(2, -1))
        for nm in ref:
            np.testing.assert_array_equal(pools[nm].cpu().numpy().astype(np.float64), ref[nm].reshape(pools[nm].shape))
        sim.forward_raw({**{k: sim._to_device(sim._tensor(k), v) for k, v in f.items()},
                         **{k: v.clone() for k, v in pools.items()}}, keep=[name])
