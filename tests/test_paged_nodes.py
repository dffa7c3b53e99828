"""The paged serving entry (models.smollm2_paged) on the CPU: its graph by the oracle's forward pass --
packed sequences against the same sequences alone, chunks against whole prompts --, the front end's
nodes for its op list, and the nodes' refusals."""
import numpy as np
import pytest

from cormorant_amd import models
from cormorant_amd.frontend import build_graph
from cormorant_amd.graph import PagedAttentionNode, SchedulerError, TensorInfo, paged_pool
from cormorant_amd.rowops_nodes import PagedPrepNode, rope_table
from oracle import graph_sim as og

SHAPE = models.LlamaShape(layers=2, batch=2, d=128, heads=2, kv=1, hd=64, ff=128, vocab=256, ctx=64)


@pytest.fixture(scope="module")
def small():
    w = models.smollm2_weights(SHAPE, 3)
    return w, models.smollm2_decode(SHAPE, seed=3, weights=w)[2]


def feeds(ids, new, kv, table):
    return {"ids": np.asarray(ids, np.float64), "q_start": np.concatenate([[0], np.cumsum(new)]).astype(np.float64),
            "kv_len": np.asarray(kv, np.float64), "table": np.asarray(table, np.float64)}


def entry(small, tokens, batch, **kw):
    return models.smollm2_paged(SHAPE, tokens, batch, 8, 16, 3, small[1], small[0], **kw)


@pytest.mark.parametrize("int8", [False, True])
def test_packed_rows_are_the_sequences_alone_and_chunks_the_prompt(small, int8):
    """h of two packed prompts (one row of padding behind them), of each alone, and of the first in two
    chunks: the same rows (every row's arithmetic is its own), and the same pages."""
    rng = np.random.default_rng(5)
    ids = rng.integers(0, SHAPE.vocab, 30)
    table = np.array([[3, 1, 6], [0, 7, 2]])
    g = entry(small, 30, 2, int8=int8)
    st = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    assert sorted(st) == ["l0.pool", "l1.pool"]
    both = og.forward(g, feeds(ids, [18, 11], [18, 11], table), states=st)["l1.h"]
    alone = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    first = og.forward(entry(small, 18, 1, int8=int8), feeds(ids[:18], [18], [18], table[:1]), states=alone)["l1.h"]
    np.testing.assert_array_equal(both[:18], first)
    second = og.forward(entry(small, 11, 1, int8=int8), feeds(ids[18:29], [11], [11], table[1:]), states=alone)["l1.h"]
    np.testing.assert_array_equal(both[18:29], second)
    chunks = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    a = og.forward(entry(small, 5, 1, int8=int8), feeds(ids[:5], [5], [5], table[:1]), states=chunks)["l1.h"]
    b = og.forward(entry(small, 13, 1, int8=int8), feeds(ids[5:18], [13], [18], table[:1]), states=chunks)["l1.h"]
    np.testing.assert_array_equal(both[:18], np.concatenate([a, b]))
    for nm in st:
        np.testing.assert_array_equal(st[nm], alone[nm])
        assert (chunks[nm][[3, 1]] == st[nm][[3, 1]]).all() and (st[nm][3] != 0).any() and (st[nm][[4, 5]] == 0).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("with_head", [False, True])
def test_front_end_builds_the_same_nodes(small, int8, with_head):
    kw = dict(int8=int8, window=7, with_head=with_head)
    g = entry(small, 4, 2, **kw)
    ops, tensors, ins, outs = entry(small, 4, 2, as_ops=True, **kw)
    f = build_graph(ops, tensors, ins, outs)
    assert [type(n).__name__ for n in f.nodes] == [type(n).__name__ for n in g.nodes]
    rng = np.random.default_rng(6)
    fd = feeds(rng.integers(0, SHAPE.vocab, 4), [1, 3], [1, 3], [[0, 1, 2], [3, 4, 5]])
    name = outs[0]
    np.testing.assert_array_equal(og.forward(f, fd)[name], og.forward(g, fd)[name])


def tensors(heads=2, kv=1, hd=64, page=16, int8=False, batch=2, f=8):
    T = TensorInfo
    return ([T("q", [4, heads * hd], exp=f), T("k", [4, kv * hd], exp=f), T("v", [4, kv * hd], exp=f),
             paged_pool("pool", 4, page, kv, hd, int8), T("qs", [batch + 1], kind="i32"), T("kl", [batch], kind="i32"),
             T("tb", [batch, 2], kind="i32")], T("qr", [4, heads * hd], exp=f))


def tables(rotary=64, n=32):
    return models.rope_half_tables(1e4, rotary, n)


def test_prep_refusals():
    cos, sin = tables()
    ins, qr = tensors()
    ok = dict(heads=2, kv_heads=1, head_dim=64, page=16, cos=cos, sin=sin)
    node = PagedPrepNode(ins, qr, **ok)
    assert node.norm_q is None and node.table.shape == [32, 128]
    for kw, msg in ((dict(page=24), "pages of 24"), (dict(page=32), "a pool of shape"), (dict(int8=True), "a pool of shape"),
                    (dict(heads=3), "shapes"), (dict(f_v=7), "V cache's exponent"), (dict(f_k=40), "RoPE exponents"),
                    (dict(cos=cos[:, :12], sin=sin[:, :12]), "multiple of 16"), (dict(gamma_q=np.ones(32)), "gamma over")):
        with pytest.raises(SchedulerError, match=msg):
            PagedPrepNode(ins, qr, **{**ok, **kw})
    with pytest.raises(SchedulerError, match="q_start"):
        PagedPrepNode(ins[:4] + [TensorInfo("qs", [2], kind="i32")] + ins[5:], qr, **ok)
    per_head = TensorInfo("q", [4, 128], exp=np.repeat([8, 9], 64))
    with pytest.raises(SchedulerError, match="one exponent"):
        PagedPrepNode([per_head] + ins[1:], qr, **ok)
    wide = dict(ok, heads=2, head_dim=128, cos=tables(256)[0], sin=tables(256)[1])
    with pytest.raises(SchedulerError, match="up to the head dim"):
        PagedPrepNode(tensors(hd=128)[0], tensors(hd=128)[1], **wide)


def test_attention_refusals():
    ins, qr = tensors()
    o = TensorInfo("o", [4, 128], exp=8)
    ok = dict(heads=2, kv_heads=1, head_dim=64, page=16)
    PagedAttentionNode([qr] + ins[3:], o, **ok)
    for kw, msg in ((dict(heads=3), "q \\["), (dict(window=-1), "window"), (dict(head_dim=32, heads=4), "head dim 32"),
                    (dict(kv_heads=3), "heads over"), (dict(int8=True), "a pool of shape")):
        with pytest.raises(SchedulerError, match=msg):
            PagedAttentionNode([qr] + ins[3:], o, **{**ok, **kw})


def test_interleaved_table():
    cos, sin = tables(32, 5)
    t = rope_table(cos, sin, interleaved=True)
    half = rope_table(cos, sin)
    assert t.shape == half.shape == (5, 64)
    for j in range(16):
        for at in (2 * j, 2 * j + 1):
            assert (t[:, at] == half[:, j]).all() and (t[:, 32 + at] == half[:, 32 + j]).all()
