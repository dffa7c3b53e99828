"""The paged cache's calls at the ends of what their contract allows: lengths that no table holds, the workspace that small
decode steps use, serving entries that share their weights."""
import numpy as np
import pytest

from test_gpu_paged import Case, check_prep, check_read, dev, paged, regs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths", [(2 ** 31 - 1, 2 ** 31 - 1), (40, 2 ** 31 - 64), (2 ** 30 + 1, 2 ** 31 - 200), (2 ** 31 - 1, 40)])
def test_lengths_past_every_table(paged, lengths, hd, int8):  # noqa: F811
    """kv_len up to 2^31 - 1, in front of more rows of padding than the table has: nothing of such a sequence is
    written, its rows are read back as 0, the other's as they are.  Its tokens attend to every row of the table."""
    import torch
    rng = np.random.default_rng(hd)
    c = Case(rng, [40, 30], [5, 3], hd=hd, int8=int8, tail=1500)
    c.kv_len = np.array(lengths, np.int32)
    cache, batch = check_prep(paged, c, rng, hd, False, False, True, rows=70)
    check_read(paged, c, cache, batch)
    attends_to_the_table(paged, c, lengths)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,wide", [((1, 1), 150), ((60, 3), 4000)])
def test_lengths_past_long_tables(paged, new, wide, hd, int8):  # noqa: F811
    """The attention's other two ways."""
    c = Case(np.random.default_rng(wide), [70, 64], list(new), kv=4, hd=hd, int8=int8, tail=1, wide=wide)
    attends_to_the_table(paged, c, (2 ** 31 - 1, 64))


def attends_to_the_table(P, c, lengths):
    """The tokens of a sequence longer than its table: the same keys as at a length whose new tokens stand just past it."""
    import torch
    cap = c.table.shape[1] * c.page
    q, o, want = dev(c.q), *(torch.zeros((c.T, c.heads * c.hd), dtype=torch.int16, device="cuda") for _ in range(2))
    for kv, out in ((lengths, o), ([cap + n if x > cap else x for x, n in zip(lengths, c.new)], want)):
        c.kv_len = np.array(kv, np.int32)
        cache, batch = c.device(P)
        P.paged_attention(cache, batch, q, out, c.heads, *regs(c.hd))
    assert torch.equal(o, want) and o[:c.new[0]].any()


@pytest.mark.parametrize("first", ["decode", "paged", "wide"])
def test_entries_that_share_weights(paged, first):  # noqa: F811
    """A decode entry and paged entries over tables of 3 and 6 pages with one set of device weights, whichever comes first:
    each one's pass is the oracle's."""
    from cormorant_amd import models
    from cormorant_amd.simulate import Simulator
    from oracle import graph_sim as og
    from test_gpu_paged_nodes import SHAPE, feeds, same
    w = models.smollm2_weights(SHAPE, 3)
    decode, inputs, exps = models.smollm2_decode(SHAPE, seed=3, weights=w, runtime_pos=True)
    graphs = {"decode": decode, **{k: models.smollm2_paged(SHAPE, 9, 2, 14, 16, n, exps, w) for k, n in (("paged", 3), ("wide", 6))}}
    rng = np.random.default_rng(2)
    sims, held = {}, None
    for k in sorted(graphs, key=lambda k: k != first):
        g = graphs[k]
        sims[k] = held = Simulator(g, share=held)
        states = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
        n = 0 if k == "decode" else int(g.input_tensors[-1].shape[1])
        f = feeds(rng.integers(0, SHAPE.vocab, 9), [8, 1], [16 * n, 8 * n], rng.permutation(14)[:2 * n].reshape(2, n)) if n else \
            {t.onnx_name: inputs[t.onnx_name] for t in g.input_tensors if t.onnx_name not in states}
        ref = {nm: v.copy() for nm, v in states.items()}
        print(f"{k} behind {first}", flush=True)
        got, want = sims[k]._forward_pass(f, states=states), og.forward(g, f, states=ref)
        same(got, want, k)
        for nm in ref:
            np.testing.assert_array_equal(states[nm], ref[nm], err_msg=f"{k}: {nm}")


@pytest.mark.parametrize("hd,kv,G,batch,page,int8", [(128, 8, 4, 128, 64, True), (128, 8, 4, 128, 128, False), (64, 5, 3, 512, 64, False),
                                                     (64, 8, 1, 512, 64, True)])
def test_single_tokens_in_the_workspace(paged, hd, kv, G, batch, page, int8):  # noqa: F811
    """Decode steps of many sequences over tables of one page: few rows a sequence, short tables, and yet the kernels that
    share the device's workspace.  One call, then captured and replayed as the lengths change, beside other calls there."""
    import torch
    from cormorant_amd import _lib
    from oracle import paged as O
    rng = np.random.default_rng(batch + hd)
    c = Case(rng, [int(x) for x in rng.integers(1, page + 1, batch)], [1] * batch, kv=kv, G=G, hd=hd, page=page, int8=int8)
    other = Case(rng, [70], [50], kv=4)
    q, oq = dev(c.q), dev(other.q)
    o, oo = torch.zeros_like(q), torch.zeros_like(oq)
    cache, step = c.device(paged)
    beside = other.device(paged)
    call = lambda: paged.paged_attention(cache, step, q, o, c.heads, *regs(hd))     # noqa: E731
    _lib.timing_reset()
    _lib.timing_enable(True)
    try:
        call()
        assert _lib.timing_read("paged_rows_kernel")[1] == 1 and _lib.timing_read("paged_short_kernel")[1] == 0
    finally:
        _lib.timing_enable(False)
        _lib.timing_reset()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for i in range(3):
        print(f"replay {i}", flush=True)
        step.kv_len.copy_(dev(np.maximum(c.kv_len - 7 * i, 1).astype(np.int32)))
        o.zero_()
        graph.replay()
        want = O.attend(c.pool, c.q_start, np.maximum(c.kv_len - 7 * i, 1), c.table, c.q, c.heads, *regs(hd))
        np.testing.assert_array_equal(o.cpu().numpy(), want)
        paged.paged_attention(*beside, oq, oo, other.heads, *regs())


def test_steps_over_growing_tables(paged):  # noqa: F811
    """24 single tokens of 32 + 8 heads over tables that widen by a page at a time: the workspaces allocated on the way
    stay within four of the last request (each at least doubles the one before; one twice the request at most)."""
    import torch
    B, kv, G, hd, page = 24, 8, 4, 128, 4096
    heads = kv * G
    cache = paged.PagedCache(1, page, kv, hd, int8=True)
    q = torch.zeros((B, heads * hd), dtype=torch.int16, device="cuda")
    o = torch.ones_like(q)
    step = [dev(np.arange(B + 1, dtype=np.int32)), dev(np.full(B, 5, np.int32))]
    tables = [dev(np.zeros((B, n), np.int32)) for n in range(8, 33)]
    torch.cuda.synchronize()
    before, last = torch.cuda.mem_get_info()[0], 0
    for table in tables:
        cap = table.shape[1] * page
        paged.paged_attention(cache, paged.PagedBatch(*step, table, B), q, o, heads, *regs(hd))
        last = B * heads * 2 * cap * 1.1        # the scores; the maxima and eight parts' sums are less than a tenth of them
    torch.cuda.synchronize()
    grown = before - torch.cuda.mem_get_info()[0]
    assert not o.any() and grown <= 4 * last + (64 << 20), (grown, last)
