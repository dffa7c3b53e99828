"""The paged cache's calls at the sizes that change their ways: more sequences than a wavefront has
lanes, more tiles than a workgroup plans, sequences of 2^20 rows (pieces of more keys than the int32
sums hold), pages that sequences share, graphs that share a workspace, heads alone and in large groups."""
import numpy as np
import pytest

from test_gpu_paged import Case, check_attention, check_prep, check_read, dev, paged, regs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,G", [(64, 3), (128, 8)])
@pytest.mark.parametrize("many", [False, True])
def test_more_than_64_sequences(paged, many, hd, G, int8):  # noqa: F811
    rng = np.random.default_rng(hd + G)
    lens = [int(x) for x in rng.integers(1, 90, 150)]
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 25 if many else 2, 150))]
    c = Case(rng, lens, new, kv=1, G=G, hd=hd, int8=int8, tail=3)
    check_attention(paged, c, *regs(hd))
    # the same over tables of more than 2048 rows
    c.table = np.concatenate([c.table, np.zeros((150, 140), np.int32)], axis=1)
    check_attention(paged, c, *regs(hd), window=33)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("batch", [1, 5, 64])
def test_more_than_256_tiles(paged, batch, int8):  # noqa: F811
    """8 heads a KV head: 275 tiles of 64 rows (head dim 128), behind windows that keep the keys few."""
    rng = np.random.default_rng(batch)
    new = [2200 // batch + (1 if b < 2200 % batch else 0) for b in range(batch)]
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 40, batch))]
    c = Case(rng, lens, new, kv=1, G=8, hd=128, page=32, int8=int8, tail=1)
    check_attention(paged, c, *regs(128), window=30)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,batch,kv", [(64, 300, 8), (64, 60, 40), (128, 300, 8)])
def test_several_tiles_a_share(paged, hd, batch, kv, int8):  # noqa: F811
    """2400 tiles of one or two steps: every workgroup has several whole ones between the ends of others."""
    rng = np.random.default_rng(batch)
    c = Case(rng, [int(x) for x in rng.integers(4, 100, batch)], [4] * batch, kv=kv, G=8, hd=hd, int8=int8)
    check_attention(paged, c, *regs(hd))


@pytest.mark.parametrize("kv,G,T", [(1, 1, 200), (5, 1, 3), (1, 40, 33), (2, 33, 1)])
def test_head_groups(paged, kv, G, T):  # noqa: F811
    c = Case(np.random.default_rng(G), [T + 70, 1], [T, 1], kv=kv, G=G)
    check_attention(paged, c, *regs())


def attend_repeated(pool, kv_len, ids, q, heads, cm, cfg):
    """The oracle's attention of the last tokens of one sequence of page ids ``ids`` (a few pages many
    times over): a row of a page weighs as often as its page stands below the token's position."""
    from oracle import paged as O
    tab, T, page = O.smx_tab(), len(q), pool.page
    G, cs, fp = heads // pool.kv, cfg & 63, (cfg >> 8) & 31
    o = np.zeros((T, heads, pool.hd), np.int64)
    rows = [[pool.read(i, s, g) for i in range(pool.pages) for s in range(page)] for g in range(pool.kv)]
    K, V = (np.stack([np.stack([r[w] for r in rows[g]]) for g in range(pool.kv)]) for w in (0, 1))
    for t in range(T):
        p = kv_len - T + t
        count = np.zeros((pool.pages, page), np.int64)
        np.add.at(count, ids[:(p + 1) // page], 1)
        if (p + 1) % page:
            count[ids[p // page], :(p + 1) % page] += 1
        n = count.reshape(-1)
        for h in range(heads):
            s = O.sat16(O.wrap32(K[h // G] @ q[t].reshape(heads, -1)[h].astype(np.int64)) >> 8)
            y = ((s[n > 0].max() - np.minimum(s, s[n > 0].max())) * cm) >> cs
            w = n * np.minimum(tab[y & 4095] >> np.minimum(y >> 12, 40), 65535)
            S, A = int(w.sum()), w @ V[h // G]
            num, den = (2 * (A << (fp - 8)) + S, 2 * S) if fp >= 8 else (2 * A + (S << (8 - fp)), S << (9 - fp))
            o[t, h] = O.sat16(num // den)
    return o.reshape(T, -1)


@pytest.mark.parametrize("hd,int8,kv,G,T", [
    (64, False, 1, 3, 1), (128, True, 2, 4, 3),              # few rows, their scores kept
    (64, False, 6, 3, 128), (64, True, 6, 3, 128), (128, False, 6, 3, 64), (128, True, 6, 3, 64),   # pieces of > 2^15 keys
    (64, False, 1, 1, 500),
])
def test_sequences_of_a_million_rows(paged, hd, int8, kv, G, T):  # noqa: F811
    """2^20 rows, the last partial page's rows among them, of 3 pages of 64 rows: every page 5461 times.
    Values at the ends of int16 in V: sums of 2^20 weights of 2^16 by 2^15, past 2^51."""
    import torch
    page, cap = 64, 1 << 20
    kv_len = cap - 5
    rng = np.random.default_rng(hd + T)
    c = Case(rng, [3 * page], [1], kv=kv, G=G, hd=hd, page=page, int8=int8, spare=0)
    for s in range(page):
        for g in range(kv):
            for i in range(3):
                k = np.clip(np.rint(rng.standard_normal(hd) * 60), -32768, 32767).astype(np.int64)
                c.pool.write(i, s, g, k, rng.choice([-32768, 32767, 1000], hd))
    ids = rng.integers(0, 3, cap // page)
    q = np.rint(rng.standard_normal((T, kv * G * hd)) * 300).astype(np.int16)
    cache = c.device(paged)[0]
    batch = paged.PagedBatch(dev(np.array([0, T], np.int32)), dev(np.array([kv_len], np.int32)),
                             dev(ids.astype(np.int32)[None]), T)
    o = torch.zeros((T, kv * G * hd), dtype=torch.int16, device="cuda")
    cm, cfg = regs(hd, 10, 8)
    print(f"hd {hd} int8 {int8} kv {kv} G {G} T {T}", flush=True)
    paged.paged_attention(cache, batch, dev(q), o, kv * G, cm, cfg)
    at = sorted({0, T // 2, T - 1})
    want = attend_repeated(c.pool, kv_len, ids, q, kv * G, cm, cfg) if T <= 3 else \
        np.concatenate([attend_repeated(c.pool, kv_len - T + 1 + t, ids, q[t:t + 1], kv * G, cm, cfg) for t in at])
    got = o.cpu().numpy()
    np.testing.assert_array_equal(got if T <= 3 else got[at], want)


@pytest.mark.parametrize("int8", [False, True])
def test_shared_pages(paged, int8):  # noqa: F811
    """Two sequences with the same first pages (a common prompt), a third with one page twice."""
    c = Case(np.random.default_rng(7), [90, 70, 64], [20, 1, 3], int8=int8)
    c.table[1, :3] = c.table[0, :3]
    c.table[2, 2] = c.table[2, 0]
    check_attention(paged, c, *regs())
    cache, batch = c.device(paged)
    check_read(paged, c, cache, batch)


@pytest.mark.parametrize("int8", [False, True])
def test_prep_and_read_of_many_sequences(paged, int8):  # noqa: F811
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(1, 60, 130)]
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 30, 130))]
    c = Case(rng, lens, new, kv=1, G=2, int8=int8, tail=2)
    cache, batch = check_prep(paged, c, rng, 64, False, False, True)
    check_read(paged, c, cache, batch, pad=8)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,rotary,interleaved,cols,norm,amp,in_place", [
    (64, 64, False, False, True, 400, False), (64, 32, True, True, True, 400, True), (128, 128, False, True, False, 40000, False),
    (128, 64, False, False, True, 40000, True), (64, 64, True, False, False, 400, False), (128, 128, True, True, True, 3, False),
])
def test_prep_of_many_tokens(paged, hd, rotary, interleaved, cols, norm, amp, in_place, int8):  # noqa: F811
    """5 passes a token, several passes and tokens a wavefront."""
    rng = np.random.default_rng(hd + rotary)
    kv, G = (4, 9) if hd == 64 else (4, 4)
    c = Case(rng, [700, 40, 1, 300], [600, 40, 1, 290], kv=kv, G=G, hd=hd, page=32, int8=int8, tail=5)
    cache, batch = check_prep(paged, c, rng, rotary, interleaved, cols, norm, amp=amp, in_place=in_place, pad=16)
    check_read(paged, c, cache, batch)


def test_two_captured_graphs_share_the_workspace(paged):  # noqa: F811
    """A graph of many rows and one of few over long tables, replayed in turn on one stream with other
    calls between them: each replay equal to its eager call."""
    import torch
    rng = np.random.default_rng(11)
    a = Case(rng, [700, 300], [200, 300], wide=150)
    b = Case(rng, [2500, 40], [1, 1], wide=20)
    runs = []
    for c in (a, b):
        cache, batch = c.device(paged)
        q = dev(c.q)
        o = torch.zeros_like(q)
        call = lambda cache=cache, batch=batch, q=q, o=o, c=c: paged.paged_attention(cache, batch, q, o, c.heads, *regs())  # noqa: E731
        call()
        want = o.clone()
        runs.append((call, o, want))
    torch.cuda.synchronize()
    graphs = []
    for call, _, _ in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    for i in range(3):
        for g, (call, o, want) in zip(graphs, runs):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want), f"replay {i}"
            runs[1 - i % 2][0]()
