"""The paged cache on the GPU, bit for bit against the 64-bit oracle (oracle/paged.py): the attention,
what stands before it and the read back, at the lengths, pages, strides, masks and values where
they can go wrong; the three together over the steps of a served batch; captured calls."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GUARD = 0x5A5A


@pytest.fixture(scope="module")
def paged():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cormorant_amd import paged as P
    return P


def dev(a, dtype=None):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda") if dtype is None else \
        torch.from_numpy(np.ascontiguousarray(a).astype(dtype)).to("cuda")


class Case:
    """Sequences of lengths ``lens`` with ``new`` new tokens each, in shuffled pages of a random pool."""

    def __init__(self, rng, lens, new, kv=2, G=3, hd=64, page=16, int8=False, tail=0, amp=400, spare=3, wide=0):
        from oracle import paged as O
        self.lens, self.new, self.kv, self.G, self.hd, self.page, self.int8 = lens, new, kv, G, hd, page, int8
        self.heads, self.T = kv * G, sum(new) + tail
        used = [-(-max(n, 1) // page) for n in lens]
        self.pages = sum(used) + spare
        self.table = np.full((len(lens), max(used) + wide), 0, np.int32)
        ids = rng.permutation(self.pages)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = ids[at:at + u]
            at += u
        self.q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kv_len = np.array(lens, np.int32)
        self.pool = O.Pool(self.pages, page, kv, hd, int8, rng.integers(0, 256, self.pages * kv * page *
                                                                        (2 * hd + 6 if int8 else 4 * hd + 4)))
        for b, n in enumerate(lens):
            for p in range(n):
                for g in range(kv):
                    k, v = (np.clip(np.rint(rng.standard_normal(hd) * amp), -32768, 32767).astype(np.int64)
                            for _ in range(2))
                    self.pool.write(int(self.table[b, p // page]), p % page, g, k, v)
        self.q = np.clip(np.rint(rng.standard_normal((self.T, self.heads * hd)) * amp), -32768, 32767).astype(np.int16)

    def device(self, P):
        cache = P.PagedCache(self.pages, self.page, self.kv, self.hd, self.int8, data=dev(self.pool.data.reshape(-1)))
        return cache, P.PagedBatch(dev(self.q_start), dev(self.kv_len), dev(self.table), self.T)


def regs(hd=64, f_s=9, f_p=14):
    from cormorant_amd.graph import softmax_regs
    return softmax_regs(f_s, 1.0 / np.sqrt(hd), f_p)


def check_attention(P, c, cm, cfg, window=0, q_pad=0, o_pad=0, q=None):
    import torch
    from oracle import paged as O
    cache, batch = c.device(P)
    W = c.heads * c.hd
    qd = torch.full((c.T, W + q_pad), GUARD, dtype=torch.int16, device="cuda")[:, q_pad // 2 // 8 * 8:][:, :W]
    qd.copy_(dev(c.q))
    ob = torch.full((c.T + 1, W + o_pad), GUARD, dtype=torch.int16, device="cuda")
    od = ob[:c.T, :W]
    P.paged_attention(cache, batch, qd, od, c.heads, cm, cfg, window=window)
    want = O.attend(c.pool, c.q_start, c.kv_len, c.table, c.q, c.heads, cm, cfg, window,
                    out=np.full((c.T, W), GUARD))
    got = ob.cpu().numpy()
    np.testing.assert_array_equal(got[:c.T, :W], want)
    assert (got[c.T:] == GUARD).all() and (got[:, W:] == GUARD).all()
    np.testing.assert_array_equal(cache.data.cpu().numpy(), c.pool.data.reshape(-1))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,new,page,G", [
    ([1], [1], 16, 1), ([17], [17], 16, 3), ([65, 1, 200], [1, 1, 1], 16, 3), ([300, 33], [40, 33], 32, 8),
    ([130, 5, 64], [3, 5, 64], 64, 4), ([63], [63], 128, 2), ([257], [20], 256, 7)])
def test_attention(paged, lens, new, page, G, hd, int8):
    rng = np.random.default_rng(len(lens) * 1000 + lens[0] + hd)
    c = Case(rng, lens, new, kv=2, G=G, hd=hd, page=page, int8=int8, tail=2, wide=1)
    check_attention(paged, c, *regs(hd))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,new,G,window", [([700, 90, 1], [1, 1, 1], 3, 0), ([530, 300], [2, 1], 16, 0),
                                               ([700, 5], [40, 5], 3, 0), ([650, 333], [70, 1], 4, 200)])
def test_attention_in_parts(paged, lens, new, G, window, hd, int8):
    """Tables of more than 2048 rows: a sequence's keys over several workgroups."""
    c = Case(np.random.default_rng(sum(lens) + hd), lens, new, kv=2, G=G, hd=hd, int8=int8, tail=1, wide=150)
    check_attention(paged, c, *regs(hd), window=window)


@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 1 << 20])
@pytest.mark.parametrize("int8", [False, True])
def test_attention_window(paged, window, int8):
    c = Case(np.random.default_rng(window), [210, 77, 3], [70, 1, 3], int8=int8)
    check_attention(paged, c, *regs(), window=window)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_rows_without_keys(paged, int8):
    """More tokens than the sequence is long (their positions negative), an empty sequence, no tokens."""
    c = Case(np.random.default_rng(5), [10, 40, 33, 20], [10, 0, 33, 20], int8=int8, tail=1)
    c.kv_len = np.array([4, 0, -7, 20], np.int32)
    check_attention(paged, c, *regs())


@pytest.mark.parametrize("int8", [False, True])
def test_attention_pages_outside_the_pool_are_masked(paged, int8):
    c = Case(np.random.default_rng(6), [120, 70, 20], [30, 1, 4], int8=int8)
    c.table[0, 2], c.table[0, 5], c.table[1, 0], c.table[2, :] = -1, c.pages, 2 ** 31 - 1, -2 ** 31
    check_attention(paged, c, *regs())
    c.kv_len = np.array([500, 90, 20], np.int32)         # positions past the table's pages
    for i in range(c.pages):                             # rows that no call wrote have no defined key term: write all
        for slot in range(c.page):
            for g in range(c.kv):
                c.pool.write(i, slot, g, *np.random.default_rng(i + slot).integers(-900, 900, (2, c.hd)))
    check_attention(paged, c, *regs())


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("fs,fp", [(3, 1), (6, 7), (8, 8), (10, 15), (12, 11)])
def test_attention_scales_and_large_values(paged, fs, fp, int8):
    """Scores that saturate and wrap, weights from every octave, outputs that saturate."""
    rng = np.random.default_rng(fs)
    c = Case(rng, [90, 66], [9, 1], int8=int8, amp=12000)
    check_attention(paged, c, *regs(64, fs, fp))
    c = Case(rng, [90], [5], int8=int8, amp=100000)     # mostly at the ends of int16
    c.q[:] = rng.choice([-32768, 32767, 0], c.q.shape)
    check_attention(paged, c, *regs(64, fs, fp))


@pytest.mark.parametrize("cm,cs", [(0, 20), (0, 63), (1, 0), (7, 0), ((1 << 24) - 1, 0), ((1 << 24) - 1, 7),
                                   (12345678, 8), ((1 << 24) - 1, 10), (65535, 0), (65536, 0), (69632, 0), (70000, 0), (12102203, 31),
                                   (8388608, 34), (16777215, 34), (5, 13)])
def test_attention_softmax_registers(paged, cm, cs):
    c = Case(np.random.default_rng(cs), [70], [7], amp=3000)
    check_attention(paged, c, cm, cs | (14 << 8))


def test_attention_equal_keys(paged):
    """Every weight at its largest: the sums' largest terms, the quotient exactly V."""
    c = Case(np.random.default_rng(3), [400], [2])
    for p in range(400):
        for g in range(c.kv):
            c.pool.write(int(c.table[0, p // 16]), p % 16, g, np.zeros(64, np.int64), np.full(64, -32768 if p % 2 else 32767))
    check_attention(paged, c, *regs(64, 9, 8))


def test_attention_strided_rows(paged):
    c = Case(np.random.default_rng(8), [50, 20], [20, 20])
    check_attention(paged, c, *regs(), q_pad=64, o_pad=24)


# ---------------------------------------------------------------- prep and read
def prep_params(rng, heads, hd, cols, norm):
    """(bytes, oracle triple) of a rotation's and a norm's parameter entries."""
    from cormorant_amd.rowops_nodes import param_block
    n = heads * hd if cols else 1
    sa, sb, sc = rng.integers(0, 3, n), rng.integers(0, 3, n), rng.integers(21, 26, n)
    shape = (heads, hd) if cols else (1, 1)
    rope = param_block(np.zeros(n), 0, sa, sb, sc), tuple(x.astype(np.int64).reshape(shape) for x in (sa, sb, sc))
    if not norm:
        return rope, None
    G, Bq, sh = rng.integers(1 << 18, 1 << 23, hd), rng.integers(-9, 9, hd), rng.integers(33, 36, hd)
    return rope, (param_block(G, Bq, 0, 0, sh), (G.astype(np.int64), Bq.astype(np.int64), sh.astype(np.int64)))


def check_prep(P, c, rng, rotary, interleaved, cols, norm, rows=None, eps=(7, 1 << 40), in_place=False, pad=0, amp=400):
    import torch
    from oracle import paged as O
    hd, W, KW = c.hd, c.heads * c.hd, c.kv * c.hd
    rows = rows or max(c.lens) + 1
    ang = rng.standard_normal((rows, rotary)) * 3
    tab = np.concatenate([np.rint(np.cos(ang) * 2 ** 23), np.rint(np.sin(ang) * 2 ** 23)], 1).astype(np.int32)
    draw = lambda w: np.clip(np.rint(rng.standard_normal((c.T, w)) * amp), -32768, 32767).astype(np.int16)  # noqa: E731
    fused = draw(W + 2 * KW + pad)
    (rq, oq), nq = prep_params(rng, c.heads, hd, cols, norm)
    (rk, ok), nk = prep_params(rng, c.kv, hd, cols, norm)
    cache, batch = c.device(P)
    prep = P.PagedPrep(dev(tab), dev(rq), dev(rk), interleaved, dev(nq[0]) if norm else None,
                       dev(nk[0]) if norm else None, eps[0], eps[1])
    f = dev(fused)
    q, k, v = f[:, :W], f[:, W:W + KW], f[:, W + KW:W + 2 * KW]
    qr = q if in_place else torch.full((c.T, W), GUARD, dtype=torch.int16, device="cuda")
    P.paged_prep(cache, batch, prep, q, k, v, qr)
    want = fused[:, :W].astype(np.int64).copy() if in_place else np.full((c.T, W), GUARD, np.int64)
    O.prep(c.pool, c.q_start, c.kv_len, c.table, fused[:, :W], fused[:, W:W + KW], fused[:, W + KW:W + 2 * KW], want, tab,
           rotary, interleaved, oq, ok, nq[1] if norm else None, nk[1] if norm else None, *eps)
    np.testing.assert_array_equal(qr.cpu().numpy(), want)
    np.testing.assert_array_equal(cache.data.cpu().numpy(), c.pool.data.reshape(-1))
    return cache, batch


def check_read(P, c, cache, batch, pad=0):
    import torch
    from oracle import paged as O
    KW = c.kv * c.hd
    k, v = (torch.full((c.T + 1, KW + pad), GUARD, dtype=torch.int16, device="cuda") for _ in range(2))
    P.paged_read(cache, batch, k[:c.T, :KW], v[:c.T, :KW])
    wk, wv = np.full((c.T, KW), GUARD), np.full((c.T, KW), GUARD)
    O.read(c.pool, c.q_start, c.kv_len, c.table, wk, wv)
    for got, want in ((k, wk), (v, wv)):
        got = got.cpu().numpy()
        np.testing.assert_array_equal(got[:c.T, :KW], want)
        assert (got[c.T:] == GUARD).all() and (got[:, KW:] == GUARD).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd,rotary,interleaved,cols,norm", [
    (64, 64, False, False, False), (64, 64, True, True, True), (64, 32, False, True, True), (64, 16, True, False, False),
    (128, 128, False, False, True), (128, 128, True, False, True), (128, 32, False, True, False),
    (128, 48, True, True, True)])
@pytest.mark.parametrize("lens,new,page", [([1], [1], 16), ([37, 5, 70], [20, 1, 70], 32), ([40, 1, 129, 16], [40, 1, 3, 16], 16)])
def test_prep_and_read(paged, hd, rotary, interleaved, cols, norm, lens, new, page, int8):
    rng = np.random.default_rng(hd + rotary + lens[0])
    c = Case(rng, lens, new, kv=2, G=3, hd=hd, page=page, int8=int8, tail=1)
    cache, batch = check_prep(paged, c, rng, rotary, interleaved, cols, norm)
    check_read(paged, c, cache, batch, pad=8)


@pytest.mark.parametrize("int8", [False, True])
def test_prep_extremes(paged, int8):
    """int16's ends, rows of zeros, a table shorter than the positions, positions without a page."""
    rng = np.random.default_rng(9)
    c = Case(rng, [60, 33, 20, 9], [60, 33, 20, 9], int8=int8)
    check_prep(paged, c, rng, 64, False, True, True, amp=60000, eps=(0, 0))
    check_prep(paged, c, rng, 32, True, False, False, rows=7, amp=0)
    c.table[0, 1], c.table[1, 0] = -1, c.pages
    c.kv_len = np.array([60, 40, 3, 0], np.int32)        # past the table, more tokens than rows, none at all
    cache, batch = check_prep(paged, c, rng, 64, False, False, True, in_place=True, pad=16)
    check_read(paged, c, cache, batch)


def test_prep_equals_the_row_ops_jobs(paged):
    """Per head the NORM job then the ROPE job of the row-ops unit (cm_rowops) on the same rows."""
    import torch
    from cormorant_amd import units
    from cormorant_amd.rowops_nodes import K_I16, K_I32, RO_NORM, RO_ROPE, norm_params, opword, param_block
    rng = np.random.default_rng(12)
    T, kv, G, hd = 19, 2, 3, 64
    c = Case(rng, [30], [T], kv=kv, G=G, hd=hd)
    H = kv * G
    tab = np.rint(rng.uniform(-1, 1, (30, 2 * hd)) * 2 ** 23).astype(np.int32)
    x = [np.rint(rng.standard_normal((T, w * hd)) * 500).astype(np.int16) for w in (H, kv, kv)]
    Gm, g, _, E = norm_params(1 + 0.1 * rng.standard_normal(hd), hd, 1e-5, 9, rms=True)
    np_, rp = param_block(Gm, 0, 0, 0, 24 + g - 9), param_block(0, 0, 0, 0, 23)
    cache, batch = c.device(paged)
    prep = paged.PagedPrep(dev(tab), dev(rp), dev(rp), False, dev(np_), dev(np_), E, E)
    qr = torch.zeros((T, H * hd), dtype=torch.int16, device="cuda")
    paged.paged_prep(cache, batch, prep, *[dev(a) for a in x], qr)
    k, v = (torch.zeros((T, kv * hd), dtype=torch.int16, device="cuda") for _ in range(2))
    paged.paged_read(cache, batch, k, v)
    for rows, got in ((x[0], qr), (x[1], k)):
        n = rows.size // hd
        y, z = (torch.zeros(n * hd + 16, dtype=torch.int16, device="cuda") for _ in range(2))
        b8 = lambda t: t.view(torch.uint8)              # noqa: E731
        units.rowops(b8(dev(rows).reshape(-1)), None, b8(y), dev(np_), opword(RO_NORM, K_I16, K_I16, K_I16), hd, n, 1,
                     2 * hd, 0, 0, 0, 2 * hd, 0, eps=E)
        tr = dev(np.repeat(tab[30 - T:30], rows.shape[1] // hd, 0))
        units.rowops(b8(y), b8(tr.reshape(-1)), b8(z), dev(rp), opword(RO_ROPE, K_I16, K_I32, K_I16, b_en=True, p_bcast=True),
                     hd, n, 1, 2 * hd, 0, 8 * hd, 0, 2 * hd, 0, aux=hd)
        np.testing.assert_array_equal(got.cpu().numpy().reshape(-1), z.cpu().numpy()[:n * hd])
    np.testing.assert_array_equal(v.cpu().numpy(), x[2])


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("int8", [False, True])
def test_steps_of_a_served_batch(paged, int8):
    """Prompts in chunks, then single tokens, sequences joining and growing across pages: prep, attention
    and read in turn on one pool, every output and the pool's bytes after each step."""
    import torch
    from cormorant_amd.rowops_nodes import param_block
    from oracle import paged as O
    rng = np.random.default_rng(31)
    kv, G, hd, page, pages = 2, 3, 64, 16, 40
    H, cm, cfg = kv * G, *regs()
    pool = O.Pool(pages, page, kv, hd, int8, rng.integers(0, 256, pages * kv * page * (2 * hd + 6 if int8 else 4 * hd + 4)))
    table = rng.permutation(pages)[:36].reshape(3, 12).astype(np.int32)
    tab = np.rint(rng.uniform(-1, 1, (192, 2 * hd)) * 2 ** 23).astype(np.int32)
    rp = param_block(0, 0, 0, 0, 23)
    sh = tuple(np.array([[s]], np.int64) for s in (0, 0, 23))
    cache = paged.PagedCache(pages, page, kv, hd, int8, data=dev(pool.data.reshape(-1)))
    prep = paged.PagedPrep(dev(tab), dev(rp), dev(rp))
    lens = np.zeros(3, np.int32)
    for new in ([40, 0, 1], [25, 30, 1], [1, 1, 0], [1, 70, 1], [1, 1, 1]):
        T = sum(new)
        lens += np.array(new, np.int32)
        qs = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        x = [np.rint(rng.standard_normal((T, w * hd)) * 300).astype(np.int16) for w in (H, kv, kv)]
        batch = paged.PagedBatch(dev(qs), dev(lens), dev(table), T)
        qr = torch.zeros((T, H * hd), dtype=torch.int16, device="cuda")
        o, k, v = torch.zeros_like(qr), *(torch.zeros((T, kv * hd), dtype=torch.int16, device="cuda") for _ in range(2))
        paged.paged_prep(cache, batch, prep, *[dev(a) for a in x], qr)
        paged.paged_attention(cache, batch, qr, o, H, cm, cfg)
        paged.paged_read(cache, batch, k, v)
        wq = np.zeros((T, H * hd), np.int64)
        O.prep(pool, qs, lens, table, *x, wq, tab, hd, False, sh, sh)
        np.testing.assert_array_equal(qr.cpu().numpy(), wq)
        np.testing.assert_array_equal(cache.data.cpu().numpy(), pool.data.reshape(-1))
        np.testing.assert_array_equal(o.cpu().numpy(), O.attend(pool, qs, lens, table, wq, H, cm, cfg))
        wk, wv = np.zeros((T, kv * hd), np.int64), np.zeros((T, kv * hd), np.int64)
        O.read(pool, qs, lens, table, wk, wv)
        np.testing.assert_array_equal(k.cpu().numpy(), wk)
        np.testing.assert_array_equal(v.cpu().numpy(), wv)


def test_against_the_contiguous_decode_step(paged):
    """One decode step beside units.decode_prep / decode_attention on contiguous caches of the same rows:
    the rotated q and the cache rows equal; o apart by the unit's rounding of P alone.

    P_j is e_j 2^fp / S rounded to an integer, off by 1/2 + 2^-9 at most (R = floor(2^40 / S): e_j 2^fp /
    2^40 <= 2^-10 at fp = 14); the weights take the largest e, 65536, as 65535, which moves a
    weight's share by at most 2^-15 of 2^fp = 1/2.  So |o - o'| <= (0.51 + 0.5) sum_j |V_j| / 256 + 2 (the
    floor of one, the half of the other)."""
    import torch
    from cormorant_amd import units
    from cormorant_amd.rowops_nodes import K_I16, K_I32, RO_ROPE, opword, param_block
    rng = np.random.default_rng(77)
    B, kv, G, hd, C = 3, 2, 3, 64, 128
    H, pos = kv * G, C - 1
    cm, cfg = regs(64, 10, 14)
    tab = np.rint(rng.uniform(-0.7, 0.7, (C, 2 * hd)) * 2 ** 23).astype(np.int32)
    kc, vc = (np.rint(rng.standard_normal((B, kv, C, hd)) * 300).astype(np.int16) for _ in range(2))
    c = Case(rng, [C] * B, [1] * B, kv=kv, G=G)
    for b in range(B):
        for p in range(C):
            for g in range(kv):
                c.pool.write(int(c.table[b, p // 16]), p % 16, g, kc[b, g, p].astype(np.int64), vc[b, g, p].astype(np.int64))
    x = [np.rint(rng.standard_normal((B, w * hd)) * 300).astype(np.int16) for w in (H, kv, kv)]
    rp = dev(param_block(0, 0, 0, 0, 23))
    op = opword(RO_ROPE, K_I16, K_I32, K_I16, b_en=True, p_bcast=True)
    q0, o0 = (torch.zeros((B, H * hd), dtype=torch.int16, device="cuda") for _ in range(2))
    kd, vd = dev(kc), dev(vc)
    units.decode_prep(*[dev(a).reshape(-1) for a in x], q0.view(-1), kd.view(-1), C, vd.view(-1), B, H, kv, hd, pos, dev(tab)[pos], rp, op, rp, op)
    units.decode_attention(q0.view(-1), kd.view(-1), vd.view(-1), o0.view(-1), B * kv, G, C, cm, cfg, C)
    cache, batch = c.device(paged)
    q1, o1 = torch.zeros_like(q0), torch.zeros_like(q0)
    paged.paged_prep(cache, batch, paged.PagedPrep(dev(tab), rp, rp), *[dev(a) for a in x], q1)
    paged.paged_attention(cache, batch, q1, o1, H, cm, cfg)
    assert torch.equal(q0, q1)
    whole = paged.PagedBatch(dev(np.arange(B + 1) * C, np.int32), batch.kv_len, batch.table, B * C)
    k, v = (torch.zeros((B * C, kv * hd), dtype=torch.int16, device="cuda") for _ in range(2))
    paged.paged_read(cache, whole, k, v)
    for got, want in ((k, kd), (v, vd)):
        assert torch.equal(got.view(B, C, kv, hd).transpose(1, 2), want.view(B, kv, C, hd))
    bound = 1.01 * np.abs(vd.cpu().numpy().astype(np.int64)).sum(2) / 256 + 2          # [B][kv][hd]
    diff = np.abs(o0.cpu().numpy().astype(np.int64) - o1.cpu().numpy()).reshape(B, kv, G, hd)
    assert (diff <= bound[:, :, None]).all()


@pytest.mark.parametrize("lens,new", [([90, 30], [1, 1]), ([100, 64], [40, 64])])
def test_captured_step_replays_over_new_lengths(paged, lens, new):
    """prep and attention captured once; replays with other rows, lengths and pages in the same buffers,
    eager work between them, equal to the eager calls."""
    import torch
    from cormorant_amd.rowops_nodes import param_block
    rng = np.random.default_rng(3)
    c = Case(rng, lens, new, wide=2)
    cache, batch = c.device(paged)
    cm, cfg = regs()
    tab = np.rint(rng.uniform(-1, 1, (200, 128)) * 2 ** 23).astype(np.int32)
    prep = paged.PagedPrep(dev(tab), dev(param_block(0, 0, 0, 0, 23)), dev(param_block(0, 0, 0, 0, 23)))
    x = [dev(np.rint(rng.standard_normal((c.T, w * 64)) * 300).astype(np.int16)) for w in (6, 2, 2)]
    qr, o = torch.zeros_like(x[0]), torch.zeros_like(x[0])

    def step():
        paged.paged_prep(cache, batch, prep, *x, qr)
        paged.paged_attention(cache, batch, qr, o, 6, cm, cfg)
    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        for t in x:
            t.copy_(dev(np.rint(rng.standard_normal(tuple(t.shape)) * 300).astype(np.int16)))
        batch.kv_len.copy_(dev(np.array([max(n, l - 9 * i) for n, l in zip(new, lens)], np.int32)))
        batch.table.copy_(dev(rng.permutation(c.pages)[c.table].astype(np.int32)))
        before = cache.data.clone()
        step()
        want, pool = o.clone(), cache.data.clone()
        cache.data.copy_(before)
        o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want), f"replay {i}"
        assert torch.equal(cache.data, pool), f"replay {i}: the pool"


def test_another_stream(paged):
    import torch
    from oracle import paged as O
    c = Case(np.random.default_rng(4), [100], [33])
    cache, batch = c.device(paged)
    q = dev(c.q)
    o = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged.paged_attention(cache, batch, q, o, c.heads, *regs())
    s.synchronize()
    np.testing.assert_array_equal(o.cpu().numpy(), O.attend(c.pool, c.q_start, c.kv_len, c.table, c.q, c.heads, *regs()))


def test_pool_past_32_bit_offsets(paged):
    """Pages whose byte offsets pass 2^32: written, attended to and read back in place."""
    import torch
    from cormorant_amd.rowops_nodes import param_block
    from oracle import paged as O
    kv, hd, page = 2, 64, 64
    pages = (1 << 32) // (kv * page * (4 * hd + 4)) + 40
    cache = paged.PagedCache(pages, page, kv, hd)
    rng = np.random.default_rng(1)
    T = 100
    ids = np.array([[pages - 1, pages - 3]], np.int32)
    small = O.Pool(2, page, kv, hd, False)
    tab = np.rint(rng.uniform(-1, 1, (T, 128)) * 2 ** 23).astype(np.int32)
    x = [np.rint(rng.standard_normal((T, w * hd)) * 300).astype(np.int16) for w in (2, kv, kv)]
    qs, lens = np.array([0, T], np.int32), np.array([T], np.int32)
    batch = paged.PagedBatch(dev(qs), dev(lens), dev(ids), T)
    rp = dev(param_block(0, 0, 0, 0, 23))
    qr = torch.zeros((T, 2 * hd), dtype=torch.int16, device="cuda")
    o = torch.zeros_like(qr)
    paged.paged_prep(cache, batch, paged.PagedPrep(dev(tab), rp, rp), *[dev(a) for a in x], qr)
    paged.paged_attention(cache, batch, qr, o, 2, *regs())
    k, v = (torch.zeros((T, kv * hd), dtype=torch.int16, device="cuda") for _ in range(2))
    paged.paged_read(cache, batch, k, v)
    wq, small_ids = np.zeros((T, 2 * hd), np.int64), np.array([[0, 1]], np.int32)
    sh = tuple(np.array([[s]], np.int64) for s in (0, 0, 23))
    O.prep(small, qs, lens, small_ids, *x, wq, tab, hd, False, sh, sh)
    np.testing.assert_array_equal(o.cpu().numpy(), O.attend(small, qs, lens, small_ids, wq, 2, *regs()))
    np.testing.assert_array_equal(v.cpu().numpy(), x[2])
    block = kv * page * (4 * hd + 4)
    got = torch.stack([cache.data[i * block:(i + 1) * block] for i in (pages - 1, pages - 3)])
    np.testing.assert_array_equal(got.cpu().numpy().reshape(-1), small.data.reshape(-1))
    assert not cache.data[:block].any() and not cache.data[(pages - 2) * block:(pages - 1) * block].any()
