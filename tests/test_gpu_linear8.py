"""The 8-bit linear layers on the GPU, bit for bit against the oracle in whole numbers (oracle/linear8.py):
sizes from one row and column on, odd widths and strides, values at the ends of their ranges, ties,
shared codes, in-place residuals, a feed-forward block of both, captured calls."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GUARD16, GUARD32 = 0x5A5A, 0x5A5A5A5A


@pytest.fixture(scope="module")
def L():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cormorant_amd import linear8
    return linear8


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def rows(rng, n, k, amp=400):
    x = np.clip(np.rint(rng.standard_normal((n, k)) * amp * np.exp(0.7 * rng.standard_normal((n, 1)))), -32768, 32767)
    return x.astype(np.int16)


def weights(rng, k, m, std=300.0):
    """(codes, multipliers of 18 bits): outputs of about ``std`` for rows of about 400."""
    w = rng.integers(-127, 128, (k, m)).astype(np.int8)
    mu = std / (400.0 * 4 * 36.0 * 73.0 * np.sqrt(k)) * np.exp(0.3 * rng.standard_normal(m))
    man, e = np.frexp(mu)
    return w, np.ldexp(np.rint(man * 2.0 ** 18), e - 18)


def strided(a, pad, fill):
    """a's values as a view of wider rows behind an odd column, and the wide buffer."""
    import torch
    wide = torch.full((a.shape[0], a.shape[1] + pad), fill, dtype=a.dtype, device="cuda")
    view = wide[:, 1:1 + a.shape[1]] if pad else wide
    view.copy_(a)
    return view, wide


def host(t):
    return t.cpu().numpy()


SIZES = [(1, 1700, 9000), (4, 4000, 300), (5, 4000, 300), (16, 2500, 170), (9, 500, 9001), (30, 2000, 100), (12, 9000, 65),
         (333, 256, 1030), (400, 1000, 1100), (401, 999, 1090), (90, 500, 2000), (91, 501, 2001),
         (128, 1500, 1600), (77, 1025, 900), (250, 1536, 1500), (131, 1301, 1601),
         (1, 1, 1), (1, 64, 32), (2, 63, 31), (1, 960, 960), (3, 65, 33), (15, 128, 70), (16, 1000, 100), (17, 129, 513),
         (31, 320, 64), (32, 64, 257), (33, 2560, 96), (47, 200, 129), (64, 1024, 64), (65, 77, 300), (100, 640, 1000), (129, 192, 257),
         (200, 2049, 65), (256, 256, 256), (257, 96, 640), (300, 960, 1600), (513, 128, 384), (777, 65, 129),
         # 32 x 32 tiles and 128 x 64 ones of 1 to 7 steps and more, their last rows, columns and tiles part empty
         (200, 4096, 1100), (1001, 2601, 999), (1025, 64, 4000), (2047, 100, 1601), (1500, 190, 2500), (800, 256, 2049),
         (2049, 257, 4097), (2049, 64, 4096), (2300, 350, 4100), (4097, 448, 2049)]


@pytest.mark.parametrize("n,k,m", SIZES, ids=str)
@pytest.mark.parametrize("form", ["plain", "bias", "residual", "both"])
def test_linear(L, n, k, m, form):
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, k, m])
    x, (w, mult) = rows(rng, n, k), weights(rng, k, m)
    bias = rng.integers(-2000, 2000, m).astype(np.int32) if form in ("bias", "both") else None
    res = rng.integers(-2 ** 20, 2 ** 20, (n, m)).astype(np.int32) if form in ("residual", "both") else None
    shift = int(rng.integers(0, 7))
    pad = int(rng.integers(0, 4)) if (n + m) % 2 else 0
    weight = L.Weight8(dev(w), dev(mult), None if bias is None else dev(bias))
    xv, _ = strided(dev(x), pad, 77)
    out, wide = strided(torch.zeros(n, m, dtype=torch.int16 if res is None else torch.int32, device="cuda"), pad,
                        GUARD16 if res is None else GUARD32)
    got = L.linear8(xv, weight, out, None if res is None else dev(res), shift)
    assert got is out
    np.testing.assert_array_equal(host(out), O.linear(x, w, mult, bias, res, shift))
    if pad:
        edge = host(wide)
        assert (np.delete(edge, np.s_[1:1 + m], axis=1) == (GUARD16 if res is None else GUARD32)).all()


@pytest.mark.parametrize("n,k,m", SIZES, ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated(L, oracle_lib, n, k, m, act):
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, k, m, len(act)])
    fg = int(rng.integers(6, 13)) if act == "silu" else 8
    x, (wg, mg), (wu, mu) = rows(rng, n, k), weights(rng, k, m, 2.0 ** fg * 3), weights(rng, k, m, 1500)
    bg = rng.integers(-500, 500, m).astype(np.int32) if (n + k) % 3 == 0 else None
    bu = rng.integers(-500, 500, m).astype(np.int32) if (n + k) % 3 == 1 else None
    pad = 3 if m % 2 else 0
    weight = L.GatedWeight8(dev(wg), dev(wu), dev(mg), dev(mu), act, fg, 9, 10, None if bg is None else dev(bg),
                            None if bu is None else dev(bu))
    xv, _ = strided(dev(x), pad, 77)
    out, wide = strided(torch.zeros(n, m, dtype=torch.int16, device="cuda"), pad, GUARD16)
    assert L.gated8(xv, weight, out) is out
    table = None if act == "silu" else oracle_lib.act_table(5 if act == "gelu" else 6)
    want = O.gated(x, wg, wu, mg, mu, act, *L.gate_shifts(act, fg, 9, 10), table, bg, bu)
    np.testing.assert_array_equal(host(out), want)
    if pad:
        assert (np.delete(host(wide), np.s_[1:1 + m], axis=1) == GUARD16).all()


# 128 x 128 and 256 x 128 tiles, steps of each residue of the ring's four or three stages
@pytest.mark.parametrize("n,k,m", [(300, 64, 8190), (300, 128, 8190), (300, 150, 8190), (300, 250, 8190), (1793, 1270, 3001), (1793, 1344, 3001),
                                   (1793, 1401, 3000)], ids=str)
@pytest.mark.parametrize("form", ["plain", "both"])
def test_large_tiles(L, n, k, m, form):
    test_linear(L, n, k, m, form)


@pytest.mark.parametrize("n,k,m", [(513, 700, 2300), (513, 768, 2300), (513, 822, 2300), (513, 886, 2300), (5000, 1280, 513), (5000, 1340, 513),
                                   (800, 1400, 3001)], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_large_gate_tiles(L, oracle_lib, n, k, m, act):
    test_gated(L, oracle_lib, n, k, m, act)


@pytest.mark.parametrize("n", [1, 9, 33, 90, 600])
def test_columns_of_one_buffer(L, n):
    """x and out as columns of the same rows, the output behind x and before it; other columns stay."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng(n)
    k, m = 200, 72
    x, (w, mult) = rows(rng, n, k), weights(rng, k, m)
    weight = L.Weight8(dev(w), dev(mult))
    for at_x, at_o in ((0, k), (m, 0), (m + 3, 1)):
        wide = torch.full((n, k + m + 5), GUARD16, dtype=torch.int16, device="cuda")
        xv, ov = wide[:, at_x:at_x + k], wide[:, at_o:at_o + m]
        xv.copy_(dev(x))
        L.linear8(xv, weight, ov)
        want = np.full((n, k + m + 5), GUARD16, np.int16)
        want[:, at_x:at_x + k], want[:, at_o:at_o + m] = x, O.linear(x, w, mult)
        np.testing.assert_array_equal(host(wide), want)


@pytest.mark.parametrize("n,k,m,pad", [(1 << 20, 2048, 40, 0), (1 << 18, 64, 10000, 0), ((1 << 22) - 5, 33, 7, 3), (300, 70, 40, (1 << 23) - 41),
                                       (40, 64, (1 << 20) - 9, 0), (7, 64, 1 << 20, 1), (50, 32768, 33, 0)], ids=str)
@pytest.mark.parametrize("kind", ["linear", "residual", "gate"])
def test_offsets_past_32_bits(L, kind, n, k, m, pad):
    """Rows, codes and outputs of more than 2^32 bytes, the most rows, columns and k, the widest strides: the first, some middle and the
    last rows and columns as of a call of their own."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n + m)
    rand = lambda lo, hi, shape, t: torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32).to(t)     # noqa: E731
    x = torch.empty(n, k + pad, dtype=torch.int16, device="cuda")[:, :k]
    for i in range(0, n, 1 << 18):
        x[i:i + (1 << 18)] = rand(-400, 401, (min(1 << 18, n - i), k), torch.int16)
    w = [rand(-127, 128, (k, m), torch.int8) for _ in range(2)]
    mult = torch.exp2(rand(-34, -28, (m,), torch.float64))
    cut = lambda c: L.GatedWeight8(w[0][:, c], w[1][:, c], mult[c], mult[c]) if kind == "gate" else L.Weight8(w[0][:, c], mult[c])     # noqa: E731
    run = lambda x, weight, out: L.gated8(x, weight, out) if kind == "gate" else \
        L.linear8(x, weight, out, residual=out if kind == "residual" else None, shift=3)                # noqa: E731
    dtype = torch.int32 if kind == "residual" else torch.int16
    out = torch.empty(n, m + pad, dtype=dtype, device="cuda")[:, :m]
    for i in range(0, n, 1 << 18):
        out[i:i + (1 << 18)] = 1000
    run(x, cut(slice(0, m)), out)
    for r in (slice(0, 33), slice(n // 2, n // 2 + 40), slice(max(0, n - 70), n)):
        for c in (slice(0, min(m, 65)), slice(max(0, m - 70), m)):
            want = torch.full((x[r].shape[0], w[0][:, c].shape[1]), 1000, dtype=dtype, device="cuda")
            run(x[r].contiguous(), cut(c), want)
            assert torch.equal(out[r, c], want), (r, c)


def test_two_streams(L):
    """Products of their own Rows8 on two streams, replayed beside each other."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng(5)
    n, k, m = 600, 1500, 700
    xs, (w, mult) = [rows(rng, n, k) for _ in range(2)], weights(rng, k, m)
    weight = L.Weight8(dev(w), dev(mult))
    torch.cuda.synchronize()
    dx, codes = [dev(x) for x in xs], [L.Rows8(n, k) for _ in range(2)]
    outs, graphs, streams = [torch.zeros(n, m, dtype=torch.int16, device="cuda") for _ in xs], [], [torch.cuda.Stream() for _ in xs]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            L.linear8(L.quant_rows(dx[i], codes[i]), weight, outs[i])
        graphs.append(g)
    for turn in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            np.testing.assert_array_equal(host(o), O.linear(x, w, mult), err_msg=f"turn {turn}")


@pytest.mark.parametrize("n,k", [(1, 1), (1, 17), (5, 63), (16, 64), (17, 65), (33, 1000), (64, 4096), (7, 32768), (700, 129), (1, 8192),
                                 (300, 2100), (300, 4097), (300, 8000), (257, 16400), (40, 20001), (1030, 8200), (4100, 1100), (4111, 2050), (5000, 65)], ids=str)
def test_rows(L, n, k):
    """The codes themselves, where the documented layout puts them, and the rows' maxima; k's padding is zeros."""
    from oracle import linear8 as O
    rng = np.random.default_rng([n, k, 1])
    x = rng.integers(-32768, 32768, (n, k)).astype(np.int16) >> rng.integers(0, 16, (n, 1)).astype(np.int16)
    xv, _ = strided(dev(x), 3, 77)
    r = L.quant_rows(xv)
    steps, blocks = -(-k // 64), -(-n // 32)
    data = host(r.data)
    codes = data[:blocks * steps * 2048].view(np.int8).reshape(blocks, steps, 4, 32, 16).transpose(0, 3, 1, 2, 4).reshape(blocks * 32, -1)
    want, a = O.quant(x)
    np.testing.assert_array_equal(codes[:n, :k], want)
    assert (codes[:n, k:] == 0).all()
    np.testing.assert_array_equal(data[blocks * steps * 2048:].view(np.int32)[:n], a)


def extreme(n, k, m, rng):
    """Rows and weights at the ends of their ranges: zero rows, single values, the lowest int16 everywhere."""
    x = rows(rng, n, k)
    kinds = [0, 1, -1, 32767, -32768]
    for t in range(min(n, 5)):
        x[t] = kinds[t]
    if n > 6:
        x[5] = 0
        x[5, k - 1] = -32768
        x[6, ::2], x[6, 1::2] = 32767, -32768
    w = rng.integers(-128, 128, (k, m)).astype(np.int8)
    w[:, 0], w[:, m // 2], w[:, m - 1] = -128, 127, 0
    return x, w


@pytest.mark.parametrize("n,k,m", [(7, 100, 40), (16, 32768, 33), (40, 4096, 64), (300, 32768, 40), (260, 64, 300)], ids=str)
def test_extremes(L, n, k, m):
    """Saturation on both sides, zero and negative multipliers, the largest multiplier, sums of 32768 products of 127 128."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, k, m, 3])
    x, w = extreme(n, k, m, rng)
    mult = np.ldexp(rng.integers(1, 2 ** 18, m).astype(np.float64), -rng.integers(20, 60, m))
    mult[:3] = 64.0, -64.0, 0.0
    mult[3::4] *= -1
    bias = rng.integers(-2 ** 31, 2 ** 31, m).astype(np.int32)
    bias[::2] = 0
    weight, out = L.Weight8(dev(w), dev(mult), dev(bias)), torch.zeros(n, m, dtype=torch.int16, device="cuda")
    L.linear8(dev(x), weight, out)
    np.testing.assert_array_equal(host(out), O.linear(x, w, mult, bias, exact=True))
    res = rng.integers(-2 ** 31, 2 ** 31, (n, m)).astype(np.int32)
    res[0], res[-1] = 2 ** 31 - 1, -2 ** 31
    out32 = torch.zeros(n, m, dtype=torch.int32, device="cuda")
    L.linear8(dev(x), weight, out32, dev(res), 16)
    np.testing.assert_array_equal(host(out32), O.linear(x, w, mult, bias, res, 16, exact=True))


@pytest.mark.parametrize("n", [3, 40, 300])
def test_one_rounding(L, n):
    """Multipliers of 53 bits and exact ties: the nearest whole number of the exact product, ties to even."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, 4])
    k, m = 70, 64
    x, (w, _) = rows(rng, n, k), weights(rng, k, m)
    x[:, 0] = 127                                    # rows whose maximum is 127: codes are the values
    x[:, 1:] = rng.integers(-127, 128, (n, k - 1))
    w[:, :32] = np.where(rng.random((k, 32)) < 0.05, rng.integers(-3, 4, (k, 32)), 0)
    mult = rng.random(m) * 2.0 ** -14
    mult[:32] = 0.5 / 127 * 127 / 128               # acc 127 / 256: ties where acc is an odd multiple of 128
    mult[:16] = 0.5                                  # every odd sum a tie
    bias = rng.integers(-5, 6, m).astype(np.int32)
    out = torch.zeros(n, m, dtype=torch.int16, device="cuda")
    L.linear8(dev(x), L.Weight8(dev(w), dev(mult), dev(bias)), out)
    np.testing.assert_array_equal(host(out), O.linear(x, w, mult, bias, exact=True))


@pytest.mark.parametrize("act,fg,fu,fy", [("silu", 0, 0, 20), ("silu", 14, 14, 0), ("silu", 14, 43, 0), ("silu", 3, 8, 9), ("gelu", 8, 0, 8),
                                          ("gelu", 8, 8, 8), ("gelu_tanh", 8, 12, 3), ("gelu", 8, 55, 0)], ids=str)
@pytest.mark.parametrize("n", [5, 260])
def test_gate_ranges(L, oracle_lib, act, fg, fu, fy, n):
    """Every gate value of the int16 range against up values at its ends, at the ends of the shifts."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, fg, fu, fy])
    k, m = 64, 96
    x, w = extreme(n, k, m, rng)
    wu = rng.integers(-128, 128, (k, m)).astype(np.int8)
    mg, mu = (np.ldexp(rng.integers(2 ** 17, 2 ** 18, m).astype(np.float64), -rng.integers(32, 44, m)) for _ in range(2))
    weight = L.GatedWeight8(dev(w), dev(wu), dev(mg), dev(mu), act, fg, fu, fy)
    out = torch.zeros(n, m, dtype=torch.int16, device="cuda")
    L.gated8(dev(x), weight, out)
    table = None if act == "silu" else oracle_lib.act_table(5 if act == "gelu" else 6)
    np.testing.assert_array_equal(host(out), O.gated(x, w, wu, mg, mu, act, *L.gate_shifts(act, fg, fu, fy), table))


def gate_and_job(L, n, m, fg):
    """gated8's rows, and the gate of two linear8 outputs by the row-ops unit's MULACT job."""
    import torch
    from cormorant_amd import units as U
    from cormorant_amd.rowops_nodes import SiluMulRoNode
    from cormorant_amd.graph import TensorInfo
    rng = np.random.default_rng([6, n])
    k, fu, fy = 320, 9, 10
    x, (wg, mg), (wu, mu) = dev(rows(rng, n, k)), weights(rng, k, m, 3000), weights(rng, k, m, 2000)
    g, u, y, z = (torch.zeros(n, m, dtype=torch.int16, device="cuda") for _ in range(4))
    L.linear8(x, L.Weight8(dev(wg), dev(mg)), g)
    L.linear8(x, L.Weight8(dev(wu), dev(mu)), u)
    L.gated8(x, L.GatedWeight8(dev(wg), dev(wu), dev(mg), dev(mu), "silu", fg, fu, fy), y)
    T = lambda name, e: TensorInfo(name, [n, m], exp=e)              # noqa: E731
    node = SiluMulRoNode([T("g", fg), T("u", fu)], T("y", fy))
    job = node.jobs()[0]
    b = lambda t: t.view(-1).view(torch.uint8)                       # noqa: E731
    U.rowops(b(g), b(u), b(z), dev(np.asarray(node._params).reshape(-1).view(np.uint8)), job.op, m, n, 1, 2 * m, 0, 2 * m, 0, 2 * m, 0)
    return host(y), host(z)


def test_gate_is_the_row_ops_job(L):
    np.testing.assert_array_equal(*gate_and_job(L, 24, 128, 10))


@pytest.mark.parametrize("n,m", [(24, 128), (100, 128), (400, 2048)], ids=str)
def test_gate_of_an_installed_table(L, n, m):
    """A caller's sigmoid (cm_rowops_tables_init) in the gate as in the MULACT job, and the library's own again."""
    from cormorant_amd import units as U
    img = U.host_rowops_table_image()
    own = gate_and_job(L, n, m, 6)[0]
    changed, rng = img.copy(), np.random.default_rng(n)
    e = changed[:32768].view(np.uint64)
    e[:] = rng.integers(0, 2 ** 24, 4096).astype(np.uint64) | rng.integers(0, 2 ** 24, 4096).astype(np.uint64) << np.uint64(25)
    try:
        U.rowops_tables_init(changed)
        y, z = gate_and_job(L, n, m, 6)
        np.testing.assert_array_equal(y, z)
        assert (y != own).any()
    finally:
        U.rowops_tables_init(img)
    np.testing.assert_array_equal(gate_and_job(L, n, m, 6)[0], own)


@pytest.mark.parametrize("n", [1, 20, 300])
def test_feed_forward(L, n):
    """A run of them as a decoder layer uses them: one row's codes read by three projections, the gate, the down
    projection into the residual in place, twice over."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, 7])
    d, ff = 192, 320
    x = rows(rng, n, d)
    q, g, u, dn = (weights(rng, *s, a) for s, a in (((d, 256), 900), ((d, ff), 2500), ((d, ff), 2000), ((ff, d), 500)))
    h = rng.integers(-2 ** 18, 2 ** 18, (n, d)).astype(np.int32)
    Wq, Wgu, Wd = L.Weight8(dev(q[0]), dev(q[1])), L.GatedWeight8(dev(g[0]), dev(u[0]), dev(g[1]), dev(u[1]), "silu", 10, 9, 9), \
        L.Weight8(dev(dn[0]), dev(dn[1]))
    xd, hd = dev(x), dev(h)
    codes, mid_codes = L.Rows8(n + 3, d), L.Rows8(n, ff)
    qo, mid = torch.zeros(n, 256, dtype=torch.int16, device="cuda"), torch.zeros(n, ff, dtype=torch.int16, device="cuda")
    want_h = h
    for _ in range(2):
        L.quant_rows(xd, codes)
        L.linear8(codes, Wq, qo)
        L.gated8(codes, Wgu, mid)
        L.linear8(L.quant_rows(mid, mid_codes), Wd, hd, residual=hd, shift=5)
        m_want = O.gated(x, g[0], u[0], g[1], u[1], "silu", *L.gate_shifts("silu", 10, 9, 9))
        want_h = O.linear(m_want, dn[0], dn[1], None, want_h, 5)
    np.testing.assert_array_equal(host(qo), O.linear(x, q[0], q[1]))
    np.testing.assert_array_equal(host(mid), m_want)
    np.testing.assert_array_equal(host(hd), want_h)


@pytest.mark.parametrize("n", [1, 16, 40, 200])
def test_captured(L, n):
    """Captured calls (x, its codes, a gate, a residual in place), replayed with new rows and eager work between."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, 8])
    d, ff = 256, 320
    g, u, dn = (weights(rng, *s, a) for s, a in (((d, ff), 2500), ((d, ff), 2000), ((ff, d), 500)))
    Wgu, Wd = L.GatedWeight8(dev(g[0]), dev(u[0]), dev(g[1]), dev(u[1]), "silu", 10, 9, 9), L.Weight8(dev(dn[0]), dev(dn[1]))
    xd, hd = dev(rows(rng, n, d)), dev(np.zeros((n, d), np.int32))
    mid = torch.zeros(n, ff, dtype=torch.int16, device="cuda")

    def step():
        L.gated8(xd, Wgu, mid)
        L.linear8(mid, Wd, hd, residual=hd, shift=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x, h = rows(rng, n, d), rng.integers(-2 ** 18, 2 ** 18, (n, d)).astype(np.int32)
        xd.copy_(dev(x))
        hd.copy_(dev(h))
        graph.replay()
        torch.cuda.synchronize()
        m_want = O.gated(x, g[0], u[0], g[1], u[1], "silu", *L.gate_shifts("silu", 10, 9, 9))
        np.testing.assert_array_equal(host(hd), O.linear(m_want, dn[0], dn[1], None, h, 3))
        other = dev(rows(rng, 7, d))                          # eager work of other sizes between the replays
        L.gated8(other, Wgu, torch.zeros(7, ff, dtype=torch.int16, device="cuda"))


def test_weights_of_any_strides(L):
    """A weight as [k][m], as the transpose of [m][k] and as a cut of a wider one give one image."""
    import torch
    rng = np.random.default_rng(9)
    k, m = 130, 70
    w, mult = weights(rng, k, m)
    x = dev(rows(rng, 3, k))
    wide = np.zeros((k, m + 9), np.int8)
    wide[:, 4:4 + m] = w
    outs = []
    for codes in (dev(w), dev(w.T).t(), dev(wide)[:, 4:4 + m]):
        out = torch.zeros(3, m, dtype=torch.int16, device="cuda")
        weight = L.Weight8(codes, dev(mult))
        codes.zero_()                                         # its values were copied
        outs.append(host(L.linear8(x, weight, out)))
    np.testing.assert_array_equal(outs[0], outs[1])
    np.testing.assert_array_equal(outs[0], outs[2])


def test_other_stream(L):
    """Calls enqueue on the current stream: behind work there that writes their rows."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng(10)
    n, k, m = 100, 512, 192
    x, (w, mult) = rows(rng, n, k), weights(rng, k, m)
    weight, xd, out = L.Weight8(dev(w), dev(mult)), torch.zeros(n, k, dtype=torch.int16, device="cuda"), \
        torch.zeros(n, m, dtype=torch.int16, device="cuda")
    src = dev(x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(20):
            xd.zero_()
        xd.copy_(src)
        L.linear8(xd, weight, out)
    s.synchronize()
    np.testing.assert_array_equal(host(out), O.linear(x, w, mult))


def test_refusals(L):
    import torch
    rng = np.random.default_rng(11)
    k, m = 64, 40
    w, mult = (dev(t) for t in weights(rng, k, m))
    weight = L.Weight8(w, mult)
    gate = L.GatedWeight8(w, w, mult, mult, "silu", 8, 8, 8)
    x, out = dev(rows(rng, 4, k)), torch.zeros(4, m, dtype=torch.int16, device="cuda")
    out32, res = torch.zeros(4, m, dtype=torch.int32, device="cuda"), torch.zeros(4, m, dtype=torch.int32, device="cuda")
    codes = L.quant_rows(x)
    for bad in [lambda: L.Weight8(w, mult.float()), lambda: L.Weight8(w, mult[:-1]), lambda: L.Weight8(w.int(), mult),
                lambda: L.Weight8(w, mult * float("nan")), lambda: L.Weight8(w, mult + 65), lambda: L.Weight8(w, mult - 65),
                lambda: L.Weight8(w, mult, torch.zeros(m, dtype=torch.int16, device="cuda")), lambda: L.Weight8(w, mult.cpu()),
                lambda: L.Weight8(w[0], mult), lambda: L.GatedWeight8(w, w[:, :-1], mult, mult[:-1]),
                lambda: L.GatedWeight8(w, w, mult, mult, "relu"), lambda: L.GatedWeight8(w, w, mult, mult, "gelu", 9),
                lambda: L.linear8(x, gate, out), lambda: L.gated8(x, weight, out), lambda: L.linear8(x[:, :-1], weight, out),
                lambda: L.linear8(x, weight, out[:3]), lambda: L.linear8(x, weight, out[:, :-1]), lambda: L.linear8(x, weight, out32),
                lambda: L.linear8(x, weight, out, residual=res), lambda: L.linear8(x, weight, out32, residual=out),
                lambda: L.linear8(x, weight, out32, residual=res, shift=17), lambda: L.linear8(x, weight, out32, residual=res, shift=-1),
                lambda: L.linear8(x.int(), weight, out), lambda: L.linear8(x.t(), weight, out), lambda: L.linear8(x.cpu(), weight, out),
                lambda: L.linear8(x[:1].expand(4, k), weight, out), lambda: L.linear8(x, weight, out[:1].expand(4, m)),
                lambda: L.linear8(L.Rows8(4, k + 1), weight, out), lambda: L.linear8(L.Rows8(4, k), weight, out),
                lambda: L.quant_rows(x, L.Rows8(3, k)), lambda: L.quant_rows(x, L.Rows8(4, k + 64)), lambda: L.quant_rows(x.int()),
                lambda: L.linear8(dev(rows(rng, 4, k))[:, ::2], L.Weight8(w[:32], mult), out),
                lambda: L.gated8(x[:, :m], L.GatedWeight8(w[:m], w[:m], mult, mult), x[:, :m]),
                lambda: L.linear8(codes, weight, out[:, ::2])]:
        with pytest.raises(ValueError):
            bad()
    assert L.linear8(x[:0], weight, out[:0]).shape == (0, m) and L.gated8(x[:0], gate, out[:0]).shape == (0, m)
    assert L.quant_rows(x[:0]).n == 0
    torch.cuda.synchronize()
