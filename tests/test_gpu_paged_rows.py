"""The paged attention's three ways against the oracle -- one launch for short tables, kept scores, and
tiles of many rows whose keys are divided evenly over the workgroups --, each where it is the one taken
(asserted by the kernels launched), over the same lengths, masks, values and strides."""
import numpy as np
import pytest

from test_gpu_paged import Case, check_attention, paged, regs  # noqa: F401

pytestmark = pytest.mark.gpu

WAYS = {"short": ("paged_short_kernel", 0), "kept": ("paged_few_kernel", 150), "many": ("paged_rows_kernel", 4000)}


def check(P, c, way, cm, cfg, **kw):
    """The case over a table widened so that the estimates choose ``way``."""
    from cormorant_amd import _lib
    kernel, wide = WAYS[way]
    c.table = np.concatenate([c.table, np.zeros((len(c.lens), wide * 16 // c.page), np.int32)], axis=1)
    _lib.timing_reset()
    _lib.timing_enable(True)
    try:
        check_attention(P, c, cm, cfg, **kw)
        launched = {k: _lib.timing_read(k)[1] for k, _ in WAYS.values()}
    finally:
        _lib.timing_enable(False)
        _lib.timing_reset()
    assert launched == {k: int(k == kernel) for k in launched}


ROWS = [([17, 60], [17, 60], 16, 3), ([300, 333], [40, 33], 32, 8), ([130, 64], [33, 64], 64, 4), ([63, 200], [63, 20], 128, 4),
        ([700, 90, 5], [100, 90, 5], 16, 3)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,new,page,G", ROWS)
def test_many_rows(paged, lens, new, page, G, hd, int8):  # noqa: F811
    c = Case(np.random.default_rng(sum(lens) + hd), lens, new, kv=4, G=G, hd=hd, page=page, int8=int8, tail=2)
    check(paged, c, "many", *regs(hd))


@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 1 << 20])
@pytest.mark.parametrize("hd,int8", [(64, False), (64, True), (128, False), (128, True)])
def test_many_rows_in_windows(paged, window, hd, int8):  # noqa: F811
    c = Case(np.random.default_rng(window), [210, 177], [70, 90], kv=4, hd=hd, int8=int8)
    check(paged, c, "many", *regs(hd), window=window)


@pytest.mark.parametrize("way", ["short", "kept", "many"])
@pytest.mark.parametrize("hd,int8", [(64, False), (64, True), (128, False), (128, True)])
def test_rows_and_pages_without_keys(paged, way, hd, int8):  # noqa: F811
    """Negative positions, an empty and a waiting sequence; page ids outside the pool; lengths past the pages."""
    n = 1 if way == "kept" else 60
    new = [n, 0, n, n]
    c = Case(np.random.default_rng(5), [60, 40, 63, 20 + n], new, kv=4, hd=hd, int8=int8, tail=1)
    c.kv_len = np.array([0 if n == 1 else 40, 0, -7, 20 + n], np.int32)
    check(paged, c, way, *regs(hd))
    c = Case(np.random.default_rng(6), [120, 170, 60], [n, n, n], kv=4, hd=hd, int8=int8)
    c.table[0, 2], c.table[0, 5], c.table[1, 0], c.table[2, :] = -1, c.pages, 2 ** 31 - 1, -2 ** 31
    check(paged, c, way, *regs(hd))


@pytest.mark.parametrize("way", ["short", "kept", "many"])
@pytest.mark.parametrize("hd,int8", [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("fs,fp", [(3, 1), (8, 8), (10, 15)])
def test_large_values(paged, way, fs, fp, hd, int8):  # noqa: F811
    """Scores that saturate and wrap, sums at the ends of their ranges, outputs that saturate."""
    rng = np.random.default_rng(fs)
    n = 1 if way == "kept" else 50
    c = Case(rng, [90, 66], [n, n], kv=4, hd=hd, int8=int8, amp=12000)
    check(paged, c, way, *regs(hd, fs, fp))
    c = Case(rng, [90, 70], [n, n], kv=4, hd=hd, int8=int8, amp=100000)
    c.q[:] = rng.choice([-32768, 32767, 0], c.q.shape)
    check(paged, c, way, *regs(hd, fs, fp))


@pytest.mark.parametrize("way", ["short", "kept", "many"])
@pytest.mark.parametrize("cm,cs", [(0, 20), (1, 0), ((1 << 24) - 1, 0), (12345678, 8), (65536, 0), (12102203, 31), (8388608, 34),
                                   (5, 13)])
def test_softmax_registers(paged, way, cm, cs):  # noqa: F811
    n = 1 if way == "kept" else 50
    c = Case(np.random.default_rng(cs), [70, 64], [n, n], kv=4, amp=3000)
    check(paged, c, way, cm, cs | (14 << 8))


@pytest.mark.parametrize("cm,cs", [(0, 20), (1, 0), (7, 0), ((1 << 24) - 1, 0), ((1 << 24) - 1, 7), (12345678, 8), (65535, 0),
                                   (65536, 0), (69632, 0), (12102203, 31), (8388608, 34), (16777215, 34), (5, 13)])
def test_many_rows_softmax_registers_128(paged, cm, cs):  # noqa: F811
    """Int16 rows of 128: the exponential's table in 16 bits."""
    c = Case(np.random.default_rng(cs), [70, 64], [50, 50], kv=4, hd=128, amp=2000)
    check(paged, c, "many", cm, cs | (14 << 8))


@pytest.mark.parametrize("way", ["short", "kept", "many"])
def test_strided_rows(paged, way):  # noqa: F811
    n = 1 if way == "kept" else 50
    c = Case(np.random.default_rng(8), [70, 64], [n, n], kv=4)
    check(paged, c, way, *regs(), q_pad=64, o_pad=24)


@pytest.mark.parametrize("hd,int8", [(64, False), (128, True)])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([40, 64, 65, 1], [40, 1, 33, 1]), ([500, 30], [15, 30])])
def test_short_tables(paged, lens, new, hd, int8):  # noqa: F811
    """Tiles of the one-launch kernel: one token, tiles that end inside a token's heads, a full tile."""
    for G in (1, 4, 15, 16):
        c = Case(np.random.default_rng(G), lens, new, kv=2, G=G, hd=hd, int8=int8, tail=1)
        check(paged, c, "short", *regs(hd))
