"""The paged cache's entry points without a GPU: the refusals of the C ABI (made on the host before
any device work) and of the Python layer, and the oracle's own rules."""
import ctypes
import os

import numpy as np
import pytest

OK = 0x1000                        # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    from cormorant_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libcormo_hip.so is not built (run __graft_entry__.build())")
    return _lib.lib()


def cache(**kw):
    from cormorant_amd import _lib
    return _lib.CmPagedCache(**{**dict(data=OK, pages=4, page=16, kv_heads=2, head_dim=64, int8=0), **kw})


def batch(**kw):
    from cormorant_amd import _lib
    return _lib.CmPagedBatch(**{**dict(q_start=OK, kv_len=OK, table=OK, batch=2, tokens=5, max_pages=3, table_ld=3), **kw})


def prep(**kw):
    from cormorant_amd import _lib
    return _lib.CmPagedPrepArgs(**{**dict(q=OK, k=OK, v=OK, qr=OK, q_ld=384, k_ld=128, v_ld=128, qr_ld=384, heads=6, rope=OK,
                                          rope_rows=9, rotary=64, interleaved=0, rope_q=OK, rope_k=OK), **kw})


BAD_CACHE = [dict(data=0), dict(data=OK + 8), dict(pages=0), dict(page=8), dict(page=24), dict(page=8192), dict(kv_heads=0),
             dict(kv_heads=2000), dict(head_dim=32), dict(head_dim=96), dict(int8=2)]
BAD_BATCH = [dict(q_start=0), dict(kv_len=0), dict(table=0), dict(max_pages=0), dict(max_pages=(1 << 16) + 1),
             dict(tokens=1 << 25), dict(batch=1 << 21)]


def refused(lib, rc):
    from cormorant_amd import _lib
    assert rc in (_lib.CM_EINVAL, _lib.CM_EALIGN), rc
    assert lib.cm_last_error().decode().startswith("paged")


def calls(lib, c, b):
    p = prep()
    yield lib.cm_paged_prep(ctypes.byref(c), ctypes.byref(b), ctypes.byref(p), None)
    yield lib.cm_paged_attention(ctypes.byref(c), ctypes.byref(b), OK, OK, 384, 384, 6, 0, 1 << 23, 20 | 14 << 8, None)
    yield lib.cm_paged_read(ctypes.byref(c), ctypes.byref(b), OK, OK, 128, 128, None)


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_caches(lib, kw):
    for rc in calls(lib, cache(**kw), batch()):
        refused(lib, rc)


@pytest.mark.parametrize("kw", BAD_BATCH, ids=str)
def test_bad_batches(lib, kw):
    for rc in calls(lib, cache(), batch(**kw)):
        refused(lib, rc)


@pytest.mark.parametrize("kw", [dict(q=0), dict(k=0), dict(v=0), dict(qr=0), dict(rope=0), dict(rope_q=0), dict(rope_k=0),
                                dict(q=OK + 2), dict(qr=OK + 8), dict(rope=OK + 4), dict(norm_q=OK + 4), dict(q_ld=388),
                                dict(q_ld=376), dict(k_ld=64), dict(heads=0), dict(rotary=0), dict(rotary=8),
                                dict(rotary=80), dict(rope_rows=0), dict(eps_q=-1), dict(eps_k=1 << 62)], ids=str)
def test_bad_prep(lib, kw):
    c, b, p = cache(), batch(), prep(**kw)
    refused(lib, lib.cm_paged_prep(ctypes.byref(c), ctypes.byref(b), ctypes.byref(p), None))


@pytest.mark.parametrize("kw", [dict(q=0), dict(o=0), dict(q=OK + 2), dict(o_ld=380), dict(q_ld=320), dict(heads=0), dict(heads=5),
                                dict(cfg=20), dict(cfg=20 | 16 << 8), dict(cfg=35 | 14 << 8), dict(cm=1, cfg=12 | 14 << 8), dict(window=1 << 31)], ids=str)
def test_bad_attention(lib, kw):
    a = {**dict(q=OK, o=OK, q_ld=384, o_ld=384, heads=6, window=0, cm=1 << 23, cfg=20 | 14 << 8), **kw}
    c, b = cache(), batch()
    refused(lib, lib.cm_paged_attention(ctypes.byref(c), ctypes.byref(b), a["q"], a["o"], a["q_ld"], a["o_ld"], a["heads"],
                                        a["window"], a["cm"], a["cfg"], None))


@pytest.mark.parametrize("kw", [dict(k=0), dict(v=0), dict(k=OK + 2), dict(k_ld=132), dict(v_ld=64)], ids=str)
def test_bad_read(lib, kw):
    a = {**dict(k=OK, v=OK, k_ld=128, v_ld=128), **kw}
    c, b = cache(), batch()
    refused(lib, lib.cm_paged_read(ctypes.byref(c), ctypes.byref(b), a["k"], a["v"], a["k_ld"], a["v_ld"], None))


def test_null_arguments(lib):
    refused(lib, lib.cm_paged_read(None, None, OK, OK, 128, 128, None))
    c, b = cache(), batch()
    refused(lib, lib.cm_paged_prep(ctypes.byref(c), ctypes.byref(b), None, None))


def test_python_layer_refusals():
    import torch
    from cormorant_amd import paged as P
    i32 = dict(dtype=torch.int32)
    for kw in (dict(page=8), dict(page=48), dict(head_dim=32), dict(pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            P.PagedCache(**{**dict(pages=2, page=16, kv_heads=2, head_dim=64), **kw}, data=torch.zeros(8, dtype=torch.uint8))
    with pytest.raises(ValueError):
        P.PagedCache(2, 16, 2, 64, data=torch.zeros(2 * 2 * 16 * 260, dtype=torch.uint8))        # not on a GPU
    with pytest.raises(ValueError):
        P.PagedBatch(torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros(2, 4, **i32), 5)
    for cols in (16, 40, 48):
        with pytest.raises(ValueError):
            P.PagedPrep(torch.zeros(4, cols, **i32), torch.zeros(16, dtype=torch.uint8), torch.zeros(16, dtype=torch.uint8))


def test_block_bytes(lib):
    from cormorant_amd import paged as P
    for page in (16, 64, 4096):
        for hd in (64, 128):
            for i8 in (False, True):
                assert P.block_bytes(page, hd, i8) == lib.cm_paged_block_bytes(page, hd, int(i8))


def test_oracle_quantise_and_pool():
    """The 8-bit form by its definition in fractions, and rows through the pool's bytes."""
    from fractions import Fraction
    from oracle import paged as O
    rng = np.random.default_rng(0)
    for row in ([0, 0, 5], [127, -128, 1], [128, 3, -3], [-129, 128, 2], [32767, -32768, 255], [-32768, 384, 128], [255, 1, 1]):
        codes, e = O.quantise(np.array(row))
        m = max(x if x >= 0 else -1 - x for x in row)
        assert e == min(s for s in range(9) if m < 128 << s)
        for x, c in zip(row, codes):
            assert c == min(127, round(Fraction(x, 1 << e)))         # Python rounds half to even
    for int8 in (False, True):
        pool = O.Pool(3, 16, 2, 64, int8)
        rows = {}
        for pid, slot, g in ((0, 0, 0), (0, 15, 1), (2, 7, 0)):
            k, v = (rng.integers(-32768, 32768, 64) for _ in range(2))
            pool.write(pid, slot, g, k, v)
            rows[pid, slot, g] = k, v
        for at, (k, v) in rows.items():
            for x, y in zip((k, v), pool.read(*at)):
                if int8:
                    codes, e = O.quantise(x)
                    x = codes << e
                np.testing.assert_array_equal(x, y)


def test_prep_operands_pack_as_the_structure(lib):
    """paged_prep packs the call's operands itself: the structure's leading fields, byte for byte."""
    from cormorant_amd import _lib as L
    from cormorant_amd import paged as P
    a = L.CmPagedPrepArgs(q=1, k=2, v=3, qr=1 << 40, q_ld=5, k_ld=6, v_ld=7, qr_ld=1 << 33, heads=9)
    assert bytes(a)[:P._OPERANDS.size] == P._OPERANDS.pack(1, 2, 3, 1 << 40, 5, 6, 7, 1 << 33, 9)
    assert L.CmPagedPrepArgs.heads.offset + L.CmPagedPrepArgs.heads.size == P._OPERANDS.size
