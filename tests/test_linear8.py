"""The 8-bit linear layers without a GPU: the refusals of the C ABI (made on the host before any device
work) and of the Python layer, the weights' quantisation and the oracle's own rules."""
import ctypes
import os
from fractions import Fraction

import numpy as np
import pytest

OK = 0x10000                       # an aligned address that no refused call reads, TO another
TO = 0x20000


@pytest.fixture(scope="module")
def lib():
    from cormorant_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libcormo_hip.so is not built (run __graft_entry__.build())")
    return _lib.lib()


def weight(**kw):
    from cormorant_amd import _lib
    return _lib.CmLinear8Weight(**{**dict(image=OK, k=96, m=40, gated=0, act=0, gate_shift=0, out_shift=0), **kw})


def refused(lib, rc):
    from cormorant_amd import _lib
    assert rc in (_lib.CM_EINVAL, _lib.CM_EALIGN), rc
    assert lib.cm_last_error().decode().startswith("linear8")


def linear(lib, w, **kw):
    a = {**dict(x=OK, x_ld=96, rows=None, n=5, out=TO, out_ld=40, res=None, res_ld=0, shift=0), **kw}
    return lib.cm_linear8(None if w is None else ctypes.byref(w), *a.values(), None)


def gated(lib, w, **kw):
    a = {**dict(x=OK, x_ld=96, rows=None, n=5, out=TO, out_ld=40), **kw}
    return lib.cm_linear8_gated(None if w is None else ctypes.byref(w), *a.values(), None)


@pytest.mark.parametrize("kw", [dict(image=0), dict(image=OK + 16), dict(k=0), dict(k=32769), dict(m=0), dict(m=(1 << 20) + 1)], ids=str)
def test_bad_weights(lib, kw):
    refused(lib, linear(lib, weight(**kw)))
    refused(lib, gated(lib, weight(gated=1, **kw)))


def test_wrong_kind_of_weight(lib):
    refused(lib, linear(lib, weight(gated=1)))
    refused(lib, gated(lib, weight()))
    refused(lib, linear(lib, None))
    refused(lib, gated(lib, None))


@pytest.mark.parametrize("kw", [dict(act=3), dict(gate_shift=15), dict(out_shift=64)], ids=str)
def test_bad_gates(lib, kw):
    refused(lib, gated(lib, weight(gated=1, **kw)))


@pytest.mark.parametrize("kw", [dict(x=None), dict(rows=OK), dict(x=None, rows=OK + 16), dict(x=OK + 1), dict(x_ld=95),
                                dict(n=(1 << 22) + 1), dict(out=None), dict(out=OK + 1), dict(out_ld=39), dict(out_ld=1 << 23)], ids=str)
def test_bad_operands(lib, kw):
    refused(lib, linear(lib, weight(), **kw))
    refused(lib, gated(lib, weight(gated=1), **kw))


@pytest.mark.parametrize("kw", [dict(res=OK + 2, res_ld=40), dict(res=3 * OK, res_ld=39), dict(res=TO, res_ld=48), dict(res=3 * OK, res_ld=40, shift=17),
                                dict(res=3 * OK, res_ld=40, out=TO + 2), dict(shift=17), dict(res=3 * OK, res_ld=1 << 23),
                                dict(res=TO + 4, res_ld=40), dict(res=TO - 4 * 40, res_ld=40), dict(res=TO + 4 * 39, out_ld=80, res_ld=80),
                                dict(res=OK + 64, res_ld=40, out=3 * OK, x=OK + 64, rows=TO)], ids=str)
def test_bad_residuals(lib, kw):
    refused(lib, linear(lib, weight(), **kw))


@pytest.mark.parametrize("kw", [dict(out=OK), dict(out=OK + 190), dict(out=OK + 2 * 4 * 96 + 190), dict(out=OK - 2 * (4 * 40 + 39)),
                                dict(x_ld=136, out=OK + 2 * 95, out_ld=136), dict(x_ld=136, out=OK - 2 * 39, out_ld=136),
                                dict(x_ld=136, out=OK + 2 * 97, out_ld=136), dict(x_ld=200, out=OK + 2 * 96, out_ld=204)], ids=str)
def test_outputs_over_x(lib, kw):
    """An output that shares an element with x, at its ends and as columns of x's buffer, or reaches into it at another stride."""
    refused(lib, linear(lib, weight(), **kw))
    assert b"overlaps x" in lib.cm_last_error()
    refused(lib, gated(lib, weight(gated=1), **kw))
    assert b"overlaps x" in lib.cm_last_error()


@pytest.mark.parametrize("kw", [dict(w=None), dict(mult=None), dict(image=None), dict(image=OK + 128), dict(mult=OK + 4), dict(bias=OK + 2), dict(k=0),
                                dict(k=32769), dict(m=0), dict(m=(1 << 20) + 1), dict(part=3)], ids=str)
def test_bad_packs(lib, kw):
    a = {**dict(w=OK, ks=40, ms=1, mult=OK, bias=None, image=OK, k=96, m=40, part=0), **kw}
    refused(lib, lib.cm_linear8_pack(*a.values(), None))


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=OK + 1), dict(x_ld=95), dict(rows=None), dict(rows=OK + 128), dict(n=(1 << 22) + 1), dict(k=0),
                                dict(k=32769)], ids=str)
def test_bad_rows(lib, kw):
    a = {**dict(x=OK, x_ld=96, rows=OK, n=5, k=96), **kw}
    refused(lib, lib.cm_linear8_rows(*a.values(), None))


def test_no_rows(lib):
    """A call of no rows does nothing and needs no operand."""
    from cormorant_amd import _lib
    assert linear(lib, weight(), n=0, x=None, out=None) == _lib.CM_OK
    assert gated(lib, weight(gated=1), n=0, x=None, out=None) == _lib.CM_OK
    assert lib.cm_linear8_rows(None, 0, None, 0, 96, None) == _lib.CM_OK


def test_sizes(lib):
    """Whole 32-line blocks of 64-k steps, 16 bytes a channel, 4 a row."""
    assert lib.cm_linear8_image_bytes(65, 33, 0) == 2 * 2 * 2048 + 64 * 16
    assert lib.cm_linear8_image_bytes(129, 33, 0) == 2 * 3 * 2048 + 64 * 16
    assert lib.cm_linear8_image_bytes(65, 33, 1) == 2 * lib.cm_linear8_image_bytes(65, 33, 0)
    assert lib.cm_linear8_rows_bytes(1, 64) == 2048 + 128
    assert lib.cm_linear8_rows_bytes(33, 32768) == 64 * 32768 + 256


def test_python_refusals():
    """Host tensors and wrong kinds are refused before any device work."""
    import torch
    from cormorant_amd import linear8 as L
    codes, mult = torch.zeros(8, 4, dtype=torch.int8), torch.zeros(4, dtype=torch.float64)
    with pytest.raises(ValueError):
        L.Weight8(codes, mult)                                      # not on a GPU
    with pytest.raises(ValueError):
        L.GatedWeight8(codes, codes, mult, mult)
    for n, k in ((0, 8), (8, 0), (8, 32769), ((1 << 22) + 1, 8)):
        with pytest.raises(ValueError):
            L.Rows8(n, k)
    x = torch.zeros(2, 8, dtype=torch.int16)
    with pytest.raises(ValueError):
        L.linear8(x, None, x)
    with pytest.raises(ValueError):
        L.gated8(x, None, x)
    with pytest.raises(ValueError):
        L.quant_rows(x[0])


@pytest.mark.parametrize("args", [("relu", 8, 8, 8), ("silu", 15, 8, 8), ("silu", -1, 8, 8), ("gelu", 9, 8, 8), ("gelu_tanh", 7, 8, 8),
                                  ("silu", 8, 0, 21), ("silu", 8, 44, 0), ("gelu", 8, 0, 9)], ids=str)
def test_gates_beyond_the_shifts(args):
    from cormorant_amd import linear8 as L
    with pytest.raises(ValueError):
        L.gate_shifts(*args)


def test_gate_shifts():
    from cormorant_amd import linear8 as L
    assert L.gate_shifts("silu", 10, 9, 11) == (4, 18)
    assert L.gate_shifts("gelu", 8, 9, 11) == (0, 6)


def test_codes_stand_for_the_rows():
    """|x - c a / 127| <= a / 254 (half a step) and what the reciprocal's rounding adds: R is off by at most
    1/2, so the code's real value by |x| / 2^25 <= 2^-10 of a step."""
    from oracle import linear8 as O
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.integers(-32768, 32768, (20, 300)), rng.integers(-3, 4, (20, 300)), np.zeros((1, 300)),
                        np.full((1, 300), -32768), np.full((1, 300), 1)]).astype(np.int16)
    c, a = O.quant(x)
    assert np.abs(c).max() == 127 and (c[40] == 0).all() and a[41] == 32768 and (c[41] == -127).all() and (c[42] == 127).all()
    step = a[:, None] / 127.0
    assert (np.abs(x - c * step) <= step * (0.5 + 2.0 ** -10)).all()


def test_every_row_maximum_fits_32_bits():
    """The kernel's 32-bit arithmetic: |x R| + 2^23 < 2^31 and codes of at most 127 for every maximum."""
    a = np.arange(1, 32769, dtype=np.int64)
    r = (127 * 2 ** 24 + a // 2) // a
    assert (a * r + 2 ** 23 < 2 ** 31).all() and (-a * r + 2 ** 23 >= -2 ** 31).all() and (r < 2 ** 31).all()
    assert ((a * r + 2 ** 23) >> 24 == 127).all() and ((-a * r + 2 ** 23) >> 24 == -127).all()


def test_oracle_forms_agree():
    """The int64 form of the scaling equals the exact one, and a double's fused multiply-add onto 1.5 2^52 as well."""
    from oracle import linear8 as O
    rng = np.random.default_rng(1)
    acc = rng.integers(-2 ** 24, 2 ** 24, (6, 40))
    a = rng.integers(0, 32769, 6)
    M = rng.integers(2 ** 17, 2 ** 18, 40)
    s = rng.integers(35, 48, 40)
    s[:5], M[:5] = 30, 2 ** 17                                     # many ties: multiples of 2^-13
    mult, bias = np.ldexp(M.astype(np.float64), -s), rng.integers(-3000, 3000, 40)
    np.testing.assert_array_equal(O.scaled(acc, a, mult, bias), O.scaled_fast(acc, a, mult, bias))


def test_quantise_weight():
    from cormorant_amd import linear8 as L
    rng = np.random.default_rng(2)
    w = rng.standard_normal((64, 9)).astype(np.float32) * 0.02
    w[:, 3] = 0
    codes, mult = L.quantise_weight(w, 9, 11)
    assert codes.dtype == np.int8 and (codes[:, 3] == 0).all() and mult[3] == 0 and np.abs(codes).max() == 127
    step = np.abs(w.astype(np.float64)).max(axis=0) / 127
    assert (np.abs(w - codes * step) <= step / 2 * (1 + 1e-12)).all()
    live = step > 0
    assert np.allclose(mult[live], step[live] * 4 / 127, rtol=2.0 ** -18)
    for f in mult:
        assert Fraction(float(f)).numerator.bit_length() <= 18
    per = L.quantise_weight(w, 9, np.arange(9))[1]
    assert np.allclose(per[live], (step * 2.0 ** (np.arange(9) - 9) / 127)[live], rtol=2.0 ** -18)
    for bad in (np.full((2, 2), np.nan), np.full((2, 2), np.inf), np.full((2, 2), 1e9)):
        with pytest.raises(ValueError):
            L.quantise_weight(bad, 0, 11)
