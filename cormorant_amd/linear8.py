"""A decoder's linear layers in 8 bits, as calls on device tensors: int16 rows quantised a token at a time,
their product with 8-bit weights (a scale a channel) into int16 rows or added to the int32 residual
stream (``linear8``), and a feed-forward block's gate: two products of the same rows, the activation
of one times the other (``gated8``).

Beside the int16 products of ``units.matmul`` and ``units.matmul_skinny_planes*``: half a weight's bytes
and a quarter of the byte products.  The reference's MatmulKernel has no 8-bit weights; the residual add
and the gate are its row-ops jobs (rowops_nodes.py:401-447, 540-563), GELU its activation unit's table.
The framework trains nothing, so neither has a backward pass.

A ``Weight8`` / ``GatedWeight8`` lays its codes out once, on the stream that is current then.  ``Rows8`` holds the
codes of rows that several products read (``quant_rows``); a call given int16 rows makes them itself.  Calls enqueue on
the current torch stream of the weight's device, which must be the current device.  A call given int16 rows may hold
their codes in the device's workspace, like the units' calls: one stream at a time, and once before a capture at the
same sizes.  A call given a Rows8 takes no workspace, so that two streams, or graphs replayed beside each other, each
with a Rows8 of its own, do not meet.  A replayed graph writes the rows it was captured with; ``Rows8.n`` is of the last
call, not of a replay.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Union

import torch

from . import _lib

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
MAX_K, MAX_M, MAX_N, MAX_MULT = 32768, 1 << 20, 1 << 22, 64.0
SILU_BITS, G_BITS, ACT_BITS, MULT_BITS = 20, 14, 8, 18


def _buffer(nbytes: int, device) -> torch.Tensor:
    """A 256-byte aligned uint8 buffer."""
    t = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    return t[(-t.data_ptr()) % 256:][:nbytes]


def _check_codes(codes: torch.Tensor, mult: torch.Tensor, bias: Optional[torch.Tensor], what: str):
    if codes.dim() != 2 or codes.dtype is not torch.int8 or not codes.is_cuda:
        raise ValueError(f"{what}: the codes must be a GPU int8 [k][m] tensor")
    k, m = codes.shape
    if not (1 <= k <= MAX_K and 1 <= m <= MAX_M):
        raise ValueError(f"{what}: a weight of {k} x {m} (up to {MAX_K} x {MAX_M})")
    if codes.stride(0) < 0 or codes.stride(1) < 0:
        raise ValueError(f"{what}: codes at negative strides")
    for name, t, dtype in (("mult", mult, torch.float64), ("bias", bias, torch.int32)):
        if t is None and name == "bias":
            continue
        if t is None or t.dtype is not dtype or t.device != codes.device or t.numel() != m or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be {m} contiguous {dtype} values beside the codes")
    if not bool((mult.abs() <= MAX_MULT).all()):                     # False for a NaN too
        raise ValueError(f"{what}: multipliers beyond +-{MAX_MULT:g}")
    return k, m


class _Packed:
    """A weight's image on its device and the structure that the calls take."""

    def _lay(self, k: int, m: int, gated: bool, device, act: int = 0, gate_shift: int = 0, out_shift: int = 0):
        self.k, self.m, self.device = k, m, device
        lib = _lib.lib()
        self.image = _buffer(lib.cm_linear8_image_bytes(k, m, int(gated)), device)
        self.index = self.image.get_device()
        self._c = _lib.CmLinear8Weight(self.image.data_ptr(), k, m, int(gated), act, gate_shift, out_shift)
        self._ref = ctypes.byref(self._c)

    def _pack(self, codes, mult, bias, part: int):
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream().cuda_stream
            _lib.check(_lib.lib().cm_linear8_pack(codes.data_ptr(), codes.stride(0), codes.stride(1), mult.data_ptr(),
                                                  None if bias is None else bias.data_ptr(), self.image.data_ptr(),
                                                  self.k, self.m, part, stream), "cm_linear8_pack")


class Weight8(_Packed):
    """An 8-bit weight: ``codes`` int8 [k][m] (any strides: the view ``w.t()`` of [m][k] rows), ``mult``
    float64 [m], each channel's multiplier (its scale, times 2^(f_out - f_in), over 127; at most 64 in
    size) and optionally ``bias`` int32 [m] at the output's exponent.  Their values are copied."""

    def __init__(self, codes: torch.Tensor, mult: torch.Tensor, bias: Optional[torch.Tensor] = None):
        k, m = _check_codes(codes, mult, bias, "Weight8")
        self._lay(k, m, False, codes.device)
        self._pack(codes, mult, bias, 0)


class GatedWeight8(_Packed):
    """A feed-forward block's gate and up weights (codes int8 [k][m] each, multipliers and biases as
    Weight8's, into rows at 2^-gate_exp and 2^-up_exp) and its activation: "silu" (the row-ops unit's, gate_exp
    0 .. 14), "gelu" or "gelu_tanh" (the activation unit's, gate_exp 8); the result at 2^-out_exp."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, gate_mult: torch.Tensor, up_mult: torch.Tensor,
                 act: str = "silu", gate_exp: int = 8, up_exp: int = 8, out_exp: int = 8,
                 gate_bias: Optional[torch.Tensor] = None, up_bias: Optional[torch.Tensor] = None):
        k, m = _check_codes(gate, gate_mult, gate_bias, "GatedWeight8: gate")
        if _check_codes(up, up_mult, up_bias, "GatedWeight8: up") != (k, m) or up.device != gate.device:
            raise ValueError("GatedWeight8: gate and up of different sizes or devices")
        gate_shift, out_shift = gate_shifts(act, gate_exp, up_exp, out_exp)
        self.act = act
        self._lay(k, m, True, gate.device, ACTS[act], gate_shift, out_shift)
        self._pack(gate, gate_mult, gate_bias, 1)
        self._pack(up, up_mult, up_bias, 2)


def gate_shifts(act: str, gate_exp: int, up_exp: int, out_exp: int):
    """(gate_shift, out_shift) of a gate's exponents; ValueError where the unit's shifts do not reach."""
    if act not in ACTS:
        raise ValueError(f"gated8: activation '{act}' (one of {', '.join(ACTS)})")
    gate_shift, f = (G_BITS - gate_exp, SILU_BITS) if act == "silu" else (0, ACT_BITS)
    if act != "silu" and gate_exp != ACT_BITS:
        raise ValueError(f"gated8: a {act} gate at 2^-{gate_exp} (the activation unit's rows are at 2^-{ACT_BITS})")
    out_shift = f + up_exp - out_exp
    if not (0 <= gate_shift <= G_BITS and 0 <= out_shift <= 63):
        raise ValueError(f"gated8: exponents {gate_exp}, {up_exp} -> {out_exp} beyond the shifts")
    return gate_shift, out_shift


class Rows8:
    """The codes of up to ``n`` rows of ``k`` (quant_rows writes them; ``self.n`` rows of its last call are valid).  The rows' maxima
    lie behind the blocks of that many rows, so the products take all of them, never their first few."""

    def __init__(self, n: int, k: int, device="cuda"):
        if not (1 <= n <= MAX_N and 1 <= k <= MAX_K):
            raise ValueError(f"Rows8: {n} rows of {k} (up to {MAX_N} of {MAX_K})")
        self.cap, self.k, self._n = n, k, 0
        self.data = _buffer(_lib.lib().cm_linear8_rows_bytes(n, k), device)
        self.device, self.index, self.at = self.data.device, self.data.get_device(), self.data.data_ptr()

    @property
    def n(self) -> int:
        return self._n


def _stride(t: torch.Tensor, name: str, dtype, n: int, width: int) -> int:
    """The row stride of an operand [n][width] of contiguous columns (a call's checks are a third of its time on the host)."""
    if t.dtype is not dtype or t.shape != (n, width):
        raise ValueError(f"{name} must be a GPU {dtype} tensor [{n}][{width}], got {t.dtype} {list(t.shape)}")
    rows, cols = t.stride()
    if cols != 1 and width > 1:
        raise ValueError(f"{name} must be rows of contiguous columns, got strides {[rows, cols]}")
    if n <= 1:
        return width
    if rows < width:
        raise ValueError(f"{name}: rows of {width} columns overlap at a stride of {rows}")
    return rows


def _on(index: int, *on) -> int:
    """The current stream of device ``index``, which every operand must be on and which must be current."""
    for t in on:
        if t.get_device() != index:
            raise ValueError(f"the weight is on cuda:{index}, an operand on {t.device}")
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"the weight is on cuda:{index}, the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(index)         # torch.cuda.current_stream() takes 2.8 us of a 10 us call


def quant_rows(x: torch.Tensor, rows: Optional[Rows8] = None) -> Rows8:
    """cm_linear8_rows: the codes of x's int16 rows [n][k], for the products that read them."""
    if x.dim() != 2:
        raise ValueError(f"quant_rows: x must be [n][k], got {list(x.shape)}")
    n, k = x.shape
    if rows is None:
        rows = Rows8(max(n, 1), k, x.device)
    if rows.k != k or n > rows.cap:
        raise ValueError(f"quant_rows: {n} rows of {k} into codes of {rows.cap} rows of {rows.k}")
    ld = _stride(x, "x", torch.int16, n, k)
    stream = _on(rows.index, x)
    _lib.check(_lib.lib().cm_linear8_rows(x.data_ptr(), ld, rows.data.data_ptr(), n, k, stream), "cm_linear8_rows")
    rows._n = n
    return rows


def _x(x: Union[torch.Tensor, Rows8], k: int, what: str):
    """(n, x's address, its row stride, its codes' address, the tensor to check) of a call's rows."""
    if isinstance(x, Rows8):
        if x.k != k:
            raise ValueError(f"{what}: rows of {x.k} against a weight of {k}")
        return x._n, None, 0, x.at, x.data
    shape = x.shape
    if len(shape) != 2 or shape[1] != k or shape[0] > MAX_N:
        raise ValueError(f"{what}: x must be [n][{k}] of up to {MAX_N} rows, got {list(shape)}")
    n = shape[0]
    return n, x.data_ptr(), _stride(x, "x", torch.int16, n, k), None, x


def linear8(x: Union[torch.Tensor, Rows8], weight: Weight8, out: torch.Tensor, residual: Optional[torch.Tensor] = None,
            shift: int = 0) -> torch.Tensor:
    """cm_linear8: out [n][m] = x's rows (int16 [n][k], or their codes) times the weight, int16; with a
    ``residual`` (int32 [n][m]) out is int32, the residual plus the product << ``shift`` (0 .. 16), and may
    be the residual.  Rows may be strided (out's and the residual's below 2^23 elements).  out shares no element
    with x, nor with a residual that it is not."""
    if type(weight) is not Weight8:
        raise ValueError("linear8: a Weight8")
    n, at, ld, codes, t = _x(x, weight.k, "linear8")
    out_at = out.data_ptr()
    if residual is None:
        out_ld = _stride(out, "out", torch.int16, n, weight.m)
        stream = _on(weight.index, t, out)
        rc = _lib.lib().cm_linear8(weight._ref, at, ld, codes, n, out_at, out_ld, None, 0, 0, stream)
    else:
        if not 0 <= shift <= 16:
            raise ValueError(f"linear8: a residual shift of {shift} (0 .. 16)")
        out_ld = _stride(out, "out", torch.int32, n, weight.m)
        res_ld = _stride(residual, "residual", torch.int32, n, weight.m)
        stream = _on(weight.index, t, out, residual)
        rc = _lib.lib().cm_linear8(weight._ref, at, ld, codes, n, out_at, out_ld, residual.data_ptr(), res_ld, shift, stream)
    if rc:
        _lib.check(rc, "cm_linear8")
    return out


def gated8(x: Union[torch.Tensor, Rows8], weight: GatedWeight8, out: torch.Tensor) -> torch.Tensor:
    """cm_linear8_gated: out [n][m] int16 = act(x Wg) (x Wu), x and out as linear8's."""
    if type(weight) is not GatedWeight8:
        raise ValueError("gated8: a GatedWeight8")
    n, at, ld, codes, t = _x(x, weight.k, "gated8")
    out_at = out.data_ptr()
    out_ld = _stride(out, "out", torch.int16, n, weight.m)
    stream = _on(weight.index, t, out)
    rc = _lib.lib().cm_linear8_gated(weight._ref, at, ld, codes, n, out_at, out_ld, stream)
    if rc:
        _lib.check(rc, "cm_linear8_gated")
    return out


def quantise_weight(w, f_in: int, f_out) -> tuple:
    """(codes int8 [k][m], mult float64 [m]) of a float weight [k][m] (numpy) between rows at 2^-f_in and
    2^-f_out (one exponent, or one a channel): each channel in 127 steps of its largest value, the
    multiplier in 18 bits (2^-18 of a result of 16: acc a_t M stays below 2^62, 64-bit integers restate it)."""
    import numpy as np
    w = np.asarray(w, np.float64)
    top = np.abs(w).max(axis=0)
    if not np.isfinite(top).all():
        raise ValueError("quantise_weight: a weight that is not finite")
    step = np.where(top > 0, top, 1.0) / 127.0
    codes = np.rint(w / step).clip(-127, 127).astype(np.int8)
    mu = np.where(top > 0, step, 0.0) * 2.0 ** (np.asarray(f_out, np.float64) - f_in) / 127.0
    man, exp = np.frexp(mu)
    mult = np.ldexp(np.rint(man * 2.0 ** MULT_BITS), exp - MULT_BITS)
    if (mult > MAX_MULT).any() or math.isnan(float(mult.sum())):
        raise ValueError(f"quantise_weight: multipliers above {MAX_MULT:g} (exponents {f_in} -> {f_out})")
    return codes, mult


__all__ = ["Weight8", "GatedWeight8", "Rows8", "quant_rows", "linear8", "gated8", "quantise_weight", "gate_shifts"]
