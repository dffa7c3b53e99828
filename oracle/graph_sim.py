"""A CPU forward pass of a simulator graph that restates the reference simulator's
``_forward_pass`` (inference-scheduler/src/codegen/_simulate.py:541-769) in the value domain
with numpy float64, the way the reference computes: np.matmul / per-tap conv sums (exact for
on-grid operands), then ``truncate`` (clip + floor).  Pooling, the activation unit, softmax
and row-ops jobs use the C oracle on raw lanes; the row-ops adapters' job constants, RoPE, the
attention prep and the host ops come from this directory's own restatements.

TEST INFRASTRUCTURE ONLY: the graph-level check of cormorant_amd.simulate.Simulator and the CPU
baseline bench.py times.  It reads a graph's declared fields (tensors, shapes, exponents, node
parameters) and dispatches on the nodes' class names; it imports nothing from the product, so
no arithmetic, rounding rule or job derivation is shared with what it checks.
"""
from types import SimpleNamespace

import numpy as np

from oracle import cm
from oracle import host_ref
from oracle import linear8 as oracle_linear8
from oracle import paged as oracle_paged
from oracle import residual_ref
from oracle import rowops_adapt
from oracle import sim_ref
from oracle.attn_prep import attn_prep, clamp_n, transpose, vit_attn_prep

F = 8                                   # the element type's fraction bits (ap_fixed<16,8>)
Q_MIN, Q_MAX = -128.0, 127.99609375
_NP = {"i16": np.int16, "i32": np.int32, "f32": np.float32}
_KB = {"i16": 2, "i32": 4, "f32": 4}
ADAPTERS = ("LayerNormRoNode", "LayerNorm32RoNode", "RMSNormRoNode", "ResAddRoNode", "ResAddBiasRoNode",
            "WidenRoNode", "SiluMulRoNode", "DequantRoNode", "BiasCopyRoNode", "RopeRoNode")


class _RopeRoNode(SimpleNamespace):
    """A RoPE adapter's declared fields, for the row-ops adapter restatement (dispatched by class name)."""


_RopeRoNode.__name__ = "RopeRoNode"


def _quantize(x):
    """ApFixed.quantize (dtype.py:367-369): clip, round half to even at 2^-8."""
    return np.round(np.clip(np.asarray(x, np.float64), Q_MIN, Q_MAX) * 256.0) / 256.0


def _truncate(x):
    """ApFixed.truncate (dtype.py:371-377): clip, floor at 2^-8."""
    return np.floor(np.clip(np.asarray(x, np.float64), Q_MIN, Q_MAX) * 256.0) / 256.0


def _to_raw(v):
    return np.clip(np.round(np.asarray(v, np.float64) * 256.0), -32768, 32767).astype(np.int16)


def _from_raw(r):
    return np.asarray(r, np.float64) / 256.0


def _kind(sn):
    return type(sn).__name__


def _conv_int(x, w, sh, sw, pt, pl, dh, dw, oh, ow, dwise):
    """_conv2d_int (_simulate.py:198-220): exact per-tap sums of float64 integers."""
    N, C, H, W = x.shape
    kh, kw = w.shape[2], w.shape[3]
    need_h = (oh - 1) * sh + (kh - 1) * dh + 1
    need_w = (ow - 1) * sw + (kw - 1) * dw + 1
    xp = np.zeros((N, C, max(need_h, pt + H), max(need_w, pl + W)))
    xp[:, :, pt:pt + H, pl:pl + W] = x
    y = np.zeros((N, w.shape[0], oh, ow))
    for a in range(kh):
        for b in range(kw):
            xs = xp[:, :, a * dh:a * dh + (oh - 1) * sh + 1:sh, b * dw:b * dw + (ow - 1) * sw + 1:sw]
            if dwise:
                y += xs * w[:, 0, a, b][None, :, None, None]
            else:
                y += np.einsum("nchw,mc->nmhw", xs, w[:, :, a, b], optimize=True)
    return y


def _weight(t):
    """_weight_value (_simulate.py:531-539): quantized data, times 2^(F - wexp) when encoded."""
    v = _quantize(np.asarray(t.data, np.float64).reshape(t.shape))
    if t.wexp is not None:
        v = v * np.power(2.0, F - np.asarray(t.wexp, np.float64))
    return v


def _pow2(*ts):
    return any(t is not None and (t.exp is not None or t.wexp is not None or t.chexp is not None) for t in ts)


def _wrap_floor(acc):
    """The ap_fixed<32,16> accumulator: wrap to int32, floor(/ 2^F), saturate (_simulate.py:826-831)."""
    big = np.abs(acc) >= 2.0 ** 31
    if big.any():
        acc = np.where(big, np.mod(acc + 2.0 ** 31, 2.0 ** 32) - 2.0 ** 31, acc)
    return np.clip(np.floor(acc / float(1 << F)), -32768, 32767)


def _matmul_exp(sn, a, b):
    """_simulate.py:814-835."""
    fo = np.asarray(F if sn.output.exp is None else sn.output.exp, np.float64)
    acc = np.matmul(a, b) * np.power(2.0, fo + F)
    assert np.array_equal(acc, np.round(acc)), "accumulator not on the 2^-(f_out+F) grid"
    return _wrap_floor(acc) / np.power(2.0, fo)


def _geom(sn):
    """(batch, in_ch, in_h, in_w, out_ch, out_h, out_w, kh, kw) of a Conv node from its shapes."""
    x, w, y = sn.inputs[0].shape, sn.inputs[1].shape, sn.output.shape
    return int(x[0]), int(x[1]), int(x[2]), int(x[3]), int(y[1]), int(y[2]), int(y[3]), int(w[2]), int(w[3])


def _has_bias(sn):
    return len(sn.inputs) > 2 and sn.inputs[2] is not None


def _conv_exp(sn, x, w, bias):
    """_simulate.py:784-812."""
    xt, wt, yt = sn.inputs[0], sn.inputs[1], sn.output
    N, C, H, W_, M, OH, OW, KH, KW = _geom(sn)
    fx = (np.asarray(xt.chexp, np.float64).reshape(1, -1, 1, 1) if xt.chexp is not None
          else float(np.asarray(F if xt.exp is None else xt.exp)))
    fy = (np.asarray(yt.chexp, np.float64).reshape(1, -1, 1, 1) if yt.chexp is not None
          else float(np.asarray(F if yt.exp is None else yt.exp)))
    fw = np.asarray(F if wt.wexp is None else wt.wexp, np.float64)
    x_raw = np.asarray(x, np.float64).reshape(N, C, H, W_) * np.power(2.0, fx)
    w_raw = np.asarray(w, np.float64).reshape(M, 1 if sn.is_depthwise else C, KH, KW) * np.power(2.0, fw)
    acc = _conv_int(x_raw, w_raw, sn.stride_h, sn.stride_w, sn.pad_top, sn.pad_left, sn.dilation_h,
                    sn.dilation_w, OH, OW, sn.is_depthwise)
    if bias is not None:
        acc = acc + (np.asarray(bias, np.float64).reshape(1, -1, 1, 1) * np.power(2.0, fy)) * 2.0 ** F
    assert np.array_equal(acc, np.round(acc)), "conv operands off their grids"
    return _wrap_floor(acc) / np.power(2.0, fy)


def _raw_of(t, v):
    """Raw integers of a tensor's values (per-channel exponents of the last axis or axis 1)."""
    if t.chexp is not None:
        e = np.asarray(t.chexp, np.float64).reshape((1, -1) + (1,) * (len(t.shape) - 2))
    else:
        e = np.asarray(F if t.exp is None else t.exp, np.float64)
    return np.rint(np.asarray(v, np.float64).reshape(t.shape) * np.power(2.0, e)).astype(np.int64)


def _attn_conv(sn, w, x, pos, n):
    """LlmAttnConvNode.reference (llm_nodes.py:1407-1425) on logical arrays; raw integers."""
    keys = sn.C if sn.static else clamp_n(int(pos), int(n) if sn.has_n else sn.T, sn.T, sn.C, sn.Q)[1]
    g, HD, GT = sn.group, sn.HD, (sn.H // sn.KV) * sn.T
    if sn.kind == "qk":
        kc = _raw_of(sn.inputs[0], w)[:keys, g * HD:(g + 1) * HD].astype(np.float64)
        B = np.asarray(x, np.float64).reshape(sn.KV, HD, GT)[g]
        out = np.zeros((sn.C, GT))
        out[:keys] = _wrap_floor(kc @ B)
        return out
    P = np.asarray(w, np.float64).reshape(GT, sn.C)[:, :keys]
    vc = _raw_of(sn.inputs[1], x)[:keys, g * HD:(g + 1) * HD].astype(np.float64)
    return _wrap_floor(P @ vc)


def _rows16(x2d, kind):
    rows, w = x2d.shape
    stride = (_KB[kind] * w + 15) & ~15
    img = np.zeros((rows, stride), np.uint8)
    img[:, :_KB[kind] * w] = np.ascontiguousarray(x2d.astype(_NP[kind])).view(np.uint8).reshape(rows, -1)
    return img.reshape(-1), stride


def _mask(sn, n, get):
    """The softmax node's mask register, a runtime one from its host tensor."""
    if getattr(sn, "mask_t", None) is not None:
        return int(np.asarray(get(sn.mask_t)).reshape(-1)[0]) + sn.mask_add
    return n if sn.mask is None else sn.mask


def _view_gather(v, x):
    """A head view's operand slices: [batch seq][ld] -> [batch heads][seq][width] from columns
    col .. col + heads width of each row block of seq rows."""
    ld = x.shape[-1]
    x = x.reshape(-1, v.seq, ld)[:, :, v.col:v.col + v.heads * v.width]
    return x.reshape(-1, v.seq, v.heads, v.width).transpose(0, 2, 1, 3).reshape(-1, v.seq, v.width)


def _view_scatter(v, y, ld):
    """[batch heads][seq][width] back into token rows [batch seq][ld] (a view covering the rows)."""
    assert v.col == 0 and v.heads * v.width == ld, "an output head view covers its tensor's rows"
    y = y.reshape(-1, v.heads, v.seq, v.width).transpose(0, 2, 1, 3)
    return y.reshape(-1, ld)


def _gather_index(sn):
    """The flat input index of every output element of a Permute node (dims / strides / offset)."""
    idx = np.full(tuple(sn.dims), int(sn.offset), np.int64)
    for k, (d, st) in enumerate(zip(sn.dims, sn.strides)):
        shape = [1, 1, 1, 1]
        shape[k] = int(d)
        idx = idx + (np.arange(int(d), dtype=np.int64) * int(st)).reshape(shape)
    return idx.reshape(-1)


def _chan(t, n):
    """Per-channel exponents of the last axis, n of them."""
    return np.broadcast_to(np.asarray(F if t.exp is None else t.exp, np.int64).reshape(-1), (n,)).copy()


_HOST_OPS = ("SoftmaxNode", "LayerNormNode", "GeluNode", "LlmRMSNormNode", "LlmSiluMulNode", "LlmResAddNode",
             "LlmDequantNode", "LlmToHostNode", "LlmAttentionNode")


def _host_op(sn, ins, vals):
    """The host ops' reference() bodies (oracle/host_ref.py)."""
    name, out = type(sn).__name__, sn.output
    if name == "SoftmaxNode":
        return host_ref.softmax(ins[0], int(sn.inputs[0].shape[-1]))
    if name == "LayerNormNode":
        return host_ref.layer_norm(ins[0], int(sn.inputs[0].shape[-1]), sn.gamma, sn.beta, sn.eps, sn.tf_form)
    if name == "GeluNode":
        return host_ref.gelu(ins[0], sn.approximate, sn.c1, sn.c2, sn.k, sn.div)
    if name == "LlmRMSNormNode":
        W = int(sn.inputs[0].shape[-1])
        return host_ref.rms_norm(ins[0], sn.gamma, sn.eps, _chan(out, W), W)
    if name == "LlmSiluMulNode":
        n = int(sn.inputs[0].shape[-1])
        return host_ref.silu_mul(ins[0], ins[1], _chan(sn.inputs[0], n), _chan(out, n))
    if name == "LlmResAddNode":
        return host_ref.f32(np.asarray(ins[0], np.float64) + np.asarray(ins[1], np.float64))
    if name in ("LlmDequantNode", "LlmToHostNode"):
        return host_ref.f32(ins[0])
    # LlmAttentionNode: the caches (states) in place
    H, KV, HD = sn.heads, sn.kv_heads, sn.head_dim
    q0t, ckt, cvt = sn.inputs[0], sn.inputs[-2], sn.inputs[-1]
    T = q0t.numel // (H * HD)
    pos = int(np.asarray(ins[3]).reshape(-1)[0])
    n = int(np.asarray(ins[4]).reshape(-1)[0]) if len(sn.inputs) == 7 else T
    ck = vals[ckt.onnx_name].reshape(ckt.shape)
    cv = vals[cvt.onnx_name].reshape(cvt.shape)
    return host_ref.attention(ins[0], ins[1], ins[2], pos, n, ck, cv, _chan(ckt, KV * HD), _chan(cvt, KV * HD),
                              _chan(out, H * HD), np.asarray(sn.cos, np.float32), np.asarray(sn.sin, np.float32),
                              T, H, KV, HD)


def _oracle_matmul(sn, a, b):
    """A MatMul through the C oracle's integer product on raw lanes: wrap32 for the pow2 path
    (_simulate.py:814-835), the exact sum for Q8.8 (:620-633)."""
    at, bt, out = sn.inputs[0], sn.inputs[1], sn.output
    k, m = int(bt.shape[-2]), int(bt.shape[-1])
    pow2 = _pow2(at, bt, out)
    fo = np.broadcast_to(np.asarray(F if out.exp is None or not pow2 else out.exp, np.float64).reshape(-1), (m,))
    ra = (_raw_of(at, a) if pow2 else _to_raw(a)).reshape(-1, k).astype(np.int16)
    if pow2:
        fb = (np.asarray(F if bt.wexp is None else bt.wexp, np.float64) if bt.wexp is not None
              else np.asarray(F if bt.exp is None else bt.exp, np.float64))
        rb = np.rint(np.asarray(b, np.float64).reshape(k, m) * np.power(2.0, fb)).astype(np.int16)
    else:
        rb = _to_raw(b).reshape(k, m)
    n = ra.shape[0]
    c = cm.matmul(np.ascontiguousarray(ra).reshape(-1), np.ascontiguousarray(rb.T).reshape(-1), n, k, m,
                  b_packed=2, wrap32=pow2)
    return (c.reshape(n, m).astype(np.float64) / np.power(2.0, fo)).reshape(out.shape)


def _oracle_contract(a, b):
    """sat16(floor(wrap32(a . b) / 2^8)) of raw int16 matrices a [n][k], b [k][m] through the C oracle."""
    n, k = a.shape
    m = b.shape[1]
    c = cm.matmul(np.ascontiguousarray(a, np.int16).reshape(-1), np.ascontiguousarray(b.T, np.int16).reshape(-1),
                  n, k, m, b_packed=2, wrap32=True)
    return c.reshape(n, m).astype(np.int64)


_UNIT_ACT_OF_OP = {6: 3, 7: 4, 8: 5, 9: 6}      # the activation ops and the act they apply


def _ref_norm(sn, x):
    """A row-ops norm adapter by the reference simulator's per-row integer loop (sim_ref)."""
    kind, x_t, y = type(sn).__name__, sn.inputs[0], sn.output
    W = int(x_t.shape[-1])
    fo = rowops_adapt._chan(y, W, getattr(sn, "F", F))
    if kind == "RMSNormRoNode":
        gamma = np.asarray(sn.gamma, np.float64).reshape(-1)
        n = gamma.size
        fx = rowops_adapt._chan(x_t, W, getattr(sn, "F", F))
        raw = rowops_adapt._raw(x_t, x, W).astype(np.int64).reshape(-1, n)
        r = sim_ref.rms_norm(raw, int(fx[0]), gamma, sn.eps, fo[:n]).reshape(-1, W)
    else:
        fx = rowops_adapt._chan(x_t, W, getattr(sn, "F", F))
        raw = rowops_adapt._raw(x_t, x, W).astype(np.int64)
        gamma = np.ones(W) if sn.gamma is None else np.asarray(sn.gamma, np.float64).reshape(-1)
        beta = np.zeros(W) if sn.beta is None else np.asarray(sn.beta, np.float64).reshape(-1)
        r = sim_ref.layer_norm(raw, int(fx[0]), gamma, beta, sn.eps, fo)
    return r.astype(np.float64) / np.power(2.0, fo.astype(np.float64))


def _paged_prep(sn, pool, qs, kl, tb, x):
    """The norms at the rotation's output exponents (sim_ref.rms_norm), the rotation, the cache rows."""
    HD = sn.head_dim
    exps = [int(F if t.exp is None else t.exp) for t in list(sn.inputs[:2]) + [sn.output]]
    cos, sin = (np.rint(np.asarray(t, np.float32).astype(np.float64) * 2.0 ** 23).astype(np.int64) for t in (sn.cos, sn.sin))
    both = (lambda t: np.repeat(t, 2, axis=1)) if sn.interleaved else (lambda t: np.concatenate([t, t], axis=1))
    shifts = []
    for i, (gamma, fo) in enumerate(((sn.gamma_q, exps[2]), (sn.gamma_k, sn.f_k))):
        fi = exps[i]
        if gamma is not None:
            shape = x[i].shape
            x[i] = sim_ref.rms_norm(np.asarray(x[i], np.int64).reshape(-1, HD), fi, np.asarray(gamma, np.float64), sn.eps,
                                    np.full(HD, fo)).reshape(shape)
            fi = fo
        shifts.append((0, 0, fi + 23 - fo))
    qr = np.zeros((x[0].shape[0], sn.heads * HD), np.int64)
    oracle_paged.prep(pool, qs, kl, tb, x[0], x[1], x[2], qr, np.concatenate([both(cos), both(sin)], axis=1),
                      2 * cos.shape[1], sn.interleaved, shifts[0], shifts[1])
    return qr


ALGOS = ("port", "ref", "oracle")


def forward(graph, inputs, states=None, algo="port", errors_out=None):
    """Every tensor's float64 values.  ``states`` ({name: float64 array}) are the persistent
    states, updated in place (_simulate.py:573-577); default: zeros, or copies of the inputs
    of those names.  ``algo`` picks how the costly units are computed, with the same results:
    "port" (float64 BLAS contractions, the C oracle for the units), "ref" (as "port" but the
    row-ops norms and the activation unit by the reference simulator's own algorithms,
    oracle/sim_ref.py) or "oracle" (every MatMul and attention contraction through the C
    oracle's integer product on all cores).  ``errors_out`` (a dict) receives {output name:
    (abs_max, nrmse, sqnr_db)} of every MatMul, Conv without exponents, Pool and VectorOP node:
    the full-precision result against the stored one (_simulate.py:594-602, 814-835)."""
    if algo not in ALGOS:
        raise ValueError(f"algo {algo!r}: one of {ALGOS}")
    vals = {k: np.array(v, np.float64) for k, v in inputs.items()}      # copies: states change in place
    for t in getattr(graph, "state_tensors", []):
        if states is not None and t.onnx_name in states:
            vals[t.onnx_name] = states[t.onnx_name]
        elif t.onnx_name not in vals:
            vals[t.onnx_name] = np.zeros(t.shape)
    get = lambda t: vals[t.onnx_name] if t.onnx_name in vals else _weight(t)

    def record(sn, full):
        if errors_out is not None:
            errors_out[sn.output.onnx_name] = residual_ref.residual_stats(
                np.asarray(full).reshape(sn.output.shape), vals[sn.output.onnx_name])

    for sn in graph.nodes:
        out = sn.output
        kind = _kind(sn)
        if kind in ("MatmulNode", "MatmulConvNode"):
            # a MatMul lowered onto the conv unit computes exactly MatmulNode's result
            # (_simulate.py:620-633 treats both alike)
            a, b = get(sn.inputs[0]), get(sn.inputs[1])
            if algo == "oracle" and kind == "MatmulNode" and len(sn.inputs[1].shape) == 2:
                vals[out.onnx_name] = _oracle_matmul(sn, a, b)
            elif _pow2(sn.inputs[0], sn.inputs[1], out):
                vals[out.onnx_name] = _matmul_exp(sn, a, b).reshape(out.shape)
            else:
                vals[out.onnx_name] = _truncate(np.matmul(a, b)).reshape(out.shape)
            if errors_out is not None:
                record(sn, np.matmul(a, b))
        elif kind == "ConvNode" and _pow2(*sn.inputs[:2], out):
            vals[out.onnx_name] = _conv_exp(sn, get(sn.inputs[0]), get(sn.inputs[1]),
                                            get(sn.inputs[2]) if _has_bias(sn) else None).reshape(out.shape)
        elif kind == "LlmAttnConvNode":
            pos = get(sn.inputs[2]) if not sn.static else 0
            n = get(sn.inputs[3]) if not sn.static and sn.has_n else sn.T
            vals[out.onnx_name] = _attn_conv(sn, get(sn.inputs[0]), get(sn.inputs[1]), np.asarray(pos).reshape(-1)[0],
                                             np.asarray(n).reshape(-1)[0]).reshape(out.shape)
        elif algo == "ref" and kind in ("LayerNormRoNode", "LayerNorm32RoNode", "RMSNormRoNode"):
            vals[out.onnx_name] = _ref_norm(sn, get(sn.inputs[0])).reshape(out.shape)
        elif kind in ADAPTERS:
            host = lambda t: int(np.asarray(get(t)).reshape(-1)[0])        # noqa: E731
            vals[out.onnx_name] = rowops_adapt.adapter(sn, [get(t) for t in sn.inputs], host).reshape(out.shape)
        elif kind == "ConvNode":
            x, w = get(sn.inputs[0]), get(sn.inputs[1])
            OH, OW = _geom(sn)[5:7]
            acc = _conv_int(x * 256, w * 256, sn.stride_h, sn.stride_w, sn.pad_top, sn.pad_left,
                            sn.dilation_h, sn.dilation_w, OH, OW, sn.is_depthwise) / 65536.0
            if _has_bias(sn):
                acc = acc + get(sn.inputs[2]).reshape(1, -1, 1, 1)
            vals[out.onnx_name] = _truncate(acc).reshape(out.shape)
            record(sn, acc)
        elif kind == "AttentionNode":
            # the reference's chain per (sequence, head): s = K . Q^T keys-major (int32 wrap,
            # floor / 2^8), the softmax unit's keys-major call (VectorOP op 11), P . V
            xt = sn.inputs[0]
            B, T, H, hd = sn.batch, sn.seq, sn.heads, sn.head_dim
            x = _raw_of(xt, get(xt)).reshape(B, T, -1).astype(np.int64)
            k8 = (T + 7) & ~7
            o = np.zeros((B, T, H * hd), np.int64)
            for b in range(B):
                for h in range(H):
                    q = x[b, :, sn.q_off + h * hd:sn.q_off + (h + 1) * hd].astype(np.float64)
                    k = x[b, :, sn.k_off + h * hd:sn.k_off + (h + 1) * hd].astype(np.float64)
                    v = x[b, :, sn.v_off + h * hd:sn.v_off + (h + 1) * hd].astype(np.float64)
                    if algo == "oracle":
                        s_ = _oracle_contract(k, q.T).astype(np.int16)
                    else:
                        s_ = _wrap_floor(k @ q.T).astype(np.int16)                   # [keys][queries]
                    p_ = cm.vectorop(np.ascontiguousarray(s_.reshape(-1)), None, T * k8, T, 11, T, T, k8, 0, 0,
                                     sn.cm, sn.cfg, T).reshape(T, k8)[:, :T]
                    if algo == "oracle":
                        o[b, :, h * hd:(h + 1) * hd] = _oracle_contract(p_, v)
                    else:
                        o[b, :, h * hd:(h + 1) * hd] = _wrap_floor(p_.astype(np.float64) @ v)
            fo = float(F if out.exp is None else out.exp)
            vals[out.onnx_name] = (o.astype(np.float64) / 2.0 ** fo).reshape(out.shape)
        elif kind == "AttnSoftmaxNode":
            # LlmAttnSoftmaxVopNode.reference (smx_nodes.py:326-338): per head h', the column-mode
            # softmax of s_g[:keys][h' T + t] with the valid lengths causal_valid(T, pos + 1, T,
            # keys) (vectorop_smx.py:75-79); column mode is the row mode of the transpose
            # (softmax_cols, :69-72): one row-mode call of the C oracle per column, its valid
            # length as a period-0 mask
            st = sn.inputs[0]
            T, G, C = sn.T, sn.G, sn.C
            if len(sn.inputs) == 1:                 # static (VitAttnSoftmax): pos 0, n = T
                pos, n_in = 0, T
            else:
                pos = int(np.asarray(get(sn.inputs[1])).reshape(-1)[0])
                n_in = int(np.asarray(get(sn.inputs[2])).reshape(-1)[0]) if len(sn.inputs) == 3 else T
            n, keys = clamp_n(pos, n_in, T, C, sn.Q)
            valid = (np.minimum(keys, pos + 1 + np.arange(T)) if sn.causal
                     else np.full(T, max(min(keys, pos + n), 1)))
            s_ = _raw_of(st, get(st)).reshape(C, G * T).astype(np.int16)
            cms = np.broadcast_to(np.asarray(sn.cm).reshape(-1), (G,))
            cfgs = np.broadcast_to(np.asarray(sn.cfg).reshape(-1), (G,))
            k8 = (keys + 7) & ~7
            P = np.zeros((G * T, C))
            for h in range(G):
                for t in range(T):
                    col = np.ascontiguousarray(s_[:keys, h * T + t])
                    P[h * T + t, :keys] = cm.vectorop(col, None, k8, keys, 10, 1, k8, k8, 0, 0, int(cms[h]),
                                                      int(cfgs[h]), int(valid[t]))[:keys]
            vals[out.onnx_name] = P.reshape(out.shape)
        elif kind == "AttnMergeNode":
            # LlmAttnMergeNode.reference (llm_nodes.py:1660-1675): pv[t][(g G + h') HD + d] = o_g[h' T + t][d]
            T, H, KV, HD = sn.T, sn.H, sn.KV, sn.HD
            G = H // KV
            r = np.zeros((T, H, HD))
            for g, t_ in enumerate(sn.inputs):
                o_ = _raw_of(t_, get(t_)).reshape(G, T, HD)
                for hh in range(G):
                    r[:, g * G + hh, :] = o_[hh]
            fo = np.asarray(F if out.exp is None else out.exp, np.float64)
            vals[out.onnx_name] = (r.reshape(T, H * HD) / np.power(2.0, fo)).reshape(out.shape)
        elif kind == "SelectRowNode":
            # LlmSelectRowNode.reference (llm_nodes.py:1714-1718): row n - 1, n clamped to [1, rows]
            ht = sn.inputs[0]
            w = int(ht.shape[-1])
            rows = ht.numel // w
            r = min(max(int(np.asarray(get(sn.inputs[1])).reshape(-1)[0]), 1), rows) - 1
            y = np.asarray(get(ht), np.float64).reshape(rows, w)[r].reshape(out.shape)
            if out.onnx_name in vals and getattr(out, "state", False):
                vals[out.onnx_name][...] = y.reshape(vals[out.onnx_name].shape)       # the state, in place
            else:
                vals[out.onnx_name] = y.copy()
        elif kind == "LlmEmbedNode":
            fo = F if out.exp is None else np.asarray(out.exp).reshape(-1)[0]
            vals[out.onnx_name] = host_ref.embed(get(sn.inputs[0]), sn.table, sn.scale, fo,
                                                 out.kind == "i32").reshape(out.shape)
        elif kind in _HOST_OPS:
            vals[out.onnx_name] = _host_op(sn, [get(t) for t in sn.inputs], vals).reshape(out.shape)
        elif kind in ("TransposeRoNode", "TransposeNode"):
            xt = sn.inputs[0]
            vals[out.onnx_name] = transpose(get(xt).reshape(xt.shape), sn.perm).reshape(out.shape)
        elif kind == "AttnPrepRoNode":
            q0t, k0t, vt, pt = sn.inputs[:4]
            ckt, cvt = sn.inputs[-2], sn.inputs[-1]
            H, KV, HD = sn.heads, sn.kv_heads, sn.head_dim
            T = q0t.numel // (H * HD)
            pos = int(np.asarray(get(pt)).reshape(-1)[0])
            n = int(np.asarray(get(sn.inputs[4])).reshape(-1)[0]) if len(sn.inputs) == 7 else T
            ck = vals[ckt.onnx_name].reshape(ckt.shape)                # the states, in place
            cv = vals[cvt.onnx_name].reshape(cvt.shape)
            vals[out.onnx_name] = attn_prep(get(q0t), get(k0t), get(vt), pos, n, ck, cv, _chan(q0t, H * HD),
                                            _chan(k0t, KV * HD), _chan(vt, KV * HD), _chan(ckt, KV * HD),
                                            _chan(cvt, KV * HD), sn.fq, sn.cos, sn.sin, H, KV, HD,
                                            sn.key_quantum).reshape(out.shape)
        elif kind == "VitAttnPrepRoNode":
            H, HD = sn.heads, sn.head_dim
            D = H * HD
            rows = []
            for t_, col in zip(sn.inputs[:3], sn.cols):
                w = int(t_.shape[-1])
                r = _raw_of(t_, get(t_)).reshape(-1, w)[:, col:col + D]
                rows.append((r, _chan(t_, w)[col:col + D]))
            zero = np.zeros(D)
            b = [zero if x is None else np.asarray(x, np.float64).reshape(-1) for x in (sn.bq, sn.bk, sn.bv)]
            qx, ck, cv = vit_attn_prep(rows[0][0], rows[1][0], rows[2][0], rows[0][1], rows[1][1], rows[2][1], *b,
                                       sn.fq, sn.fk, sn.fv, H, HD, sn.query_major)
            vals[sn.inputs[3].onnx_name].reshape(-1, D)[...] = ck            # the states, in place (raw)
            vals[sn.inputs[4].onnx_name].reshape(-1, D)[...] = cv
            vals[out.onnx_name] = qx.astype(np.float64).reshape(out.shape)
        elif kind == "KvWriteNode":
            xt, ct = sn.inputs[0], sn.inputs[1]
            B, KV, C, HD = (int(v) for v in ct.shape)
            cache = vals[ct.onnx_name].reshape(B, KV, C, HD)          # the state, written in place
            pos = sn.pos if sn.pos_t is None else int(np.asarray(get(sn.pos_t)).reshape(-1)[0])
            cache[:, :, pos, :] = get(xt).reshape(B, KV, HD)
            vals[out.onnx_name] = cache
        elif kind == "ReshapeNode":
            vals[out.onnx_name] = get(sn.inputs[0]).reshape(out.shape)
        elif kind == "PoolNode":
            xt = sn.inputs[0]
            raw = _to_raw(get(xt)).reshape(-1)
            y = cm.pool(raw, xt.shape[0], xt.shape[1], xt.shape[2], xt.shape[3], out.shape[2],
                        out.shape[3], sn.pool_h, sn.pool_w, sn.stride_h, sn.stride_w, sn.pad_top,
                        sn.pad_left, sn.dil_h, sn.dil_w, sn.pool_type, sn.lp_order, sn.count_include_pad)
            vals[out.onnx_name] = _from_raw(y).reshape(out.shape)
            if errors_out is not None:
                record(sn, residual_ref.pool_full(get(xt).reshape(xt.shape), sn.pool_h, sn.pool_w, sn.stride_h,
                                                  sn.stride_w, sn.pad_top, sn.pad_left, sn.dil_h, sn.dil_w,
                                                  out.shape[2], out.shape[3], sn.pool_type, sn.lp_order,
                                                  sn.count_include_pad))
        elif kind == "SoftmaxVopNode":
            xt = sn.inputs[0]
            x = _raw_of(xt, get(xt))
            fp = (sn.cfg >> 8) & 31
            if sn.keys_major:
                # per matrix s[keys][queries] -> P[queries][keys] (VectorOP op 11)
                keys, nq = xt.shape[-2], xt.shape[-1]
                k8 = (keys + 7) & ~7
                mats = x.reshape(-1, keys, nq)
                ps = []
                for m in mats:
                    c = cm.vectorop(np.ascontiguousarray(m.reshape(-1), np.int16), None, nq * k8, keys, 11, nq, nq, k8, 0, 0,
                                    sn.cm, sn.cfg, _mask(sn, keys, get))
                    ps.append(c.reshape(nq, k8)[:, :keys])
                vals[out.onnx_name] = (np.stack(ps).astype(np.float64) / 2.0 ** fp).reshape(out.shape)
            else:
                n = x.shape[-1]
                rows = x.size // n
                n8 = (n + 7) & ~7
                xr = np.zeros((rows, n8), np.int16)
                xr[:, :n] = x.reshape(rows, n)
                c = cm.vectorop(xr.reshape(-1), None, rows * n8, n, 10, rows, n8, n8, 0, 0, sn.cm, sn.cfg,
                                _mask(sn, n, get))
                vals[out.onnx_name] = (c.reshape(rows, n8)[:, :n].astype(np.float64) / 2.0 ** fp).reshape(out.shape)
        elif kind == "DecodePrepNode":
            # RoPE of q (the output) and k (at the K cache's exponent) at the position, then the
            # cache rows: the RoPE and KV-write nodes of the unfused step
            qt, kt, vt, kct, vct = sn.inputs[:5]
            B, KV, C, HD = (int(x) for x in kct.shape)
            pos = sn.pos if sn.pos_t is None else int(np.asarray(get(sn.pos_t)).reshape(-1)[0])
            kr = SimpleNamespace(onnx_name="k_rope", shape=list(kt.shape), exp=kct.exp, kind="i16")
            rq = _RopeRoNode(inputs=[qt], output=out, heads=sn.heads, head_dim=HD, cos=sn.cos, sin=sn.sin,
                             pos=pos, pos_t=None, same_pos=True, F=getattr(sn, "F", 8))
            rk = _RopeRoNode(inputs=[kt], output=kr, heads=KV, head_dim=HD, cos=sn.cos, sin=sn.sin, pos=pos,
                             pos_t=None, same_pos=True, F=getattr(sn, "F", 8))
            vals[out.onnx_name] = rowops_adapt.adapter(rq, [get(qt)]).reshape(out.shape)
            kcache = vals[kct.onnx_name].reshape(B, KV, C, HD)       # the states, written in place
            vcache = vals[vct.onnx_name].reshape(B, KV, C, HD)
            kcache[:, :, pos, :] = rowops_adapt.adapter(rk, [get(kt)]).reshape(B, KV, HD)
            vcache[:, :, pos, :] = get(vt).reshape(B, KV, HD)
        elif kind in ("PagedPrepNode", "PagedAttentionNode"):
            pt, qst, klt, tbt = sn.inputs[-4:]
            words = vals[pt.onnx_name]                               # the state, written in place
            pool = oracle_paged.Pool(int(pt.shape[0]), sn.page, sn.kv_heads, sn.head_dim, sn.int8,
                                     np.ascontiguousarray(words).astype(np.int32).view(np.uint8))
            qs, kl, tb = (np.asarray(get(t)).astype(np.int64) for t in (qst, klt, tbt))
            rows = lambda t: _raw_of(t, get(t)).reshape(t.shape)     # noqa: E731
            if kind == "PagedAttentionNode":
                r = oracle_paged.attend(pool, qs, kl, tb, rows(sn.inputs[0]), sn.heads, sn.cm, sn.cfg, sn.window)
            else:
                r = _paged_prep(sn, pool, qs, kl, tb, [rows(t) for t in sn.inputs[:3]])
                words[...] = pool.data.view(np.int32).astype(np.float64).reshape(words.shape)
            vals[out.onnx_name] = (r / 2.0 ** float(F if out.exp is None else out.exp)).reshape(out.shape)
        elif kind in ("Linear8Node", "GatedLinear8Node"):
            xt = sn.inputs[0]
            x = _raw_of(xt, get(xt)).reshape(-1, int(xt.shape[-1]))
            if kind == "GatedLinear8Node":
                table = None if sn.act == "silu" else cm.act_table(5 if sn.act == "gelu" else 6)
                r = oracle_linear8.gated(x, sn.gate_codes, sn.up_codes, sn.gate_mult, sn.up_mult, sn.act, sn.gate_shift,
                                         sn.out_shift, table)
            else:
                res = None if len(sn.inputs) < 3 else _raw_of(sn.inputs[2], get(sn.inputs[2])).reshape(-1, int(out.shape[-1]))
                r = oracle_linear8.linear(x, sn.codes, sn.mult, sn.bias_raw, res, sn.shift)
            fo = np.asarray(F if out.exp is None else out.exp, np.float64)
            vals[out.onnx_name] = (r.reshape(out.shape) / 2.0 ** fo).reshape(out.shape)
        elif kind == "ColumnsNode":
            v = get(sn.inputs[0])
            vals[out.onnx_name] = v.reshape(-1, v.shape[-1])[:, sn.first:sn.first + int(out.shape[-1])].reshape(out.shape).copy()
        elif kind == "DecodeAttentionNode":
            # per KV group: s = q K^T (wrap rule), the row-mode softmax (VectorOP op 10), o = P V
            qt, kt, vt = sn.inputs[:3]
            B, KV, C, HD = (int(x) for x in kt.shape)
            G = sn.heads // sn.kv_heads
            qg = _raw_of(qt, get(qt)).reshape(B * KV, G, HD).astype(np.float64)
            kg = _raw_of(kt, get(kt)).reshape(B * KV, C, HD).astype(np.float64)
            vg = _raw_of(vt, get(vt)).reshape(B * KV, C, HD).astype(np.float64)
            s_ = _wrap_floor(np.matmul(qg, kg.transpose(0, 2, 1))).astype(np.int16)
            rows, c8 = B * KV * G, (C + 7) & ~7
            xr = np.zeros((rows, c8), np.int16)
            xr[:, :C] = s_.reshape(rows, C)
            p_ = cm.vectorop(xr.reshape(-1), None, rows * c8, C, 10, rows, c8, c8, 0, 0, sn.cm, sn.cfg,
                             _mask(sn, C, get)).reshape(rows, c8)[:, :C]
            o_ = _wrap_floor(np.matmul(p_.reshape(B * KV, G, C).astype(np.float64), vg))
            fo = float(F if out.exp is None else out.exp)
            vals[out.onnx_name] = (o_ / 2.0 ** fo).reshape(out.shape)
        elif kind == "AttnContractNode":
            at, bt = sn.inputs
            # operands as [slices][rows][cols]: their own 3-d shape or a head view's gather
            ops = [_raw_of(t, get(t)).reshape(t.shape) if v is None else _view_gather(v, _raw_of(t, get(t)))
                   for t, v in ((at, sn.a_view), (bt, sn.b_view))]
            ra, rb = ops
            if sn.b_trans:
                rb = rb.transpose(0, 2, 1)
            acc = np.matmul(ra.astype(np.float64), rb.astype(np.float64))   # |sums| < 2^53: exact
            fo = float(F if out.exp is None else out.exp)
            r = _wrap_floor(acc)
            if sn.c_view is not None:
                r = _view_scatter(sn.c_view, r, int(out.shape[-1]))
            vals[out.onnx_name] = (r / 2.0 ** fo).reshape(out.shape)
        elif kind == "PermuteNode":
            vals[out.onnx_name] = get(sn.inputs[0]).reshape(-1)[_gather_index(sn)].reshape(out.shape)
        elif kind == "ScheduledNode":
            # numpy broadcasting of the logical arrays (_simulate.py:721-765), on raw lanes
            full = lambda t: np.broadcast_to(get(t).reshape([1] * (len(out.shape) - len(t.shape)) + list(t.shape)),
                                             out.shape)
            binary = sn.op_code < 4                     # ADD / SUB / MUL / DIV read b
            ar = _to_raw(full(sn.inputs[0])).reshape(-1)
            br = _to_raw(full(sn.inputs[1])).reshape(-1) if binary else None
            n = ar.size
            unit_act = _UNIT_ACT_OF_OP.get(sn.op_code, sn.act if sn.act >= 3 else 0)
            if algo == "ref" and unit_act:
                # the op's floored result, then the activation unit per element with libm
                x = ar if sn.op_code in _UNIT_ACT_OF_OP else cm.vectorop(ar, br, (n + 7) & ~7, n, sn.op_code, 1, 0,
                                                                         0, 0, 0)[:n]
                vals[out.onnx_name] = _from_raw(sim_ref.act_unit(unit_act, x, sn.alpha)).reshape(out.shape)
            else:
                c = cm.vectorop(ar, br, (n + 7) & ~7, n, sn.op_code, 1, 0, 0, sn.act, sn.alpha)
                vals[out.onnx_name] = _from_raw(c[:n]).reshape(out.shape)
            if errors_out is not None:
                record(sn, residual_ref.vectorop_full(sn.op_code, sn.act, sn.alpha, full(sn.inputs[0]),
                                                      full(sn.inputs[1]) if binary else None)[0])
        else:
            raise NotImplementedError(type(sn).__name__)
    return vals
