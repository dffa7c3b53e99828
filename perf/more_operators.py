"""The 8-bit linear layers of a decoder: their measured cases, their plain forms and their definitions.

Two operators on the framework's raw int16 rows, with weights of 8 bits:

  linear   o = x W: each row's 8-bit codes (a scale a token, found in the call), the product with 8-bit
           weights, a multiplier a channel, optionally a bias; int16 out, or added to an int32 residual
  gated    y = act(x Wg) * (x Wu): a feed-forward block's gate and up products, the activation and the
           product of the two

Every output is a whole number that the operators' integer definitions give bit for bit:
  a_t = max_k |x|, R = floor((127 2^24 + floor(a_t / 2)) / a_t), c = floor((x R + 2^23) / 2^24)
  o = sat16(rne(a_t mu_j sum_k c w + b_j)); with a residual h: sat32(h + o 2^shift)
  y = sat16(rne(act(g) u / 2^sc)), g and u as o; SiLU at 2^-20 by the row-ops unit's sigmoid pieces,
  GELU at 2^-8 by the activation unit's table.

``own`` False: ``run`` is the plain form, elementary torch operations (float64 products, exact for these
operands, and int64).  ``own`` True: ``run`` is the call a program makes of the framework.
"""
import math

import torch

own = False

X_EXP = 9                        # a normalised row: raw = value 2^9
STD = 0.6                        # of its values
W_STD = 0.02                     # of a weight
MULT_BITS = 18                   # of a channel's multiplier M 2^-s
G_EXP, U_EXP, Y_EXP = 10, 10, 11
ACT_EXP = 8                      # the activation unit's rows


def listed():
    def linear(name, n, k, m, **more):
        return dict(dict(name=name, kind="linear", n=n, k=k, m=m, bias=False, residual=False, shift=0), **more)

    def gated(name, n, k, m, act="silu"):
        return dict(name=name, kind="gated", n=n, k=k, m=m, act=act)
    return [
        # one token through an output projection of the decoder configuration: launch latency alone
        linear("linear_n1_960x960", 1, 960, 960),
        # the decode step's down projection into the residual stream, 16 sequences
        linear("linear_n16_2560x960_residual", 16, 2560, 960, residual=True, shift=4),
        # the decode step's head
        linear("linear_n16_960x49152", 16, 960, 49152),
        # a prompt chunk's fused q / k / v projection of odd length, with a bias
        linear("linear_n333_960x1600_bias", 333, 960, 1600, bias=True),
        # odd sizes everywhere
        linear("linear_n77_1001x1537", 77, 1001, 1537, bias=True),
        # a prompt of 512 tokens, the down projection into the residual stream
        linear("linear_n512_2560x960_residual", 512, 2560, 960, residual=True, shift=4),
        # the matrix benchmark's rows and weight (4 x 512 rows)
        linear("linear_n2048_4096x4096", 2048, 4096, 4096),
        # a long prompt through a wide layer
        linear("linear_n8192_4096x8192", 8192, 4096, 8192),
        # one token through the decoder configuration's feed-forward gate
        gated("gated_n1_960x2560", 1, 960, 2560),
        # its decode step
        gated("gated_n16_960x2560", 16, 960, 2560),
        # a ragged prompt through a GELU gate of odd width
        gated("gated_n777_768x2049_gelu", 777, 768, 2049, act="gelu"),
        # a long prompt through a wide feed-forward block
        gated("gated_n4096_4096x8192", 4096, 4096, 8192),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    limit = {kind: max(work(c)["flops"] for c in listed() if c["kind"] == kind) for kind in ("linear", "gated")}
    while True:
        kind = rng.choice(["linear", "linear", "gated"])
        n = rng.choice([1, _log(rng, 1, 32), _log(rng, 1, 8192), _log(rng, 32, 8192)])
        k, m = _log(rng, 64, 8192), _log(rng, 64, 16384)
        if rng.random() < 0.6:                       # widths of models: multiples of 64; else any
            k, m = -(-k // 64) * 64, -(-m // 64) * 64
        case = dict(kind=kind, n=n, k=k, m=m)
        if kind == "linear":
            case.update(bias=rng.random() < 0.4, residual=rng.random() < 0.4, shift=rng.randint(0, 6))
        else:
            case.update(act=rng.choice(["silu", "silu", "gelu", "gelu_tanh"]))
        if work(case)["flops"] <= limit[kind]:
            return case


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n, k, m = case["n"], case["k"], case["m"]
    if case["kind"] == "gated":
        return {"bytes": 2 * n * k + 2 * k * m + 16 * m + 2 * n * m, "flops": 4 * n * k * m}
    out = 8 * n * m if case["residual"] else 2 * n * m
    return {"bytes": 2 * n * k + k * m + 8 * m + (4 * m if case["bias"] else 0) + out, "flops": 2 * n * k * m}


# ------------------------------------------------------------------ inputs
def _weight(gen, k, m, f_out):
    """(int8 codes [k][m], M, s, mu = M 2^-s): a weight's channels at their own scales of 127 steps,
    the multiplier of a_t acc: (channel scale) 2^(f_out - X_EXP) / 127, M of MULT_BITS bits."""
    w = torch.randn(k, m, generator=gen, device="cuda", dtype=torch.float32)
    w *= W_STD * torch.exp(0.3 * torch.randn(m, generator=gen, device="cuda"))       # channels of unequal size
    top = w.abs().amax(0)
    codes = (w * (127.0 / top)).round_().clamp_(-127, 127).to(torch.int8)
    mu = top.double() / 127.0 * 2.0 ** (f_out - X_EXP) / 127.0
    s = MULT_BITS - torch.frexp(mu)[1]
    M = torch.round(mu * torch.exp2(s.double())).long()
    return codes, M, s.long(), M.double() * torch.exp2(-s.double())


def _logical(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, k, m = case["n"], case["k"], case["m"]
    x = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float32)
    loud = torch.rand(k, generator=gen, device="cuda") < 0.005                       # a few channels speak louder
    x *= STD * 2.0 ** X_EXP * torch.where(loud, 8.0, 1.0)
    x *= torch.exp(0.5 * torch.randn(n, 1, generator=gen, device="cuda"))            # and tokens differ
    d = {"x": x.round_().clamp_(-32768, 32767).to(torch.int16)}
    if case["kind"] == "gated":
        f_g = G_EXP if case["act"] == "silu" else ACT_EXP
        d["gate"], d["up"] = _weight(gen, k, m, f_g), _weight(gen, k, m, U_EXP)
        d["sa"] = 14 - f_g
        d["sc"] = (20 if case["act"] == "silu" else ACT_EXP) + U_EXP - Y_EXP
        return d
    d["w"] = _weight(gen, k, m, 11)
    d["b"] = (torch.randn(m, generator=gen, device="cuda") * 200).round().to(torch.int32) if case["bias"] else None
    if case["residual"]:
        d["h"] = (torch.randn(n, m, generator=gen, device="cuda") * 2.0 ** 16).round().to(torch.int32)
    return d


def prepare(case, seed):
    st = _logical(case, seed)
    n, m = case["n"], case["m"]
    st["case"] = case
    st["out"] = torch.zeros(n, m, dtype=torch.int32 if case.get("residual") else torch.int16, device="cuda")
    if not own:
        if case["kind"] == "gated":
            st["sigmoid"], st["act"] = _sigmoid(), _act_table(case["act"])
        return st
    from cormorant_amd import linear8
    if case["kind"] == "gated":
        g, u = st.pop("gate"), st.pop("up")
        f_g = G_EXP if case["act"] == "silu" else ACT_EXP
        st["weight"] = linear8.GatedWeight8(g[0], u[0], g[3], u[3], act=case["act"], gate_exp=f_g, up_exp=U_EXP,
                                            out_exp=Y_EXP)
    else:
        w = st.pop("w")
        st["weight"] = linear8.Weight8(w[0], w[3], bias=st["b"])
    return st


# ------------------------------------------------------------------ plain forms
def _sigmoid():
    """The row-ops unit's pieces of the sigmoid at 2^-24: values at i / 256, i = 0 .. 4096."""
    i = torch.arange(4097, device="cuda", dtype=torch.float64)
    return torch.round(2.0 ** 24 / (1.0 + torch.exp(-i / 256.0))).long()


def _act_table(act):
    """The activation unit's GELU at 2^-8 of every int16 (None for SiLU), index raw + 32768."""
    if act == "silu":
        return None
    v = torch.arange(-32768, 32768, device="cuda", dtype=torch.float64) / 256.0
    if act == "gelu":
        f = 0.5 * v * (1.0 + torch.erf(v / math.sqrt(2.0)))
    else:
        f = 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return torch.round(f * 256.0).clamp(-32768, 32767).long()


def _rne(x, e):
    """Round half to even of x / 2^e (int64, e a tensor of shifts >= 1 that broadcasts)."""
    q = x >> e
    rem = x - (q << e)
    half = torch.ones_like(e) << (e - 1)
    return q + ((rem > half) | ((rem == half) & (q & 1 == 1))).long()


def _codes(x):
    x = x.long()
    a = x.abs().amax(1, keepdim=True)
    r = torch.where(a > 0, (127 * 2 ** 24 + (a >> 1)) // a.clamp(min=1), torch.zeros_like(a))
    return (x * r + 2 ** 23) >> 24, a


def _product(codes, a, weight, b):
    w, M, s, _ = weight
    acc = (codes.double() @ w.double()).long()
    y = acc * a * M
    if b is not None:
        y += b.long() << s
    return _rne(y, s).clamp(-32768, 32767)


def _run_plain(st):
    case, out = st["case"], st["out"]
    codes, a = _codes(st["x"])
    if case["kind"] == "linear":
        o = _product(codes, a, st["w"], st["b"])
        if case["residual"]:
            o = (st["h"].long() + (o << case["shift"])).clamp(-2 ** 31, 2 ** 31 - 1)
        return out.copy_(o)
    g, u = _product(codes, a, st["gate"], None), _product(codes, a, st["up"], None)
    if case["act"] == "silu":
        gv = g << st["sa"]
        top = 16 << 14
        at = gv.abs().clamp(max=top - 1)
        lo, hi = st["sigmoid"][at >> 6], st["sigmoid"][(at >> 6) + 1]
        sig = torch.where(gv.abs() >= top, torch.full_like(gv, 2 ** 24), lo + (((hi - lo) * (at & 63)) >> 6))
        sig = torch.where(gv < 0, 2 ** 24 - sig, sig)
        f = _rne(gv * sig, torch.tensor(18, device="cuda"))
    else:
        f = st["act"][g + 32768]
    return out.copy_(_rne(f * u, torch.tensor(st["sc"], device="cuda")).clamp(-32768, 32767))


def run(state):
    if not own:
        return _run_plain(state)
    from cormorant_amd import linear8
    if state["case"]["kind"] == "gated":
        return linear8.gated8(state["x"], state["weight"], state["out"])
    if state["case"]["residual"]:
        return linear8.linear8(state["x"], state["weight"], state["out"], residual=state["h"],
                               shift=state["case"]["shift"])
    return linear8.linear8(state["x"], state["weight"], state["out"])


# ------------------------------------------------------------------ the definitions, once more
def _nearest_even(x, half_steps):
    """The whole number next to x / (2 half_steps), ties to the even one, from the quotient and remainder."""
    q = torch.div(x, 2 * half_steps, rounding_mode="floor")
    r = x - q * 2 * half_steps
    odd = torch.remainder(q, 2)
    return q + torch.where(r == half_steps, odd, (r > half_steps).long())


def _exact_product(x, top, w, M, s, b):
    """Columns of the product: the codes from the ratio a_t / 127's reciprocal in float64 (every value a
    whole number below 2^53), the sum over k in pieces."""
    recip = torch.floor((127.0 * 2.0 ** 24 + torch.floor(top / 2.0)) / top.clamp(min=1.0)) * (top > 0)
    acc = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    for k0 in range(0, x.shape[1], 2048):
        c = torch.floor((x[:, k0:k0 + 2048] * recip + 2.0 ** 23) / 2.0 ** 24)
        acc += c @ w[k0:k0 + 2048].double()
    whole = (acc * top).long() * M[None, :]                    # below 2^62
    if b is not None:
        whole = whole + b.long()[None, :] * (2 ** s)[None, :]
    return _nearest_even(whole, (2 ** (s - 1))[None, :]).clamp(-32768, 32767)


def exact(case, seed):
    d = _logical(case, seed)
    x = d["x"].double()
    top = torch.maximum(x.amax(1, keepdim=True), -x.amin(1, keepdim=True))
    m = case["m"]
    out = torch.zeros(case["n"], m, dtype=torch.int32 if case.get("residual") else torch.int16, device="cuda")
    step = max(64, (1 << 26) // case["n"])
    for j in range(0, m, step):
        cut = lambda weight: [t[..., j:j + step] for t in weight[:3]]      # noqa: E731
        if case["kind"] == "linear":
            o = _exact_product(x, top, *cut(d["w"]), None if d["b"] is None else d["b"][j:j + step])
            if case["residual"]:
                o = (d["h"][:, j:j + step].long() + o * 2 ** case["shift"]).clamp(-2 ** 31, 2 ** 31 - 1)
        else:
            g, u = _exact_product(x, top, *cut(d["gate"]), None), _exact_product(x, top, *cut(d["up"]), None)
            o = _nearest_even(_exact_act(case["act"], g, d["sa"]) * u, torch.tensor(2 ** (d["sc"] - 1), device="cuda"))
            o = o.clamp(-32768, 32767)
        out[:, j:j + step] = o.to(out.dtype)
    return out


def _exact_act(act, g, sa):
    v = g.double()
    if act != "silu":
        v = v / 256.0
        inner = 0.7071067811865476 * v if act == "gelu" else 0.7978845608028654 * (v + 0.044715 * v ** 3)
        gate = torch.erf(inner) if act == "gelu" else torch.tanh(inner)
        return torch.round(128.0 * v * (1.0 + gate)).clamp(-32768, 32767).long()
    v = v * 2.0 ** sa                                          # at 2^-14
    piece = torch.floor(v.abs().clamp(max=2.0 ** 18 - 1) / 64.0)
    ends = [torch.round(2.0 ** 24 / (1.0 + torch.exp(-(piece + e) / 256.0))) for e in (0.0, 1.0)]
    sig = ends[0] + torch.floor((ends[1] - ends[0]) * (v.abs().clamp(max=2.0 ** 18 - 1) - 64.0 * piece) / 64.0)
    sig = torch.where(v.abs() >= 2.0 ** 18, 2.0 ** 24, sig)
    sig = torch.where(v < 0, 2.0 ** 24 - sig, sig)
    return torch.round(v * sig / 2.0 ** 18).long()             # v sig: 15 bits and a power of two by 25: exact
