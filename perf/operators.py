"""The paged-cache operators: their measured cases, their plain forms and their definitions.

A served decoder keeps the K and V rows of many sequences of different lengths in pages.  Three
operators work on such a cache, in the framework's raw fixed-point lanes:

  attend   the attention of a batch of new tokens (a prompt, a chunk of one, or one token a
           sequence) over its sequences' pages
  prep     what comes before it: q and k normalised per head (optional) and rotated at each token's
           position, k's and v's rows written into the pages (int16, or int8 with a shift a row)
  read     cache rows back out of the pages as int16 rows

Every output is a whole number that the operators' integer definitions give bit for bit.

``own`` False: ``run`` is the plain form, elementary torch operations (float64 products, exact for
these operands, and int64).  ``own`` True: ``run`` is the call a program makes of the framework.
Both take the state that ``prepare`` makes: the pool of pages, the page table, and the raw rows.

A page of one KV head (``page`` keys, head dimension ``hd``) is stored as the matrix units read it:
  int16: K's high bytes [page][hd], K's low bytes, V's high bytes [hd][page], V's low bytes, and per
         key the int32 128 sum(K) - 16384 hd; a low byte is stored as (byte ^ 0x80);
  int8:  K [page][hd], V [hd][page], per key the int32 128 sum(K), and the bytes of K's and V's shifts.
"""
import math

import torch

own = False

THETA = 100000.0
ROPE_BITS = 23
Q_EXP, K_EXP, V_EXP, P_EXP = 9, 9, 11, 14       # raw = value 2^exp; scores at 2^-(9 + 9 - 8)
STD = 0.6                                       # of a projection's values
NORM_EPS = 1e-5


def _text(sizes):
    """Whole numbers as one text (a case holds plain values): the sequences' lengths."""
    return " ".join(str(n) for n in sizes)


def _ints(text):
    return [int(x) for x in text.split()]


def listed():
    S = dict(heads=15, kv=5, hd=64, page=16, int8=False)          # the decoder configuration's head layout
    server = [8192, 301, 5003, 1024, 777, 2500, 640, 4096, 333, 7001, 1200, 900, 410, 6144, 1801, 512, 2999, 350, 1500,
              3700, 1025, 480, 7777, 2048]
    wide = dict(heads=32, kv=8, hd=128, page=64, int8=True)

    def case(name, kind, shape, lens, new, **more):
        return dict(shape, name=name, kind=kind, lens=_text(lens), new=_text(new), **more)
    packed = [1, 517, 130, 2305, 77, 1999, 641], [1, 517, 1, 301, 77, 65, 641]
    return [
        # one token of one short sequence: launch latency alone
        case("attend_decode_b1_c200", "attend", S, [200], [1], window=0),
        # the decoder configuration's step: 16 sequences, 1024 cache rows each
        case("attend_decode_b16_c1024", "attend", S, [1024] * 16, [1] * 16, window=0),
        # a busy server's step: 24 sequences from a few hundred to 8192 rows, int8 cache, wide heads
        case("attend_decode_b24_ragged_int8", "attend", wide, server, [1] * 24, window=0),
        # a chunk of a long prompt over the part that is cached already
        case("attend_chunk_t256_c4096", "attend", S, [4096], [256], window=0),
        # a mixed step: whole prompts, chunks and single tokens of odd lengths packed together
        case("attend_packed_ragged", "attend", S, *packed, window=0),
        # a sliding window over an int8 cache
        case("attend_chunk_window_int8", "attend", dict(heads=16, kv=4, hd=128, page=32, int8=True), [3001, 1100],
             [500, 333], window=1024),
        # a whole long prompt
        case("attend_prompt_t4096", "attend", S, [4096], [4096], window=0),
        # the decode step's rows of the same configuration into the cache
        case("prep_decode_b16", "prep", S, [1024] * 16, [1] * 16, norm=False, rotary=64, interleaved=False),
        # a packed step of odd lengths into an int8 cache, half of each head rotated in pairs
        case("prep_packed_norm_int8", "prep", dict(heads=12, kv=4, hd=128, page=32, int8=True), *packed, norm=True,
             rotary=64, interleaved=True),
        # a whole long prompt, q and k normalised per head
        case("prep_prompt_t8192_norm", "prep", S, [8192], [8192], norm=True, rotary=64, interleaved=False),
        # one short sequence swapped out
        case("read_b1_c200", "read", S, [200], [200]),
        # a server's int8 cache handed to a contiguous one
        case("read_b12_ragged_int8", "read", wide, server[:12], server[:12]),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 4e14


def draw(rng):
    limit = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("attend", "prep", "read")}
    while True:
        kind = rng.choice(["attend", "attend", "attend", "prep", "prep", "read"])
        kv = rng.choice([1, 2, 4, 5, 8])
        case = dict(kind=kind, kv=kv, heads=kv * rng.choice([1, 2, 3, 4, 7, 8]), hd=rng.choice([64, 64, 128]),
                    page=rng.choice([16, 32, 64, 128]), int8=rng.random() < 0.5)
        batch = _log(rng, 1, 40)
        lens = [_log(rng, 1, 8192) for _ in range(batch)]
        form = rng.choice(["decode", "chunk", "prompt", "mixed"])
        if kind == "read":
            form = rng.choice(["chunk", "prompt"])
        new = []
        for n in lens:
            f = rng.choice(["decode", "chunk", "prompt"]) if form == "mixed" else form
            new.append(1 if f == "decode" else n if f == "prompt" else rng.randint(1, n))
        case.update(lens=_text(lens), new=_text(new))
        if kind == "attend":
            case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        if kind == "prep":
            case.update(norm=rng.random() < 0.5, rotary=rng.choice([case["hd"], case["hd"] // 2, case["hd"] // 4]),
                        interleaved=rng.random() < 0.5)
        if _cost(case) <= limit[kind]:
            return case


# ------------------------------------------------------------------ what a pass cannot do without
def _keys(case):
    """Sum over the new tokens of the keys they attend to, and the cache rows read at least once."""
    pairs = rows = 0
    for n, t in zip(_ints(case["lens"]), _ints(case["new"])):
        w = case["window"] or n
        first = n - t
        pairs += sum(min(p + 1, w) for p in range(first, n))
        rows += min(n, t - 1 + w)
    return pairs, rows


def _row_bytes(case):
    """Bytes of one key and KV head in the cache, K and V."""
    hd = case["hd"]
    return 2 * hd + 6 if case["int8"] else 4 * hd + 4


def work(case):
    T, H, KV, hd = sum(_ints(case["new"])), case["heads"], case["kv"], case["hd"]
    if case["kind"] == "attend":
        pairs, rows = _keys(case)
        return {"bytes": 4 * T * H * hd + rows * KV * _row_bytes(case), "flops": 4 * pairs * H * hd}
    cache = T * KV * _row_bytes(case)
    if case["kind"] == "prep":
        rope = 8 * case["rotary"] * T
        return {"bytes": 4 * T * H * hd + 4 * T * KV * hd + rope + cache, "flops": T * (H + KV) * hd * 8}
    return {"bytes": cache + 4 * T * KV * hd, "flops": 0}


# ------------------------------------------------------------------ inputs
def _rows(gen, n, cols, exp, std=STD):
    x = torch.randn(n, cols, generator=gen, device="cuda", dtype=torch.float32) * (std * 2.0 ** exp)
    return x.round_().clamp_(-32768, 32767).to(torch.int16)


def _logical(case, seed):
    """The raw rows of a case from its seed: the cached rows of every sequence (packed), the new
    tokens' projections, the page table."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    total, T = sum(_ints(case["lens"])), sum(_ints(case["new"]))
    d = {"q": _rows(gen, T, H * hd, Q_EXP)}
    # heads whose rows differ in size by powers of two, as a model's do (and their int8 shifts with them)
    spread = torch.pow(2.0, torch.randint(-1, 2, (KV,), generator=gen, device="cuda").float()).repeat_interleave(hd)
    cached = lambda exp: (_rows(gen, total, KV * hd, exp).float() * spread).round().clamp(-32768, 32767).to(torch.int16)  # noqa: E731
    if case["kind"] == "prep":
        d["k"], d["v"] = _rows(gen, T, KV * hd, K_EXP), _rows(gen, T, KV * hd, V_EXP)
    else:
        d["K"], d["V"] = cached(K_EXP), cached(V_EXP)
    width = max(-(-n // case["page"]) for n in _ints(case["lens"])) + 1
    used = [-(-n // case["page"]) for n in _ints(case["lens"])]
    pages = sum(used) + 3
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(used), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        at += u
    d["table"], d["pages"] = table, pages
    return d


def _rope_rows(case, rows):
    """int32 [rows][2 rotary]: cos then sin at 2^-23 of each rotated column's angle."""
    rd = case["rotary"]
    inv = THETA ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    ang = ang.repeat_interleave(2, 1) if case["interleaved"] else torch.cat([ang, ang], 1)
    return torch.cat([torch.cos(ang), torch.sin(ang)], 1).mul_(2.0 ** ROPE_BITS).round_().to(torch.int32)


def _norm_params(case, seed):
    """Per-head RMSNorm of rows at 2^-Q_EXP into rows at 2^-Q_EXP: gammas, their fixed-point image
    (G at 2^-g with sqrt(hd) folded in, the shift 24 + g - 9 + 9) and eps at the rows' scale."""
    hd = case["hd"]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 77)
    gamma = 0.6 + 0.02 * torch.randn(2, hd, generator=gen, device="cuda", dtype=torch.float64)
    g = 20
    G = (gamma * math.sqrt(hd) * 2.0 ** g).round_().to(torch.int64)
    return G, 24 + g - Q_EXP, int(round(NORM_EPS * hd * 2.0 ** (2 * Q_EXP)))


def _block(case):
    return case["page"] * _row_bytes(case)


def _views(case, pool):
    """The pool's sections: K / V byte planes, the key terms and the shifts, all [pages][kv][...]."""
    page, hd = case["page"], case["hd"]
    blk = pool.view(-1, case["kv"], _block(case))
    n = page * hd
    at = lambda i: blk[..., i * n:(i + 1) * n].view(torch.int8)      # noqa: E731
    kshape, vshape = blk.shape[:2] + (page, hd), blk.shape[:2] + (hd, page)
    if case["int8"]:
        return {"k": at(0).unflatten(-1, kshape[2:]), "v": at(1).unflatten(-1, vshape[2:]),
                "t": blk[..., 2 * n:2 * n + 4 * page].view(torch.int32), "ke": blk[..., 2 * n + 4 * page:2 * n + 5 * page],
                "ve": blk[..., 2 * n + 5 * page:2 * n + 6 * page]}
    return {"kh": at(0).unflatten(-1, kshape[2:]), "kl": at(1).unflatten(-1, kshape[2:]),
            "vh": at(2).unflatten(-1, vshape[2:]), "vl": at(3).unflatten(-1, vshape[2:]),
            "t": blk[..., 4 * n:4 * n + 4 * page].view(torch.int32)}


def _rne(x, e):
    """Round half to even of x / 2^e (e a tensor of shifts >= 0)."""
    one = torch.ones_like(x)
    half = torch.where(e > 0, one << (e - 1).clamp(min=0), torch.zeros_like(x))
    q = (x + half) >> e
    tie = (e > 0) & ((x & ((one << e) - 1)) == half)
    return torch.where(tie & (q & 1 == 1), q - 1, q)


def _bits(m):
    n = torch.zeros_like(m)
    for k in range(16):
        n += (m >> k > 0).to(n.dtype)
    return n


def _quantise(x):
    """int rows [...][hd] -> (8-bit codes, shifts [...])."""
    e = (_bits(torch.where(x >= 0, x, -1 - x).amax(-1)) - 7).clamp(min=0)
    return _rne(x, e[..., None].expand_as(x)).clamp(max=127), e


def _write(case, pool, page_id, slot, k, v):
    """Rows k, v (int64 [n][kv][hd]) into slots of pages."""
    w = _views(case, pool)
    if case["int8"]:
        (kc, ke), (vc, ve) = _quantise(k), _quantise(v)
        w["k"][page_id, :, slot] = kc.to(torch.int8)
        w["v"][page_id, :, :, slot] = vc.to(torch.int8)
        w["ke"][page_id, :, slot] = ke.to(torch.uint8)
        w["ve"][page_id, :, slot] = ve.to(torch.uint8)
        w["t"][page_id, :, slot] = (128 * kc.sum(-1)).to(torch.int32)
    else:
        low = lambda x: ((x & 255) - 128).to(torch.int8)         # noqa: E731
        w["kh"][page_id, :, slot], w["kl"][page_id, :, slot] = (k >> 8).to(torch.int8), low(k)
        w["vh"][page_id, :, :, slot], w["vl"][page_id, :, :, slot] = (v >> 8).to(torch.int8), low(v)
        w["t"][page_id, :, slot] = (128 * k.sum(-1) - 16384 * case["hd"]).to(torch.int32)


def _softmax_regs(hd):
    """(Cm, Cs): log2(e) / sqrt(hd) 2^-(score exponent) 2^12 = Cm 2^-Cs, Cm of 24 bits."""
    c = math.log2(math.e) / math.sqrt(hd) * 2.0 ** -(Q_EXP + K_EXP - 8) * 4096.0
    cs = 23 - math.floor(math.log2(c))
    return int(round(c * 2.0 ** cs)), cs


def prepare(case, seed):
    L = _logical(case, seed)
    KV, hd, page = case["kv"], case["hd"], case["page"]
    lens, new = _ints(case["lens"]), _ints(case["new"])
    dev = "cuda"
    pool = torch.zeros(L["pages"] * KV * _block(case), dtype=torch.uint8, device=dev)
    if case["kind"] != "prep":
        seq = torch.repeat_interleave(torch.arange(len(lens), device=dev), torch.tensor(lens, device=dev))
        pos = torch.cat([torch.arange(n, device=dev) for n in lens])
        for a in range(0, seq.numel(), 8192):              # in parts: the conversions are of int64 rows
            s, p = seq[a:a + 8192], pos[a:a + 8192]
            k, v = (L[x][a:a + 8192].long().view(-1, KV, hd) for x in ("K", "V"))
            _write(case, pool, L["table"][s, p // page].long(), p % page, k, v)
    q_start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
    st = {"case": case, "pool": pool, "table": L["table"], "q_start": q_start,
          "kv_len": torch.tensor(lens, dtype=torch.int32, device=dev)}
    T = sum(new)
    if case["kind"] == "prep":
        st.update(q=L["q"], k=L["k"], v=L["v"], qr=torch.zeros_like(L["q"]), rope=_rope_rows(case, max(lens)))
        if case["norm"]:
            st["G"], st["norm_shift"], st["eps"] = _norm_params(case, seed)
    elif case["kind"] == "attend":
        st.update(q=L["q"], o=torch.zeros_like(L["q"]))
        st["cm"], cs = _softmax_regs(hd)
        st["cfg"] = cs | (P_EXP << 8)
    else:
        st.update(k_out=torch.zeros(T, KV * hd, dtype=torch.int16, device=dev),
                  v_out=torch.zeros(T, KV * hd, dtype=torch.int16, device=dev))
    if own:
        from cormorant_amd import paged
        from cormorant_amd.rowops_nodes import param_block
        st["cache"] = paged.PagedCache(L["pages"], page, KV, hd, int8=case["int8"], data=pool)
        st["batch"] = paged.PagedBatch(st["q_start"], st["kv_len"], st["table"], T)
        if case["kind"] == "prep":
            prm = lambda *a: torch.from_numpy(param_block(*a)).to(dev)     # noqa: E731
            rope = dict(table=st["rope"], interleaved=case["interleaved"], params_q=prm(0, 0, 0, 0, ROPE_BITS),
                        params_k=prm(0, 0, 0, 0, ROPE_BITS))
            if case["norm"]:
                G = st["G"].cpu().numpy()
                rope.update(norm_q=prm(G[0], 0, 0, 0, st["norm_shift"]), norm_k=prm(G[1], 0, 0, 0, st["norm_shift"]),
                            eps_q=st["eps"], eps_k=st["eps"])
            st["prep"] = paged.PagedPrep(**rope)
    return st


# ------------------------------------------------------------------ plain forms
def _tab():
    k = torch.arange(4096, device="cuda", dtype=torch.float64)
    return torch.exp2(-k / 4096.0).mul_(65536.0).round_().to(torch.int64)


def _gather(case, pool, table_row, n):
    """The K and V rows 0 .. n - 1 of a sequence from its pages: int16-ranged int32 [kv][n][hd]."""
    w = _views(case, pool)
    ids = table_row[:-(-n // case["page"])].long()
    rows = lambda x: x[ids].to(torch.int32).permute(1, 0, 2, 3).flatten(1, 2)[:, :n]               # noqa: E731
    cols = lambda x: x[ids].to(torch.int32).permute(1, 0, 3, 2).flatten(1, 2)[:, :n]               # noqa: E731
    if case["int8"]:
        flat = lambda e: e[ids].to(torch.int32).permute(1, 0, 2).flatten(1)[:, :n, None]           # noqa: E731
        return rows(w["k"]) << flat(w["ke"]), cols(w["v"]) << flat(w["ve"])
    return rows(w["kh"]) * 256 + rows(w["kl"]) + 128, cols(w["vh"]) * 256 + cols(w["vl"]) + 128


def _sat16(x):
    return x.clamp(-32768, 32767)


def _wrap32(x):
    return ((x + 2 ** 31) & (2 ** 32 - 1)) - 2 ** 31


def _attend_plain(st):
    case = st["case"]
    H, KV, hd, G = case["heads"], case["kv"], case["hd"], case["heads"] // case["kv"]
    cm, cs, fp = st["cm"], st["cfg"] & 63, st["cfg"] >> 8
    tab = _tab()
    o = torch.zeros_like(st["q"])
    at = 0
    for b, (n, t) in enumerate(zip(_ints(case["lens"]), _ints(case["new"]))):
        K, V = _gather(case, st["pool"], st["table"][b], n)
        q = st["q"][at:at + t].view(t, KV, G, hd)
        j = torch.arange(n, device="cuda")
        step = max(1, (1 << 25) // (n * G))                 # rows at a time: the scores are 64-bit matrices
        for r0 in range(0, t, step):
            r1 = min(t, r0 + step)
            p = torch.arange(n - t + r0, n - t + r1, device="cuda").repeat_interleave(G)[:, None]
            seen = j[None, :] <= p
            if case["window"]:
                seen &= j[None, :] > p - case["window"]
            for g in range(KV):
                rows = q[r0:r1, g].reshape(-1, hd).double()
                s = _sat16(_wrap32((rows @ K[g].double().T).long()) >> 8)
                m = torch.where(seen, s, -32768).amax(1, keepdim=True)
                y = ((m - s).clamp(min=0) * cm) >> cs
                w = (tab[y & 4095] >> (y >> 12).clamp(max=40)).clamp(max=65535) * seen
                S = w.sum(1, keepdim=True)
                A = (w.double() @ V[g].double()).long()
                out = torch.div(2 * (A << (fp - 8)) + S, 2 * S, rounding_mode="floor")
                o[at + r0:at + r1].view(-1, KV, G, hd)[:, g] = _sat16(out).to(torch.int16).view(r1 - r0, G, hd)
        at += t
    return o


def _mul_hi32(a, b):
    """floor(a b / 2^32) of factors below 2^32, in int64."""
    return ((a >> 16) * b + (((a & 65535) * b) >> 16)) >> 16


def _rsqrt(D):
    """(Rm, shift): 1 / sqrt(D) ~ Rm 2^-shift, Rm of 32 bits, by one Newton step from a table."""
    e = torch.zeros_like(D)
    for k in range(62):
        e += (D >> k > 0).to(e.dtype)
    d = e - 32
    d = d + (d & 1)
    Dm = torch.where(d >= 0, D >> d.clamp(min=0), D << (-d).clamp(min=0))
    y0 = torch.round(2.0 ** 47 / torch.sqrt(((Dm >> 19).double() + 0.5) * 524288.0)).long().clamp(max=2 ** 32 - 1)
    u = _mul_hi32(_mul_hi32(Dm, y0), y0)
    r = (1 << 30) - u                                        # |r| < 2^30
    step = ((y0 >> 16) * r * 2 + (((y0 & 65535) * r) >> 15)) >> 16
    return (y0 + step).clamp(2 ** 31, 2 ** 32 - 1), 47 + (d >> 1)


def _norm_plain(x, G, shift, eps):
    """The row-ops RMSNorm of int64 rows [...][hd] into int16-ranged rows."""
    D = (x * x).sum(-1) + eps
    Rm, sh = _rsqrt(D.clamp(min=1))
    P1 = (x * Rm[..., None]) >> (sh - 24)[..., None]
    return _sat16(_rne(P1 * G, torch.full_like(P1, shift)))


def _rope_plain(case, x, cs):
    """x int64 [n][heads][hd] at the table rows cs [n][2 rotary]."""
    rd = case["rotary"]
    a = x[..., :rd]
    if case["interleaved"]:
        rot = torch.stack([-a[..., 1::2], a[..., 0::2]], -1).flatten(-2)
    else:
        rot = torch.cat([-a[..., rd // 2:], a[..., :rd // 2]], -1)
    num = a * cs[:, None, :rd] + rot * cs[:, None, rd:]
    z = _sat16(_rne(num, torch.full_like(num, ROPE_BITS)))
    return torch.cat([z, x[..., rd:]], -1)


def _prep_plain(st):
    case = st["case"]
    H, KV, hd, page = case["heads"], case["kv"], case["hd"], case["page"]
    new = torch.diff(st["q_start"]).long()
    seq = torch.repeat_interleave(torch.arange(len(_ints(case["new"])), device="cuda"), new)
    pos = st["kv_len"].long()[seq] - new[seq] + torch.arange(seq.numel(), device="cuda") - st["q_start"].long()[seq]
    q, k, v = (st[x].long().view(seq.numel(), -1, hd) for x in "qkv")
    if case["norm"]:
        q = _norm_plain(q, st["G"][0], st["norm_shift"], st["eps"])
        k = _norm_plain(k, st["G"][1], st["norm_shift"], st["eps"])
    cs = st["rope"][pos].long()
    st["qr"].copy_(_rope_plain(case, q, cs).view(-1, H * hd).to(torch.int16))
    _write(case, st["pool"], st["table"][seq, pos // page].long(), pos % page, _rope_plain(case, k, cs), v)
    return [st["qr"], st["pool"]]


def _read_plain(st):
    case = st["case"]
    at = 0
    for b, (n, t) in enumerate(zip(_ints(case["lens"]), _ints(case["new"]))):
        K, V = _gather(case, st["pool"], st["table"][b], n)
        for x, out in ((K, st["k_out"]), (V, st["v_out"])):
            out[at:at + t] = x[:, n - t:].transpose(0, 1).reshape(t, -1).to(torch.int16)
        at += t
    return [st["k_out"], st["v_out"]]


def run(state):
    st = state
    kind = st["case"]["kind"]
    if own:
        from cormorant_amd import paged
        if kind == "attend":
            return paged.paged_attention(st["cache"], st["batch"], st["q"], st["o"], st["case"]["heads"], st["cm"],
                                         st["cfg"], window=st["case"]["window"])
        if kind == "prep":
            paged.paged_prep(st["cache"], st["batch"], st["prep"], st["q"], st["k"], st["v"], st["qr"])
            return [st["qr"], st["pool"]]
        paged.paged_read(st["cache"], st["batch"], st["k_out"], st["v_out"])
        return [st["k_out"], st["v_out"]]
    return {"attend": _attend_plain, "prep": _prep_plain, "read": _read_plain}[kind](st)


# ------------------------------------------------------------------ the definitions, once more
def _held(case, x):
    """What the cache holds of int64 rows [n][kv][hd]: themselves, or their 8-bit values."""
    if not case["int8"]:
        return x
    top = torch.maximum(x.amax(-1, keepdim=True), -1 - x.amin(-1, keepdim=True))
    step = torch.ones_like(top)
    while bool((top >= 128 * step).any()):
        step = torch.where(top >= 128 * step, 2 * step, step)
    return torch.round(x.double() / step.double()).clamp(max=127).long() * step       # rounds ties to even


def _exact_attend(case, seed):
    L = _logical(case, seed)
    H, KV, hd = case["heads"], case["kv"], case["hd"]
    cm, cs = _softmax_regs(hd)
    out = torch.zeros_like(L["q"])
    q0 = k0 = 0
    for n, t in zip(_ints(case["lens"]), _ints(case["new"])):
        K = _held(case, L["K"][k0:k0 + n].long().view(n, KV, hd)).double()
        V = _held(case, L["V"][k0:k0 + n].long().view(n, KV, hd)).double()
        Q = L["q"][q0:q0 + t].view(t, H, hd).double()
        block = max(1, (1 << 24) // n)
        for h in range(H):
            for a in range(0, t, block):
                rows = Q[a:a + block, h]
                dot = rows @ K[:, h * KV // H].T
                dot = dot - torch.floor((dot + 2.0 ** 31) / 2.0 ** 32) * 2.0 ** 32
                s = torch.floor(dot / 256.0).clamp(-32768, 32767)
                last = torch.arange(n - t + a, n - t + a + rows.shape[0], device="cuda")[:, None]
                key = torch.arange(n, device="cuda")[None, :]
                hidden = key > last
                if case["window"]:
                    hidden |= key <= last - case["window"]
                s = s.masked_fill(hidden, -1e9)
                y = torch.floor((s.amax(1, keepdim=True) - s) * float(cm) / 2.0 ** cs)
                octave = torch.floor(y / 4096.0)
                mant = torch.round(65536.0 * torch.exp2(-(y - 4096.0 * octave) / 4096.0))
                w = torch.floor(mant / torch.exp2(octave.clamp(max=60.0))).clamp(max=65535.0).masked_fill(hidden, 0.0)
                num, den = (w @ V[:, h * KV // H]) * 2.0 ** (P_EXP - 8), w.sum(1, keepdim=True)
                out[q0 + a:q0 + a + rows.shape[0], h * hd:(h + 1) * hd] = \
                    _floor_ratio(2.0 * num + den, 2.0 * den).clamp(-32768, 32767).to(torch.int16)
        q0, k0 = q0 + t, k0 + n
    return out


def _floor_ratio(a, b):
    """floor(a / b) of whole numbers in float64 (below 2^63, b dividing into a quotient below 2^24):
    the quotient's estimate put right by the remainder in int64."""
    f = torch.floor(a / b)
    r = a.long() - f.long() * b.long()
    return f + (r >= b.long()).double() - (r < 0).double()


def _exact_prep(case, seed):
    L = _logical(case, seed)
    H, KV, hd, page, rd = case["heads"], case["kv"], case["hd"], case["page"], case["rotary"]
    where = [(b, p) for b, (n, t) in enumerate(zip(_ints(case["lens"]), _ints(case["new"]))) for p in range(n - t, n)]
    seq = torch.tensor([b for b, _ in where], device="cuda")
    pos = torch.tensor([p for _, p in where], device="cuda")
    rope = _rope_rows(case, max(_ints(case["lens"])))[pos].double()
    q, k, v = (L[x].view(len(where), -1, hd).double() for x in "qkv")
    if case["norm"]:
        G, shift, eps = _norm_params(case, seed)

        def norm(x, gain):
            D = (x * x).sum(-1) + float(eps)
            e = torch.frexp(D)[1].long()                       # D in [2^(e-1), 2^e)
            d = e - 32 + (e & 1)
            Dm = torch.floor(D * torch.exp2(-d.double()))
            y = torch.round(2.0 ** 47 / torch.sqrt((torch.floor(Dm / 524288.0) + 0.5) * 524288.0)).clamp(max=2.0 ** 32 - 1)
            y, Dm = y.long(), Dm.long()
            hi = lambda a, b: ((a >> 20) * b + (((a & 0xFFFFF) * b) >> 20)) >> 12      # noqa: E731
            r = (1 << 30) - hi(hi(Dm, y), y)
            y = (y + (((y >> 20) * r + (((y & 0xFFFFF) * r) >> 20)) >> 11)).clamp(2 ** 31, 2 ** 32 - 1)
            p1 = torch.floor((x.long() * y[..., None]).double() * torch.exp2(-(23 + d // 2).double())[..., None])
            return torch.round(p1 * gain.double() / 2.0 ** shift).clamp(-32768, 32767)
        q, k = norm(q, G[0]), norm(k, G[1])

    def turn(x):
        y = x.clone()
        for c in range(rd):
            if case["interleaved"]:
                other, sign = c ^ 1, (-1.0 if c % 2 == 0 else 1.0)
            else:
                other, sign = (c + rd // 2) % rd, (-1.0 if c < rd // 2 else 1.0)
            y[..., c] = torch.round((x[..., c] * rope[:, None, c] + sign * x[..., other] * rope[:, None, rd + c]) / 2.0 ** 23)
        return y.clamp(-32768, 32767)
    qr, k = turn(q).to(torch.int16).view(len(where), H * hd), turn(k).long()
    v = v.long()
    # the pool byte by byte: every page's sections at their offsets
    pool = torch.zeros(L["pages"], KV, _block(case), dtype=torch.uint8, device="cuda")
    pid, slot = L["table"][seq, torch.div(pos, page, rounding_mode="floor")].long(), pos % page
    col = torch.arange(hd, device="cuda")
    head = torch.arange(KV, device="cuda")[None, :, None]
    P, s3 = pid[:, None, None], slot[:, None, None]
    size = page * hd

    def put(at, x):
        pool[P, head, at] = (x & 255).to(torch.uint8)
    k_at, v_at = s3 * hd + col, col * page + s3
    if case["int8"]:
        kv_, vv_ = _held(case, k), _held(case, v)
        shift = lambda x: torch.log2(_step(x)).round().long()           # noqa: E731
        ke, ve = shift(k), shift(v)
        kc, vc = kv_ >> ke, vv_ >> ve
        put(k_at, kc)
        put(size + v_at, vc)
        term, base = 128 * kc.sum(-1, keepdim=True), 2 * size
        put(base + 4 * page + s3, ke)
        put(base + 5 * page + s3, ve)
    else:
        put(k_at, k >> 8)
        put(size + k_at, (k & 255) ^ 128)
        put(2 * size + v_at, v >> 8)
        put(3 * size + v_at, (v & 255) ^ 128)
        term, base = 128 * k.sum(-1, keepdim=True) - 16384 * hd, 4 * size
    for i in range(4):
        put(base + 4 * s3 + i, term >> (8 * i))
    return [qr, pool.view(-1)]


def _step(x):
    """2^shift of the rows' 8-bit form."""
    top = torch.maximum(x.amax(-1, keepdim=True), -1 - x.amin(-1, keepdim=True)).double()
    return torch.exp2(torch.floor(torch.log2(top.clamp(min=1.0))) - 6.0).clamp(min=1.0)


def _exact_read(case, seed):
    L = _logical(case, seed)
    KV, hd = case["kv"], case["hd"]
    rows, at = [], 0
    for n, t in zip(_ints(case["lens"]), _ints(case["new"])):
        rows.append(torch.arange(at + n - t, at + n, device="cuda"))
        at += n
    rows = torch.cat(rows)
    return [_held(case, L[x][rows].long().view(-1, KV, hd)).to(torch.int16).view(-1, KV * hd) for x in ("K", "V")]


def exact(case, seed):
    return {"attend": _exact_attend, "prep": _exact_prep, "read": _exact_read}[case["kind"]](case, seed)
