"""CPU restatements of the paged cache's operators, on logical rows in 64-bit integers.  TEST
INFRASTRUCTURE ONLY (the checker, never the thing measured or shipped).  Nothing here imports the
product.

A batch is described by q_start [B + 1], kv_len [B] and table [B][max_pages]; a pool by its bytes in
the layout that include/cormorant_hip.h gives for cm_paged_cache (``Pool`` writes and reads it one row
at a time)."""
import numpy as np

from oracle import sim_ref
from oracle.attn_prep import ROPE_BITS, rne_shr_vec, sat16


def smx_tab():
    return np.rint(65536.0 * np.exp2(-np.arange(4096) / 4096.0)).astype(np.int64)


def wrap32(x):
    return ((np.asarray(x, np.int64) + 2 ** 31) & (2 ** 32 - 1)) - 2 ** 31


class Pool:
    """The pool's bytes [pages][kv][block] and its rows."""

    def __init__(self, pages, page, kv, hd, int8, data=None):
        self.pages, self.page, self.kv, self.hd, self.int8 = pages, page, kv, hd, int8
        self.block = page * (2 * hd + 6 if int8 else 4 * hd + 4)
        self.data = np.zeros((pages, kv, self.block), np.uint8) if data is None else \
            np.array(data, np.uint8).reshape(pages, kv, self.block)

    def write(self, pid, slot, g, k, v):
        page, hd, b = self.page, self.hd, self.data[pid, g]
        n = page * hd
        if self.int8:
            (k8, ke), (v8, ve) = quantise(k), quantise(v)
            b[slot * hd:(slot + 1) * hd] = (k8 & 255).astype(np.uint8)
            b[n + slot:2 * n:page] = (v8 & 255).astype(np.uint8)
            at, term = 2 * n, 128 * int(k8.sum())
            b[at + 4 * page + slot], b[at + 5 * page + slot] = ke, ve
        else:
            b[slot * hd:(slot + 1) * hd] = ((k >> 8) & 255).astype(np.uint8)
            b[n + slot * hd:n + (slot + 1) * hd] = ((k & 255) ^ 128).astype(np.uint8)
            b[2 * n + slot:3 * n:page] = ((v >> 8) & 255).astype(np.uint8)
            b[3 * n + slot:4 * n:page] = ((v & 255) ^ 128).astype(np.uint8)
            at, term = 4 * n, 128 * int(k.sum()) - 16384 * hd
        b[at + 4 * slot:at + 4 * slot + 4] = np.frombuffer(np.int32(term).tobytes(), np.uint8)

    def read(self, pid, slot, g):
        page, hd, b = self.page, self.hd, self.data[pid, g]
        n = page * hd
        s8 = lambda x: x.astype(np.int8).astype(np.int64)       # noqa: E731
        if self.int8:
            at = 2 * n
            return (s8(b[slot * hd:(slot + 1) * hd]) << int(b[at + 4 * page + slot]),
                    s8(b[n + slot:2 * n:page]) << int(b[at + 5 * page + slot]))
        return (s8(b[slot * hd:(slot + 1) * hd]) * 256 + s8(b[n + slot * hd:n + (slot + 1) * hd]) + 128,
                s8(b[2 * n + slot:3 * n:page]) * 256 + s8(b[3 * n + slot:4 * n:page]) + 128)


def quantise(x):
    """An int16 row as (codes, shift): shift = max(0, bits of the row's extent - 7), codes rounded half
    to even, at most 127."""
    x = np.asarray(x, np.int64)
    m = int(np.where(x >= 0, x, -1 - x).max())
    e = max(0, m.bit_length() - 7)
    return np.minimum(rne_shr_vec(x, e), 127), e


def norm_rms(x, G, Bq, sc, eps):
    """The row-ops RMSNorm of int16 rows [..][n] with parameter entries [n]."""
    x = np.asarray(x, np.int64)
    out = np.zeros_like(x)
    for i in np.ndindex(*x.shape[:-1]):
        Rm, sh = sim_ref._rsqrt(max(1, int((x[i] * x[i]).sum()) + int(eps)))
        out[i] = sat16(rne_shr_vec(((x[i] * Rm) >> (sh - 24)) * G + Bq, sc))
    return out


def rope(x, row, rotary, interleaved, sa, sb, sc):
    """The row-ops ROPE rule on int16 rows [heads][hd] with the table row (cos [rotary], sin [rotary])."""
    x, row = np.asarray(x, np.int64), np.asarray(row, np.int64)
    hd, h = x.shape[-1], rotary // 2
    co, si = np.full(hd, 1 << ROPE_BITS, np.int64), np.zeros(hd, np.int64)
    co[:rotary], si[:rotary] = row[:rotary], row[rotary:]
    rot = np.zeros_like(x)
    if interleaved:
        rot[:, 0:rotary:2], rot[:, 1:rotary:2] = -x[:, 1:rotary:2], x[:, 0:rotary:2]
    else:
        rot[:, :h], rot[:, h:rotary] = -x[:, h:rotary], x[:, :h]
    return sat16(rne_shr_vec(((x * co) << sa) + ((rot * si) << sb), sc))


def tokens(q_start, kv_len):
    """(token, sequence, position) of every packed token."""
    for b in range(len(kv_len)):
        n = int(q_start[b + 1]) - int(q_start[b])
        for i in range(n):
            yield int(q_start[b]) + i, b, max(int(kv_len[b]), 0) - n + i


def place(pool, table, b, p):
    """(page id, slot) of a position, None where it has none."""
    if p < 0 or p >= table.shape[1] * pool.page:
        return None
    pid = int(table[b][p // pool.page])
    return (pid, p % pool.page) if 0 <= pid < pool.pages else None


def attend(pool, q_start, kv_len, table, q, heads, cm, cfg, window=0, out=None):
    """int16-ranged o [tokens][heads hd] (rows of no sequence from ``out``, else 0)."""
    hd, kv, tab = pool.hd, pool.kv, smx_tab()
    G, cs, fp = heads // kv, cfg & 63, (cfg >> 8) & 31
    q = np.asarray(q, np.int64).reshape(-1, heads, hd)
    o = np.zeros_like(q) if out is None else np.asarray(out, np.int64).reshape(q.shape).copy()
    rows = {}
    for t, b, p in tokens(q_start, kv_len):
        at = [place(pool, table, b, j) for j in range(max(0, p - window + 1) if window else 0, p + 1)]
        at = [x for x in at if x is not None]
        for g in range(kv):
            if not at:
                o[t, g * G:(g + 1) * G] = 0
                continue
            for x in at:
                if x + (g,) not in rows:
                    rows[x + (g,)] = pool.read(*x, g)
            K = np.stack([rows[x + (g,)][0] for x in at])
            V = np.stack([rows[x + (g,)][1] for x in at])
            for h in range(g * G, (g + 1) * G):
                s = sat16(wrap32(K @ q[t, h]) >> 8)
                y = ((s.max() - s) * cm) >> cs
                w = np.minimum(tab[y & 4095] >> np.minimum(y >> 12, 40), 65535)
                S, A = int(w.sum()), w @ V
                num, den = (2 * (A << (fp - 8)) + S, 2 * S) if fp >= 8 else (2 * A + (S << (8 - fp)), S << (9 - fp))
                o[t, h] = sat16(num // den)
    return o.reshape(-1, heads * hd)


def prep(pool, q_start, kv_len, table, q, k, v, qr, rope_rows, rotary, interleaved, rope_q, rope_k, norm_q=None,
         norm_k=None, eps_q=0, eps_k=0):
    """Writes qr [tokens][heads hd] and the pool in place.  rope_q / rope_k: (sa, sb, sc) arrays
    broadcast over [heads][hd]; norm_q / norm_k: (G, Bq, sc) over [hd], or None."""
    hd, kv = pool.hd, pool.kv
    for t, b, p in tokens(q_start, kv_len):
        row = rope_rows[min(max(p, 0), len(rope_rows) - 1)]
        xq, xk = np.asarray(q[t], np.int64).reshape(-1, hd), np.asarray(k[t], np.int64).reshape(-1, hd)
        xv = np.asarray(v[t], np.int64).reshape(-1, hd)
        if norm_q is not None:
            xq = norm_rms(xq, *norm_q, eps_q)
        if norm_k is not None:
            xk = norm_rms(xk, *norm_k, eps_k)
        qr[t] = rope(xq, row, rotary, interleaved, *rope_q).reshape(-1)
        xk = rope(xk, row, rotary, interleaved, *rope_k)
        at = place(pool, table, b, p)
        if at is not None:
            for g in range(kv):
                pool.write(*at, g, xk[g], xv[g])


def read(pool, q_start, kv_len, table, k, v):
    """Writes k, v [tokens][kv hd] in place."""
    for t, b, p in tokens(q_start, kv_len):
        at = place(pool, table, b, p)
        for g in range(pool.kv):
            x = pool.read(*at, g) if at is not None else (0, 0)
            k[t].reshape(pool.kv, pool.hd)[g], v[t].reshape(pool.kv, pool.hd)[g] = x
