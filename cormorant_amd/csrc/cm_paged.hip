// cm_paged.hip -- the paged K / V cache: the step's rows into it (cm_paged_prep), the attention over
// it (cm_paged_attention) and its rows back (cm_paged_read).
//
// A page holds K rows as the byte planes that an MFMA operand lane reads 16 bytes of (d contiguous for
// q.K^T) and V transposed (keys contiguous for P.V), so the attention neither splits nor transposes
// what it reads: an int16 x is 256 h + l + 128 (h = x >> 8, l = (x & 255) - 128).
#include <algorithm>
#include <type_traits>

#include "cm_common.h"
#include "cm_rowops_math.h"

namespace cm {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- the cache and the batch on the device
struct Cache {
    uint8_t* data;
    uint64_t block;                        // bytes of a (page, head) block
    uint32_t pages, page, lg, kv;          // page = 1 << lg rows
};

struct Batch {
    const int32_t *q_start, *kv_len, *table;
    uint32_t batch, tokens, max_pages, cap;   // cap = max_pages * page
    uint64_t table_ld;

    __device__ __forceinline__ uint32_t start(uint32_t b) const {
        return (uint32_t)min(max(q_start[b], 0), (int)tokens);
    }
    __device__ __forceinline__ int len(uint32_t b) const { return max(kv_len[b], 0); }
};

// The largest b of [0, n) with f(b) <= x, for an f that does not fall and f(0) <= x: 64 probes a step,
// one load of the wavefront for 64 sequences.  Every lane returns it; the interval shrinks each step.
template <class F>
__device__ __forceinline__ uint32_t find_le(uint32_t n, uint32_t x, F f) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const bool le = i < n && f(lo + i) <= x;
        const uint32_t cnt = max(1u, (uint32_t)__popcll(__ballot(le)));
        const uint32_t at = (cnt - 1) * step;
        lo += at;
        n = min(step, n - at);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

__host__ __device__ inline size_t block_bytes(uint32_t page, uint32_t hd, bool i8) {
    return (size_t)page * (i8 ? 2 * hd + 6 : 4 * hd + 4);
}

// Byte offsets of a block's sections
template <uint32_t HD, bool I8>
struct Block {
    static __device__ __forceinline__ uint32_t k(uint32_t page, uint32_t plane) { return plane * page * HD; }
    static __device__ __forceinline__ uint32_t v(uint32_t page, uint32_t plane) { return ((I8 ? 1 : 2) + plane) * page * HD; }
    static __device__ __forceinline__ uint32_t term(uint32_t page) { return (I8 ? 2 : 4) * page * HD; }
    static __device__ __forceinline__ uint32_t ke(uint32_t page) { return term(page) + 4 * page; }
    static __device__ __forceinline__ uint32_t ve(uint32_t page) { return term(page) + 5 * page; }
};

__device__ __forceinline__ v4i mfma(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int sat16i(int x) { return min(max(x, -32768), 32767); }

// ---------------------------------------------------------------- prep
struct Prep {
    const int16_t *q, *k, *v;
    int16_t* qr;
    uint64_t q_ld, k_ld, v_ld, qr_ld;
    uint32_t heads, rope_rows, rotary, interleaved;
    const int32_t* rope;
    const uint8_t *rope_q, *rope_k, *norm_q, *norm_k;
    uint32_t rope_q_cols, rope_k_cols;
    int64_t eps_q, eps_k;
    const uint8_t* tab;                    // the row-ops table image (rsqrt entries)
};

// rsqrt_bf (cm_rowops_math.h) for D below 2^63; tab: the table image's entries from index 2048 on (Dm >= 2^30)
constexpr uint32_t kRsqrt = 8192 - 2048;
__device__ __forceinline__ void rsqrt64(uint64_t D, uint64_t& Rm, int& sh, const uint32_t* tab) {
    const int e = 64 - __clzll((long long)D);
    int d = e - 32;
    d += d & 1;
    const uint32_t Dm = (uint32_t)(d >= 0 ? D >> d : D << -d);
    const uint32_t y0 = tab[(Dm >> 19) - 2048];
    const int64_t r = ((int64_t)1 << 30) - (int64_t)__umulhi(__umulhi(Dm, y0), y0);     // above -2^32
    // y0 r >> 31 in 64 bits where r is below 2^31 (the unit's own table: below 2^18), else in two halves of y0
    const int64_t step = r >= -((int64_t)1 << 31) ? ((int64_t)y0 * r) >> 31
                                                  : ((int64_t)(y0 >> 16) * r + (((int64_t)(y0 & 0xFFFFu) * r) >> 16)) >> 15;
    const int64_t y1 = (int64_t)y0 + step, lo = (int64_t)1 << 31, hi = ((int64_t)1 << 32) - 1;
    Rm = (uint64_t)(y1 < lo ? lo : y1 > hi ? hi : y1);
    sh = 47 + d / 2;
}

__device__ __forceinline__ int rne_sat(int64_t v, uint32_t sc) {
    return (int)(sc <= 61 ? ro::sat16(ro::rne_shr_fast(v, sc)) : ro::sat16(ro::rne_shr((__int128)v, (int)sc)));
}
// v scale rounded half to even and saturated (|v scale| < 2^31): the sum with 1.5 2^52 has its units in the low word,
// one v_fma_f64 for a product, a rounding and a conversion
__device__ __forceinline__ int rne_sat_f64(double v, double scale) {
    return sat16i((int)(uint32_t)__builtin_bit_cast(uint64_t, __builtin_fma(v, scale, 0x1.8p52)));
}
// x as a double: the low word of 2^52 + 2^31 + x, less 2^52 + 2^31 (an exclusive or and a v_add_f64)
__device__ __forceinline__ double f64(int x) {
    return __builtin_bit_cast(double, (uint64_t)0x43300000u << 32 | ((uint32_t)x ^ 0x80000000u)) - 0x1.00000800p52;
}
__device__ __forceinline__ double pow2(int e) { return __builtin_bit_cast(double, (uint64_t)(1023 + e) << 52); }

// Over the L = 8 or 16 lanes of a row (DPP, no LDS)
template <uint32_t L, class F>
__device__ __forceinline__ uint32_t row_all(uint32_t x, F f) {
    x = f(x, ro::row16_step<0>(x));
    x = f(x, ro::row16_step<1>(x));
    x = f(x, ro::row16_step<2>(x));
    if constexpr (L == 16) x = f(x, ro::row16_step<3>(x));
    return x;
}
template <uint32_t L>
__device__ __forceinline__ uint64_t row_sum64(uint64_t x) {
    auto add = [&](uint32_t lo, uint32_t hi) { x += (uint64_t)hi << 32 | lo; };
    add(ro::row16_step<0>((uint32_t)x), ro::row16_step<0>((uint32_t)(x >> 32)));
    add(ro::row16_step<1>((uint32_t)x), ro::row16_step<1>((uint32_t)(x >> 32)));
    add(ro::row16_step<2>((uint32_t)x), ro::row16_step<2>((uint32_t)(x >> 32)));
    if constexpr (L == 16) add(ro::row16_step<3>((uint32_t)x), ro::row16_step<3>((uint32_t)(x >> 32)));
    return x;
}
// the sum of 8 int16 squares: two a v_dot2_i32_i16, at most 2^31 as an unsigned word
__device__ __forceinline__ uint64_t squares8(const int4 v) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    auto sq = [](int w) {
        const s16x2 x = __builtin_bit_cast(s16x2, w);
        return (uint64_t)(uint32_t)__builtin_amdgcn_sdot2(x, x, 0, false);
    };
    return sq(v.x) + sq(v.y) + sq(v.z) + sq(v.w);
}

// The 8-bit form of a row held by L lanes of 8 columns: its shift, and the codes in place
template <uint32_t L>
__device__ __forceinline__ uint32_t quantise(int (&x)[8]) {
    int m = 0;
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) m = max(m, x[l] ^ (x[l] >> 31));
    m = (int)row_all<L>((uint32_t)m, [](uint32_t p, uint32_t q) { return max(p, q); });
    const int e = max(0, 25 - __clz(m));                       // bits(m) - 7
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) {
        // round half to even in 32 bits: x + 2^(e-1) - 1 + bit e, shifted
        x[l] = min(127, e ? (x[l] + (1 << (e - 1)) - 1 + ((x[l] >> e) & 1)) >> e : x[l]);
    }
    return (uint32_t)e;
}

constexpr uint32_t kPrepGroup = 4;

// 64-row chunks of the sequences' new positions, aligned to 64 (so to pages and 16-row groups): sequence b's have the
// slots from floor(start(b) / 64) + 2 b on.
struct Chunk {
    uint32_t b, q0;
    int base, at, beg, end;                 // position of token q0; the chunk's first position; its valid rows [beg, end)
    const int32_t* tb;
    __device__ __forceinline__ Chunk(const Batch& bt, uint32_t slot) {
        b = find_le(bt.batch, slot, [&](uint32_t i) { return bt.start(i) / 64 + 2 * i; });
        q0 = bt.start(b);
        // A length past 2^30 stands for any past the table (2^20 rows at most): the places below stay within int32 whatever
        // kv_len holds (a length near 2^31 with more than a table's rows of padding wrapped to places outside q, k and v).
        const int n = max((int)bt.start(b + 1) - (int)q0, 0), len = min(bt.len(b), 1 << 30);
        base = len - n;
        const int ci = (int)(slot - (q0 / 64 + 2 * b));
        at = (base >> 6) * 64 + 64 * ci;
        beg = max(max(base, 0) - at, 0);
        end = min(min(len, (int)bt.cap) - at, 64);
        tb = bt.table + b * bt.table_ld;
    }
};
inline uint64_t chunk_slots(const Batch& b) { return (uint64_t)b.tokens / 64 + 2 * (uint64_t)b.batch; }

// One launch, two kinds of workgroups.  q and k: HD / 8 lanes a head row, 8 columns a lane; a wavefront takes PG passes
// of 64 / L of a token's rows and `tpw` tokens, so that PG rows' loads are in flight and a token's table row is
// converted once for them.  Its arithmetic is the row-ops unit's, in double where every product is a whole number below
// 2^53 (the norm's x Rm and P1 G, the rotation's two products; rounded by the sum with 1.5 2^52).  V: a chunk of 64
// positions of a head, transposed through LDS and stored as whole 16-key pieces where all 16 are new.
// 8192 tokens of 15 + 5 heads of 64 with norms: 31 us for 63 MB (2.0 TB/s, a copy's rate 5.2); without the norms'
// arithmetic 23, without the rotation's 21, V's part alone 5.5: bound by the doubles at 2 wavefronts a SIMD (four passes
// take 235 registers; 56 SGPRs go to vector lanes, no register to memory).
template <uint32_t HD, bool I8, uint32_t PG>
__global__ __launch_bounds__(256) void paged_prep_kernel(Cache c, Batch bt, Prep a, uint32_t qk_blocks, uint32_t passes, uint32_t tpw) {
    constexpr uint32_t L = HD / 8, RW = 64 / L;
    typedef Block<HD, I8> B;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kRsqrt];       // the rsqrt table, or V's transposition
    static_assert(64 * (HD + 2) * 2 <= sizeof(lds), "a chunk of V");
    const uint32_t t = threadIdx.x, lane = t & 63, u = lane % L, d0 = 8 * u;
    if (blockIdx.x >= qk_blocks) {
        int16_t (*vt)[HD + 2] = reinterpret_cast<int16_t (*)[HD + 2]>(lds);
        const uint32_t vb = blockIdx.x - qk_blocks, head = vb % c.kv;
        const Chunk ch(bt, vb / c.kv);
        if (ch.beg >= ch.end) return;
        for (uint32_t i = t; i < 64 * L; i += 256) {
            const int j = (int)(i / L);
            const bool on = j >= ch.beg && j < ch.end;
            if (__ballot(on) == 0) continue;
            const int64_t tok = (int64_t)ch.q0 + ch.at + j - ch.base;
            const int4 w = on ? *reinterpret_cast<const int4*>(a.v + tok * a.v_ld + head * HD + d0) : make_int4(0, 0, 0, 0);
            int x[8];
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) x[l] = (int)reinterpret_cast<const int16_t*>(&w)[l];
            if constexpr (I8) {
                const uint32_t e = quantise<L>(x);
                if (on && u == 0) {
                    const uint32_t id = (uint32_t)ch.tb[(uint32_t)(ch.at + j) >> c.lg];
                    if (id < c.pages)
                        c.data[((uint64_t)id * c.kv + head) * c.block + B::ve(c.page) + ((uint32_t)(ch.at + j) & (c.page - 1))] = (uint8_t)e;
                }
            }
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) vt[j][d0 + l] = (int16_t)x[l];
        }
        __syncthreads();
        for (uint32_t i = t; i < 4 * HD; i += 256) {
            const uint32_t d = i % HD, j0 = 16 * (i / HD);
            const int gb = max(ch.beg - (int)j0, 0), ge = min(ch.end - (int)j0, 16);
            if (gb >= ge) continue;
            const uint32_t p0 = (uint32_t)(ch.at + (int)j0), id = (uint32_t)ch.tb[p0 >> c.lg];
            if (id >= c.pages) continue;
            uint8_t* dst = c.data + ((uint64_t)id * c.kv + head) * c.block + B::v(c.page, 0) + d * c.page + (p0 & (c.page - 1));
            uint32_t h[4], lo[4];
#pragma unroll
            for (uint32_t q = 0; q < 4; q++) {
                h[q] = lo[q] = 0;
#pragma unroll
                for (uint32_t l = 0; l < 4; l++) {
                    const uint32_t x = (uint16_t)vt[j0 + 4 * q + l][d];
                    h[q] |= ((I8 ? x : x >> 8) & 255u) << (8 * l);
                    lo[q] |= ((x & 255u) ^ 128u) << (8 * l);
                }
            }
            if (gb == 0 && ge == 16) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
                if constexpr (!I8) *reinterpret_cast<uint4*>(dst + HD * c.page) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            } else {
#pragma unroll
                for (int l = 0; l < 16; l++) {
                    if (l < gb || l >= ge) continue;
                    dst[l] = (uint8_t)(h[l / 4] >> (8 * (l & 3)));
                    if constexpr (!I8) dst[HD * c.page + l] = (uint8_t)(lo[l / 4] >> (8 * (l & 3)));
                }
            }
        }
        return;
    }
    // every load that needs no other comes first: the rsqrt table, the first token's x, the parameters, the batch
    __shared__ double nG[2][HD];            // the norms' G 2^-sc
    const bool norms = a.norm_q != nullptr || a.norm_k != nullptr;
    if (norms) {
#pragma unroll
        for (uint32_t i = 0; i < kRsqrt / 1024; i++)
            __builtin_amdgcn_global_load_lds(a.tab + 32768 + 4 * 2048 + 16 * (t + 256 * i),
                                             (__attribute__((address_space(3))) void*)(lds + 16 * (64 * (t >> 6) + 256 * i)), 16, 0, 0);
    }
    const uint32_t groups = (passes + PG - 1) / PG;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (t >> 6)), ps0 = wv % groups * PG;
    const uint32_t t0 = min(wv / groups * tpw, bt.tokens - 1);      // past the end: below
    const bool idle = wv / groups * tpw >= bt.tokens;
    const uint32_t rows = a.heads + c.kv;
    // the lane's row of pass p: on, of q or of k, its head
    auto row = [&](uint32_t p) { return (ps0 + p) * RW + lane / L; };
    auto on = [&](uint32_t p) { return row(p) < rows; };
    auto isq = [&](uint32_t p) { return row(p) < a.heads; };
    auto head = [&](uint32_t p) { return isq(p) ? row(p) : on(p) ? row(p) - a.heads : 0u; };
    int4 xn[PG], c0, c1, s0, s1;            // the next token's
    auto load_x = [&](uint32_t tok) {
#pragma unroll
        for (uint32_t p = 0; p < PG; p++)
            xn[p] = *reinterpret_cast<const int4*>((isq(p) ? a.q + tok * a.q_ld : a.k + tok * a.k_ld) + head(p) * HD + d0);
    };
    load_x(t0);
    // The double forms: a lane's 8 columns at the same shifts, the norm's Bq 0.  x cos + y sin is below 2^47 for any
    // int32 table, its rounded quotient below 2^30; |P1 G| below 2^52 (see below), its quotient below 2^30.
    double rS[PG];
    uint32_t plain = 0;                     // a bit a pass
    {
        uint4 rw[PG];
#pragma unroll
        for (uint32_t p = 0; p < PG; p++)
            rw[p] = *reinterpret_cast<const uint4*>(isq(p) ? a.rope_q + (a.rope_q_cols ? 16 * (head(p) * HD + d0) : 0u)
                                                           : a.rope_k + (a.rope_k_cols ? 16 * (head(p) * HD + d0) : 0u));
#pragma unroll
        for (uint32_t p = 0; p < PG; p++) {
            const ro::Param r0 = ro::param_of(rw[p]);
            bool ok = r0.sa == r0.sb && r0.sc >= r0.sa + 17;
            if (isq(p) ? a.rope_q_cols : a.rope_k_cols) {
                const uint8_t* rp = (isq(p) ? a.rope_q : a.rope_k) + 16 * (head(p) * HD + d0);
#pragma unroll
                for (uint32_t l = 1; l < 8; l++)
                    ok = ok && ((reinterpret_cast<const uint4*>(rp)[l].z ^ rw[p].z) & 0x3F3F3Fu) == 0;
            }
            rS[p] = pow2(r0.sa - r0.sc);
            plain |= __all(ok || !on(p)) ? 1u << p : 0u;
        }
    }
    uint32_t b, next, total;
    int64_t base;                           // position = base + token
    if (bt.batch <= 64) {
        const uint32_t i = min(lane, bt.batch - 1), s0 = bt.start(i), s1 = bt.start(i + 1), l = (uint32_t)bt.len(i);
        b = max((uint32_t)__popcll(__ballot(lane < bt.batch && s0 <= t0)), 1u) - 1;
        next = (uint32_t)__builtin_amdgcn_readlane((int)s1, b);
        base = (int64_t)__builtin_amdgcn_readlane((int)l, b) - next;
        total = (uint32_t)__builtin_amdgcn_readlane((int)s1, bt.batch - 1);
    } else {
        b = find_le(bt.batch, t0, [&](uint32_t i) { return bt.start(i); });
        next = bt.start(b + 1);
        base = (int64_t)bt.len(b) - next;
        total = bt.start(bt.batch);
    }
    bool nplain[2] = {true, true};
    if (norms) {
#pragma unroll
        for (uint32_t k = 0; k < 2; k++) {
            const uint8_t* np = k == 0 ? a.norm_q : a.norm_k;
            bool ok = true;
            if (np != nullptr && t < HD) {
                const ro::Param n = ro::ld_param(np, t, false);
                nG[k][t] = (double)(int)n.g * pow2(-n.sc);
                ok = n.sc >= 22 && n.bq == 0 && n.g < (1 << 27) && n.g > -(1 << 27);
            }
            nplain[k] = __syncthreads_and(ok) != 0;
        }
        __builtin_amdgcn_s_waitcnt(0x0070);
        __syncthreads();
    }
    if (idle || t0 >= total) return;
    const uint32_t t1 = min(t0 + tpw, total), half = a.rotary / 2;
    const bool rot = d0 < a.rotary, upper = !a.interleaved && d0 >= half;
    const int pl = (int)(!rot || a.interleaved ? lane : d0 < half ? lane + half / 8 : lane - half / 8);
    const uint32_t minus = a.interleaved || upper ? 0u : 0x80000000u;     // the partner's sign, on its product's high word
    // A token's loads are issued before the stores of the one before: a wait for a load is a wait for every older store
    int64_t pos;
    const int32_t* cs;
    uint32_t id;
    auto fetch = [&](uint32_t tok) {
        while (tok >= next && b + 1 < bt.batch) {
            next = bt.start(++b + 1);
            base = (int64_t)bt.len(b) - next;
        }
        pos = base + tok;
        const uint32_t trow = (uint32_t)min(max(pos, (int64_t)0), (int64_t)a.rope_rows - 1);
        cs = a.rope + (uint64_t)trow * 2 * a.rotary + (rot ? d0 : 0u);
        c0 = *reinterpret_cast<const int4*>(cs);
        c1 = *reinterpret_cast<const int4*>(cs + 4);
        s0 = *reinterpret_cast<const int4*>(cs + a.rotary);
        s1 = *reinterpret_cast<const int4*>(cs + a.rotary + 4);
        id = pos >= 0 && pos < (int64_t)bt.cap ? (uint32_t)bt.table[b * bt.table_ld + (uint32_t)(pos >> c.lg)] : ~0u;
    };
    // x[l] = f(l, x[l]) one column at a time, in the lane's LDS words: a loop's index into registers costs 60 of them
    __shared__ __attribute__((aligned(16))) int16_t slow_x[256][8], slow_y[256][8];
    auto slow = [&](int (&x)[8], auto f) {
        *reinterpret_cast<int4*>(slow_x[t]) = ro::pack16(x);
#pragma unroll 1
        for (uint32_t l = 0; l < 8; l++) slow_x[t][l] = (int16_t)f(l, (int)slow_x[t][l]);
        const int4 w = *reinterpret_cast<const int4*>(slow_x[t]);
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) x[l] = (int)reinterpret_cast<const int16_t*>(&w)[l];
    };
    fetch(t0);
    for (uint32_t tok = t0; tok < t1; tok++) {
        double co[8], si[8];
        {
            const int ci[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, sj[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) {
                co[l] = rot ? f64(ci[l]) : 0x1p23;
                si[l] = rot ? f64(sj[l]) : 0.0;
            }
        }
        int4 xc[PG];
#pragma unroll
        for (uint32_t p = 0; p < PG; p++) xc[p] = xn[p];
        const uint32_t slot = (uint32_t)pos & (c.page - 1), page = id;
        const int32_t* trow = cs;
        if (tok + 1 < t1) {
            load_x(tok + 1);
            fetch(tok + 1);
        }
#pragma unroll
        for (uint32_t p = 0; p < PG; p++) {
            if (p && ps0 + p >= passes) break;
            const uint32_t g = head(p);
            const bool q_row = isq(p), live = on(p);
            int x[8];
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) x[l] = (int)reinterpret_cast<const int16_t*>(&xc[p])[l];
            if (norms) {                    // every lane: the sums are the wavefront's
                const uint64_t s2 = row_sum64<L>(squares8(xc[p]));
                const uint8_t* np = q_row ? a.norm_q : a.norm_k;
                if (np != nullptr) {
                    const uint64_t D = max(s2 + (uint64_t)(q_row ? a.eps_q : a.eps_k), (uint64_t)1);
                    uint64_t Rm;
                    int sh;
                    rsqrt64(D, Rm, sh, reinterpret_cast<const uint32_t*>(lds));
                    const double scale = (double)Rm * pow2(24 - sh);        // x scale: 48 bits, exact
                    // |x| <= sqrt(D), so |P1| <= sqrt(D) scale + 1; below 2^25 (the unit's own table: 2^24) P1 G is below 2^52
                    if (nplain[q_row ? 0 : 1] && scale * scale * (double)D < 0x1p49) {
#pragma unroll
                        for (uint32_t l = 0; l < 8; l++)
                            x[l] = rne_sat_f64(__builtin_floor(f64(x[l]) * scale), nG[q_row ? 0 : 1][d0 + l]);
                    } else {
                        slow(x, [&](uint32_t l, int v) {
                            const ro::Param n = ro::ld_param(np, d0 + l, false);
                            return rne_sat((((int64_t)v * (int64_t)Rm) >> (sh - 24)) * n.g + n.bq, (uint32_t)n.sc);
                        });
                    }
                }
            }
            int y[8];                       // the partners
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) y[l] = a.interleaved ? x[l ^ 1] : __shfl(x[l], pl, 64);
            if (plain >> p & 1) {
#pragma unroll
                for (uint32_t l = 0; l < 8; l++) {
                    const uint32_t m = a.interleaved && !(l & 1) ? 0x80000000u : minus;
                    const double ys = f64(y[l]) * si[l];
                    const double z = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, ys) ^ (uint64_t)m << 32);
                    x[l] = rne_sat_f64(__builtin_fma(f64(x[l]), co[l], z), rS[p]);
                }
            } else {
                const uint8_t* rp = q_row ? a.rope_q : a.rope_k;
                const bool cols = (q_row ? a.rope_q_cols : a.rope_k_cols) != 0;
                *reinterpret_cast<int4*>(slow_y[t]) = ro::pack16(y);
                slow(x, [&](uint32_t l, int v) {
                    const bool neg = a.interleaved ? !(l & 1) : !upper;
                    const int w = slow_y[t][l];
                    return ro::rope_elem(v, neg ? -w : w, rot ? trow[l] : 1 << 23, rot ? trow[a.rotary + l] : 0,
                                         ro::ld_param(rp, g * HD + d0 + l, !cols));
                });
            }
            if (live && q_row) *reinterpret_cast<int4*>(a.qr + tok * a.qr_ld + g * HD + d0) = ro::pack16(x);
            if ((ps0 + p + 1) * RW <= a.heads) continue;      // no k row in this pass
            uint32_t e = 0;
            if constexpr (I8) e = quantise<L>(x);
            int s = 0;
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) s += x[l];
            s = (int)row_all<L>((uint32_t)s, [](uint32_t p, uint32_t q) { return p + q; });
            if (!live || q_row || page >= c.pages) continue;
            uint8_t* blk = c.data + ((uint64_t)page * c.kv + g) * c.block;
            if constexpr (I8) {
                uint32_t h[2];
#pragma unroll
                for (uint32_t w = 0; w < 2; w++)
                    h[w] = (x[4 * w] & 255) | (x[4 * w + 1] & 255) << 8 | (x[4 * w + 2] & 255) << 16 | (uint32_t)x[4 * w + 3] << 24;
                *reinterpret_cast<uint2*>(blk + B::k(c.page, 0) + slot * HD + d0) = make_uint2(h[0], h[1]);
            } else {
                uint2 h, lo;
                split8(ro::pack16(x), h, lo);
                *reinterpret_cast<uint2*>(blk + B::k(c.page, 0) + slot * HD + d0) = h;
                *reinterpret_cast<uint2*>(blk + B::k(c.page, 1) + slot * HD + d0) = lo;
            }
            if (u == 0) {
                reinterpret_cast<int32_t*>(blk + B::term(c.page))[slot] = 128 * s - (I8 ? 0 : 16384 * (int)HD);
                if constexpr (I8) blk[B::ke(c.page) + slot] = (uint8_t)e;
            }
        }
    }
}

// ---------------------------------------------------------------- read
// A workgroup per 64-position chunk of a head: K rows as they lie, V 16 keys a lane through LDS.
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_read_kernel(Cache c, Batch bt, int16_t* k, int16_t* v, uint64_t k_ld, uint64_t v_ld) {
    constexpr uint32_t L = HD / 8;
    typedef Block<HD, I8> B;
    __shared__ int16_t vt[64][HD + 2];
    const uint32_t t = threadIdx.x, head = blockIdx.y;
    const Chunk ch(bt, blockIdx.x);
    const int n = (int)bt.start(ch.b + 1) - (int)ch.q0;
    const int rb = max(ch.base - ch.at, 0), re = min(ch.base + n - ch.at, 64);     // the chunk's tokens (without a row: zeros)
    if (rb >= re) return;
    auto block = [&](int j) -> const uint8_t* {
        if (j < ch.beg || j >= ch.end) return nullptr;
        const uint32_t id = (uint32_t)ch.tb[(uint32_t)(ch.at + j) >> c.lg];
        return id < c.pages ? c.data + ((uint64_t)id * c.kv + head) * c.block : nullptr;
    };
    for (uint32_t i = t; i < 4 * HD; i += 256) {
        const uint32_t d = i % HD, j0 = 16 * (i / HD);
        const int gb = max(ch.beg - (int)j0, 0), ge = min(ch.end - (int)j0, 16);
        uint32_t h[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0}, es[4] = {0, 0, 0, 0};
        const uint8_t* blk = gb < ge ? block((int)j0 + gb) : nullptr;
        if (blk != nullptr) {                                  // the whole 16-key piece lies in the page
            const uint32_t in = (uint32_t)(ch.at + (int)j0) & (c.page - 1);
            const uint8_t* p = blk + B::v(c.page, 0) + d * c.page + in;
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            h[0] = a.x; h[1] = a.y; h[2] = a.z; h[3] = a.w;
            const uint4 z = *reinterpret_cast<const uint4*>(I8 ? blk + B::ve(c.page) + in : p + HD * c.page);
            (I8 ? es : lo)[0] = z.x; (I8 ? es : lo)[1] = z.y; (I8 ? es : lo)[2] = z.z; (I8 ? es : lo)[3] = z.w;
        }
#pragma unroll
        for (uint32_t l = 0; l < 16; l++) {
            const int hb = (int8_t)(h[l / 4] >> (8 * (l & 3))), lb = (int8_t)(lo[l / 4] >> (8 * (l & 3)));
            const int x = I8 ? hb << ((es[l / 4] >> (8 * (l & 3))) & 15u) : hb * 256 + lb + 128;
            vt[j0 + l][d] = (int16_t)((int)l >= gb && (int)l < ge && blk != nullptr ? x : 0);
        }
    }
    __syncthreads();
    for (uint32_t i = t; i < 64 * L; i += 256) {
        const int j = (int)(i / L);
        const uint32_t d0 = 8 * (i % L);
        if (j < rb || j >= re) continue;
        const uint64_t tok = (uint64_t)((int64_t)ch.q0 + ch.at + j - ch.base);
        int x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, y[8];
        if (const uint8_t* blk = block(j)) {
            const uint32_t slot = (uint32_t)(ch.at + j) & (c.page - 1);
            const uint8_t* kp = blk + B::k(c.page, 0) + slot * HD + d0;
            const uint2 h = *reinterpret_cast<const uint2*>(kp);
            uint2 lo = make_uint2(0, 0);
            uint32_t e = 0;
            if constexpr (I8) e = blk[B::ke(c.page) + slot] & 15u;
            else lo = *reinterpret_cast<const uint2*>(kp + c.page * HD);
#pragma unroll
            for (uint32_t l = 0; l < 8; l++) {
                const int hb = (int8_t)((l < 4 ? h.x : h.y) >> (8 * (l & 3))), lb = (int8_t)((l < 4 ? lo.x : lo.y) >> (8 * (l & 3)));
                x[l] = I8 ? hb << e : hb * 256 + lb + 128;
            }
        }
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) y[l] = vt[j][d0 + l];
        *reinterpret_cast<int4*>(k + tok * k_ld + head * HD + d0) = ro::pack16(x);
        *reinterpret_cast<int4*>(v + tok * v_ld + head * HD + d0) = ro::pack16(y);
    }
}

// ---------------------------------------------------------------- attention
// The exponential of d = max - s: y = (d Cm) >> Cs, e = TAB[y & 4095] >> (y >> 12).  The kernels take 4 y, a byte
// offset into TAB, as the high word of (min(d, dlim) << sh) mul: one product.  At dlim, the least d with y >= 17 * 4096,
// e is 0; y there stays below 2^17, a shift below 32 (the host replaces register pairs whose single step passes 15
// octaves by one of the same exponentials).  Cm counts from its top bit (its pair is as good with both moved), so
// mul = Cm 2^8 has 32 bits and sh = 26 - Cs with d below 2^(Cs - 5) or 2^16; Cs above 34 would need sh < -8: all 65535
// steps of a score within 1/128 octave, which the host refuses.
struct Smx {
    uint32_t mul, sh, dlim;                    // dlim at most 65535: no d passes it
};

bool smx_of(uint32_t cm24, uint32_t cs, Smx* r) {
    r->mul = r->sh = 0;
    r->dlim = 65535;
    if (cm24 == 0) return true;                // e = TAB[0] for every d
    const uint32_t dlim = smx_dlim(cm24, cs), step = cs < 32 ? cm24 >> cs : 0u;
    r->dlim = dlim < 65535u ? dlim : 65535u;
    if (step >= 61440u) {                      // d = 1 has y = step, every d >= 2 gives 0
        cs = 0;
        r->dlim = step > 65536u ? 1u : 2u;     // above 2^16: e(1) = 0
        cm24 = step > 65536u ? kSmxYZero : (step < 65535u ? step : 65535u);   // e(1) is 1 at 65535 as at 65536
    }
    const uint32_t up = (uint32_t)__builtin_clz(cm24) - 8;
    cm24 <<= up;
    cs += up;
    // 4 y = (d cm24) >> (cs - 2) = (d 2^sh mul) >> 32, sh + log2(mul / cm24) = 34 - cs
    if (cs > 34) return false;
    const uint32_t total = 34 - cs, low = total < 8 ? total : 8u;
    r->mul = cm24 << low;
    r->sh = total - low;
    return true;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

// The exponentials of two scores s (saturated to int16 as they are packed) under the maximum m: the TAB words and
// their shifts; w = min(word >> shift, 65535) is taken where two are packed again (v_cvt_pk_u16_u32 saturates).
// dl = min(dlim, 65535): d <= 65535.
struct Exp2 {
    uint32_t t0, t1, k0, k1;
    __device__ __forceinline__ uint32_t e0() const { return t0 >> k0; }
    __device__ __forceinline__ uint32_t e1() const { return t1 >> k1; }
};
// HALF: tab holds TAB - 1 in 16 bits
template <bool HALF = false>
__device__ __forceinline__ Exp2 exps(int s0, int s1, uint32_t m2, uint32_t dl2, const Smx& x, const int32_t* tab) {
    const u16x2 s = __builtin_bit_cast(u16x2, __builtin_amdgcn_cvt_pk_i16(s0, s1));
    const u16x2 d = __builtin_elementwise_min(__builtin_bit_cast(u16x2, m2) - s, __builtin_bit_cast(u16x2, dl2));
    const uint32_t y0 = __umulhi((uint32_t)d[0] << x.sh, x.mul), y1 = __umulhi((uint32_t)d[1] << x.sh, x.mul);
    const uint8_t* tb = reinterpret_cast<const uint8_t*>(tab);
    if constexpr (HALF)
        return Exp2{*reinterpret_cast<const uint16_t*>(tb + (y0 >> 1 & 0x1FFEu)) + 1u,
                    *reinterpret_cast<const uint16_t*>(tb + (y1 >> 1 & 0x1FFEu)) + 1u, y0 >> 14, y1 >> 14};
    return Exp2{*reinterpret_cast<const uint32_t*>(tb + (y0 & 0x3FFCu)), *reinterpret_cast<const uint32_t*>(tb + (y1 & 0x3FFCu)),
                y0 >> 14, y1 >> 14};
}
__device__ __forceinline__ uint32_t pair16(uint32_t a, uint32_t b) {      // saturated to 65535
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_u16(a, b));
}
__device__ __forceinline__ uint32_t add16(uint32_t p, uint32_t sum) {     // sum + both halves of p
    return __builtin_amdgcn_udot2(__builtin_bit_cast(u16x2, p), u16x2{1, 1}, sum, false);
}
__device__ __forceinline__ uint32_t twice(uint32_t x) { return (x & 0xFFFFu) | x << 16; }

struct Attn {
    const int16_t* q;
    int16_t* o;
    uint64_t q_ld, o_ld;
    uint32_t G, window, fp;
    Smx smx;
};

// 8 int16 -> their high bytes and low bytes ^ 0x80 (two dwords each)
__device__ __forceinline__ void limbs16(const int16_t* p, v4i& hi, v4i& lo, int& sum) {
    const int4 a = *reinterpret_cast<const int4*>(p), b = *reinterpret_cast<const int4*>(p + 8);
    uint2 ha, la, hb, lb;
    split8(a, ha, la);
    split8(b, hb, lb);
    sum += sum8(a) + sum8(b);
    hi = v4i{(int)ha.x, (int)ha.y, (int)hb.x, (int)hb.y};
    lo = v4i{(int)la.x, (int)la.y, (int)lb.x, (int)lb.y};
}

// floor(2^(fp - 8) A / S + 1/2) saturated to int16, A and S the exact sums of a row.  The quotient is estimated with
// the row's reciprocal in double (at most 2^23, the estimate off by less than 2^-27) and put right by the remainder
// in int64: 2 |A| 2^7 < 2^59 and f den < 2^61.
struct Divide {
    int64_t S, den;
    double inv;
    uint32_t fp;
    __device__ __forceinline__ Divide(int64_t S_, uint32_t fp_) : S(S_), fp(fp_) {
        den = fp >= 8 ? 2 * S : S << (9 - fp);
        inv = S ? 1.0 / (double)den : 0.0;
    }
    __device__ __forceinline__ int operator()(int64_t A) const {
        const int64_t num = (fp >= 8 ? A << (fp - 7) : 2 * A) + (den >> 1);
        int f = (int)floor((double)num * inv);
        const int64_t r = num - (int64_t)f * den;
        f += r >= den ? 1 : r < 0 ? -1 : 0;
        return S ? sat16i(f) : 0;
    }
};

__device__ __forceinline__ void store_out(int16_t* p, const Divide& q, const int64_t (&x)[4]) {
    const uint32_t y0 = (uint32_t)q(x[0]), y1 = (uint32_t)q(x[1]), y2 = (uint32_t)q(x[2]), y3 = (uint32_t)q(x[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2((y0 & 0xFFFFu) | y1 << 16, (y2 & 0xFFFFu) | y3 << 16);
}

// ---- the split of the work.  A tile is R rows (token, head of the group) of one sequence and KV head; sequence b's
// tiles have the slots from floor(start(b) G / R) + b on (at least as many as it needs, known without a scan).  The
// 64-key steps that any row of the tile sees go to workgroups in parts of `per` steps (the same for every tile: a short
// sequence has fewer parts, not smaller ones).

// What a tile of many rows costs beside its steps, in steps: its queries, maxima and first keys, its sums' end.  A prompt
// of 4096 tokens: 3 and 6 for 4 take 169 and 168 us for 161 (the weights' kernel alone: 1 and 2 for 4, 140 and 135 for 120).
constexpr uint32_t kTileCost = 4;

template <uint32_t R>
struct Tile {
    struct Seqs {                          // lane i: sequence i's first token, the next one's, its length (batch <= 64)
        uint32_t s0, s1, len;
        Seqs() = default;
        __device__ __forceinline__ Seqs(const Batch& bt) {
            const uint32_t i = min(threadIdx.x & 63, bt.batch - 1);
            s0 = bt.start(i);
            s1 = bt.start(i + 1);
            len = (uint32_t)bt.len(i);
        }
    };
    uint32_t b, q0, n, row0, rows;         // sequence, its first token, tokens; the tile's first row, the sequence's rows
    uint32_t lo, hi, nt;                   // keys [lo, hi) that a row sees, lo a multiple of 64; 64-key steps
    uint32_t all_lo, all_hi;               // keys that every row sees
    int base;
    const int32_t* tb;
    bool on;

    __device__ __forceinline__ Tile(const Batch& bt, const Attn& a, uint32_t slot) : Tile(bt, a, slot, Seqs(bt)) {}
    __device__ __forceinline__ Tile(const Batch& bt, const Attn& a, uint32_t slot, const Seqs& sq) {
        uint32_t q1, first;
        int len;
        if (bt.batch <= 64) {
            const uint32_t f = (uint32_t)((uint64_t)sq.s0 * a.G / R) + min(threadIdx.x & 63, bt.batch - 1);
            b = max((uint32_t)__popcll(__ballot((threadIdx.x & 63) < bt.batch && f <= slot)), 1u) - 1;
            q0 = (uint32_t)__builtin_amdgcn_readlane((int)sq.s0, b);
            q1 = (uint32_t)__builtin_amdgcn_readlane((int)sq.s1, b);
            len = __builtin_amdgcn_readlane((int)sq.len, b);
            first = (uint32_t)__builtin_amdgcn_readlane((int)f, b);
        } else {
            auto at = [&](uint32_t i) { return (uint32_t)((uint64_t)bt.start(i) * a.G / R) + i; };
            b = find_le(bt.batch, slot, at);
            q0 = bt.start(b);
            q1 = bt.start(b + 1);
            len = bt.len(b);
            first = at(b);
        }
        n = (uint32_t)max((int)q1 - (int)q0, 0);
        row0 = (slot - first) * R;
        rows = n * a.G;
        on = row0 < rows;
        base = len - (int)n;
        tb = bt.table + b * bt.table_ld;
        const uint32_t tf = row0 / a.G, tl = on ? min((row0 + R - 1) / a.G, n - 1) : tf;
        lo = __builtin_amdgcn_readfirstlane(begin(a, tf) & ~63u);
        hi = __builtin_amdgcn_readfirstlane(seen(bt, tl));
        all_lo = __builtin_amdgcn_readfirstlane(begin(a, tl));
        all_hi = __builtin_amdgcn_readfirstlane(seen(bt, tf));
        nt = hi > lo ? (hi - lo + 63) / 64 : 0u;
    }
    // A lane's own tile: its steps, one at least (a tile without keys has zeros to write), 0 past the sequence's rows
    static __device__ __forceinline__ uint32_t lane_steps(const Batch& bt, const Attn& a, uint32_t slot, const Seqs* seqs) {
        auto start = [&](uint32_t i) { return seqs ? seqs[i].s0 : bt.start(i); };
        uint32_t b = 0, e = bt.batch;
        while (e - b > 1) {
            const uint32_t m = (b + e) / 2;
            const bool le = (uint32_t)((uint64_t)start(m) * a.G / R) + m <= slot;
            b = le ? m : b;
            e = le ? e : m;
        }
        const uint32_t s0 = start(b), s1 = seqs ? seqs[b].s1 : bt.start(b + 1), n = (uint32_t)max((int)s1 - (int)s0, 0);
        const uint32_t row0 = (slot - ((uint32_t)((uint64_t)s0 * a.G / R) + b)) * R;
        if (row0 >= n * a.G) return 0;
        const int base = (seqs ? (int)seqs[b].len : bt.len(b)) - (int)n, tf = (int)(row0 / a.G), tl = (int)min((row0 + R - 1) / a.G, n - 1);
        const int lo = a.window ? max(base + tf + 1 - (int)a.window, 0) & ~63 : 0, hi = min(max(base + tl + 1, 0), (int)bt.cap);
        return kTileCost + (hi > lo ? (uint32_t)(hi - lo + 63) / 64 : 1u);
    }
    __device__ __forceinline__ uint32_t seen(const Batch& bt, uint32_t tk) const {   // keys end
        return (uint32_t)min(max(base + (int)tk + 1, 0), (int)bt.cap);
    }
    __device__ __forceinline__ uint32_t begin(const Attn& a, uint32_t tk) const {
        return a.window ? (uint32_t)max(base + (int)tk + 1 - (int)a.window, 0) : 0u;
    }
    __device__ __forceinline__ uint32_t parts(uint32_t per) const { return max((nt + per - 1) / per, 1u); }
};

// Few rows, the call's workspace: per row (head, token, head of the group: (head T + token) G + i) the maxima of its
// parts, its scores, its partial sums of w V and of w.
struct Work {
    int32_t* mx;                           // [rows][splits] raw q.K^T sums, kNone: no key
    int16_t* sc;                           // [rows][cap]
    int64_t* part;                         // [rows][splits][HD + 2]
    uint32_t splits, per;                  // most parts of a tile, steps of a part
    uint32_t splits_s, per_s;              // the same of the maxima's parts
};
constexpr int kNone = (int)0x80000000;
constexpr uint32_t kMaxPart = 32768;           // keys of a part of a tile: the int32 limb sums

// V's sums and the bytes' offsets put back: the exact sum of w V (int16: hh, mid, ll of w's and V's bytes; int8: the
// three bytes of w 2^e; every byte was taken less 128)
template <bool I8>
__device__ __forceinline__ int64_t whole_sum(int a0, int a1, int a2, int vs0, int vs1, int64_t wsum) {
    const int64_t x = (int64_t)a0 * 65536 + (int64_t)a1 * 256 + a2;
    return x + (I8 ? (int64_t)vs0 * (128 * 65793) : ((int64_t)vs0 * 256 + vs1) * 32896 + 128 * wsum);
}

// four weights as two pairs (int8: shifted by the bytes of es) -> dword q of the byte operands
template <bool I8>
__device__ __forceinline__ void weight_bytes(uint32_t w01, uint32_t w23, uint32_t es, v4i (&p)[I8 ? 3 : 2], uint32_t q) {
    if constexpr (I8) {
        const uint32_t x0 = (w01 & 0xFFFFu) << (es & 15u), x1 = (w01 >> 16) << ((es >> 8) & 15u);
        const uint32_t x2 = (w23 & 0xFFFFu) << ((es >> 16) & 15u), x3 = (w23 >> 16) << ((es >> 24) & 15u);
        const uint32_t t01 = __builtin_amdgcn_perm(x1, x0, 0x05010400u), t23 = __builtin_amdgcn_perm(x3, x2, 0x05010400u);
        p[0][q] = (int)(__builtin_amdgcn_perm(t23, t01, 0x05040100u) ^ 0x80808080u);
        p[1][q] = (int)(__builtin_amdgcn_perm(t23, t01, 0x07060302u) ^ 0x80808080u);
        const uint32_t u01 = __builtin_amdgcn_perm(x1, x0, 0x0c0c0602u), u23 = __builtin_amdgcn_perm(x3, x2, 0x0c0c0602u);
        p[2][q] = (int)(__builtin_amdgcn_perm(u23, u01, 0x05040100u) ^ 0x80808080u);
    } else {
        p[0][q] = (int)(__builtin_amdgcn_perm(w23, w01, 0x06040200u) ^ 0x80808080u);
        p[1][q] = (int)(__builtin_amdgcn_perm(w23, w01, 0x07050301u) ^ 0x80808080u);
    }
}

// the raw int32 sum of a lane's key r from the limb products (e: the key's shift)
template <bool I8>
__device__ __forceinline__ int raw_sum(int hh, int mid, int ll, uint32_t es, uint32_t r, int qterm) {
    if constexpr (I8) return (int)((((uint32_t)mid << 8) + (uint32_t)ll) << ((es >> (8 * r)) & 31u));
    return (int)((((((uint32_t)hh << 8) + (uint32_t)mid) << 8) + (uint32_t)ll) + (uint32_t)qterm);
}

template <bool I8>
__device__ __forceinline__ void qk(const v4i kh, const v4i kl, const v4i qh, const v4i ql, v4i& hh, v4i& mid, v4i& ll) {
    if constexpr (I8) {
        mid = mfma(kh, qh, mid);
        ll = mfma(kh, ql, ll);
    } else {
        hh = mfma(kh, qh, hh);
        mid = mfma(kh, ql, mid);
        ll = mfma(kl, ql, ll);
        mid = mfma(kl, qh, mid);
    }
}

__device__ __forceinline__ void stage_tab(int32_t* stab, const int32_t* tab) {
    const uint32_t t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6);
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        __builtin_amdgcn_global_load_lds(tab + 4 * (t + 256 * i),
                                         (__attribute__((address_space(3))) void*)(stab + 4 * (64 * w + 256 * i)), 16, 0, 0);
}

// TAB - 1 in 16 bits (TAB is 32774 .. 65536)
__device__ __forceinline__ void stage_tab_half(int32_t* stab, const int32_t* tab) {
#pragma unroll
    for (uint32_t i = threadIdx.x; i < 1024; i += 256) {
        const int4 v = reinterpret_cast<const int4*>(tab)[i];
        reinterpret_cast<uint2*>(stab)[i] = make_uint2((uint32_t)(v.x - 1) | (uint32_t)(v.y - 1) << 16,
                                                       (uint32_t)(v.z - 1) | (uint32_t)(v.w - 1) << 16);
    }
}

// ---------------------------------------------------------------- attention of few rows
// Tiles of 15 rows: decode steps, where the cache's bytes are what costs.  Wavefronts take steps in turn and read K and
// V straight into the MFMA operands; the MFMA's sixteenth column is all ones, so V's sums (for the offset of the
// weights' bytes) come with the products.  Short caches: one kernel, every score in its wavefront's registers.
// Long ones: a kernel that leaves the scores and the maxima, a kernel for the weights and P.V, a join of the parts.
constexpr uint32_t kFewRows = 15;

template <uint32_t HD, bool I8>
struct Few {
    static constexpr uint32_t KS = HD / 64, DB = HD / 16, NP = I8 ? 1 : 2;
    typedef Block<HD, I8> B;
    const Cache& c;
    const Batch& bt;
    const Tile<kFewRows>& tl;
    uint32_t head, lane, c16, g, w, row, vend, vbeg;
    bool mine;
    uint64_t wrow;                          // the row in the workspace's order

    __device__ __forceinline__ Few(const Cache& c_, const Batch& bt_, const Attn& a, const Tile<kFewRows>& tl_, uint32_t head_)
        : c(c_), bt(bt_), tl(tl_), head(head_) {
        lane = threadIdx.x & 63;
        c16 = lane & 15;
        g = lane >> 4;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        mine = c16 < kFewRows && tl.row0 + c16 < tl.rows;
        row = mine ? tl.row0 + c16 : tl.row0;
        vend = mine ? tl.seen(bt, row / a.G) : 0u;
        vbeg = tl.begin(a, row / a.G);
        wrow = ((uint64_t)head * bt.tokens + tl.q0) * a.G + row;
    }
    struct Query {
        v4i h[KS], l[KS];
        int term;
    };
    __device__ __forceinline__ Query query(const Attn& a) const {
        Query q;
        const int16_t* qp = a.q + (uint64_t)(tl.q0 + row / a.G) * a.q_ld + (uint64_t)(head * a.G + row % a.G) * HD + 16 * g;
        int qs = 0;
#pragma unroll
        for (uint32_t s = 0; s < KS; s++) limbs16(qp + 64 * s, q.h[s], q.l[s], qs);
        qs += __shfl_xor(qs, 16, 64);
        qs += __shfl_xor(qs, 32, 64);
        q.term = I8 ? 0 : 128 * qs;
        return q;
    }
    // the page ids of the lane's K row and of its own 16 keys in step i (~0: none)
    __device__ __forceinline__ uint32_t id_at(uint32_t key, bool in) const {
        const uint32_t id = in && key < bt.cap ? (uint32_t)tl.tb[key >> c.lg] : ~0u;
        return id < c.pages ? id : ~0u;
    }
    __device__ __forceinline__ uint32_t id_row(uint32_t i, uint32_t end) const { return id_at(tl.lo + 64 * i + 16 * (c16 >> 2), i < end); }
    __device__ __forceinline__ uint32_t id_own(uint32_t i, uint32_t end) const { return id_at(tl.lo + 64 * i + 16 * g, i < end); }
    __device__ __forceinline__ const uint8_t* block(uint32_t id) const {
        return c.data + ((uint64_t)(id == ~0u ? 0u : id) * c.kv + head) * c.block;
    }
    // the scores of step i's keys 16 g .. 16 g + 15 of query c16, packed, and the maximum of the raw sums
    __device__ __forceinline__ void scores(uint32_t i, uint32_t idr, uint32_t ido, const Query& q, uint32_t (&out)[8], int& mx) const {
        const v4i zero = {0, 0, 0, 0};
        const uint32_t k0 = tl.lo + 64 * i, kr = k0 + 16 * (c16 >> 2) + (c16 & 3), kg = k0 + 16 * g, in = kg & (c.page - 1);
        const uint8_t *kp = block(idr) + (kr & (c.page - 1)) * HD + 16 * g, *tp = block(ido);
        v4i kh[4][KS], kl[4][KS], term[4], es = zero;
#pragma unroll
        for (uint32_t kb = 0; kb < 4; kb++) {
#pragma unroll
            for (uint32_t s = 0; s < KS; s++) {
                kh[kb][s] = *reinterpret_cast<const v4i*>(kp + 4 * kb * HD + 64 * s);
                if constexpr (!I8) kl[kb][s] = *reinterpret_cast<const v4i*>(kp + B::k(c.page, 1) + 4 * kb * HD + 64 * s);
            }
            term[kb] = *reinterpret_cast<const v4i*>(tp + B::term(c.page) + 4 * (in + 4 * kb));
        }
        if constexpr (I8) es = *reinterpret_cast<const v4i*>(tp + B::ke(c.page) + in);
#pragma unroll
        for (uint32_t kb = 0; kb < 4; kb++) {
            v4i hh = zero, mid = zero, ll = term[kb];
#pragma unroll
            for (uint32_t s = 0; s < KS; s++) qk<I8>(kh[kb][s], kl[kb][s], q.h[s], q.l[s], hh, mid, ll);
            int x[4];
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                x[r] = raw_sum<I8>(hh[r], mid[r], ll[r], (uint32_t)es[kb], r, q.term);
                const uint32_t key = kg + 4 * kb + r;
                mx = max(mx, ido != ~0u && key >= vbeg && key < vend ? x[r] : kNone);
            }
            out[2 * kb] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_i16(x[0] >> 8, x[1] >> 8));
            out[2 * kb + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_i16(x[2] >> 8, x[3] >> 8));
        }
    }
    // the weights of step i's scores in pairs, and their sum on top of sum (a lane's: below 2^16 * 16 * kMaxPart / 64)
    __device__ __forceinline__ void weights(uint32_t i, uint32_t ido, const uint32_t (&sw)[8], uint32_t m2, uint32_t dl2, const Smx& smx,
                                            const int32_t* stab, uint32_t (&wp)[8], uint32_t& sum) const {
        const uint32_t kg = tl.lo + 64 * i + 16 * g;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            const Exp2 x = exps((int)(int16_t)sw[j], (int)sw[j] >> 16, m2, dl2, smx, stab);
            auto on = [&](uint32_t key) { return ido != ~0u && key >= vbeg && key < vend; };
            wp[j] = pair16(on(kg + 2 * j) ? x.e0() : 0u, on(kg + 2 * j + 1) ? x.e1() : 0u);
            sum = add16(wp[j], sum);
        }
    }
    // their byte operands; the column of ones
    __device__ __forceinline__ void operands(const uint32_t (&wp)[8], const v4i es, v4i (&p)[I8 ? 3 : 2]) const {
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
            weight_bytes<I8>(wp[2 * q], wp[2 * q + 1], (uint32_t)es[q], p, q);
#pragma unroll
            for (uint32_t x = 0; x < (I8 ? 3u : 2u); x++) p[x][q] = c16 == kFewRows ? 0x01010101 : p[x][q];
        }
    }
    static __device__ __forceinline__ void pv(const v4i vh, const v4i vl, const v4i (&p)[I8 ? 3 : 2], v4i& a0, v4i& a1, v4i& a2) {
        if constexpr (I8) {
            a0 = mfma(vh, p[I8 ? 2 : 0], a0);
            a1 = mfma(vh, p[1], a1);
            a2 = mfma(vh, p[0], a2);
        } else {
            a0 = mfma(vh, p[1], a0);
            a1 = mfma(vh, p[0], a1);
            a2 = mfma(vl, p[0], a2);
            a1 = mfma(vl, p[1], a1);
        }
    }
};

// The workgroup's sums of a tile: products [row][d] (the bytes' offsets out), weights [row], V's [d].
template <uint32_t HD>
struct FewSums {
    int64_t part[kFewRows][HD], w[kFewRows], v[HD];
    __device__ __forceinline__ void clear() {
        for (uint32_t i = threadIdx.x; i < sizeof(FewSums) / 8; i += blockDim.x) reinterpret_cast<int64_t*>(this)[i] = 0;
    }
    static __device__ __forceinline__ void put(int64_t* p, int64_t x) {
        atomicAdd(reinterpret_cast<unsigned long long*>(p), (unsigned long long)x);
    }
    // a wavefront's sums added (LDS atomics of integers: the order is free): of its weights, and of 16 columns m
    template <bool I8>
    __device__ __forceinline__ void add_w(const Few<HD, I8>& f, uint32_t sum) {
        int64_t ws = sum;
        ws += (int64_t)ro::shfl64((uint64_t)ws, 16);
        ws += (int64_t)ro::shfl64((uint64_t)ws, 32);
        if (f.mine && f.g == 0) put(&w[f.c16], ws);
    }
    template <bool I8>
    __device__ __forceinline__ void add_v(const Few<HD, I8>& f, uint32_t m, const v4i a0, const v4i a1, const v4i a2) {
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) {
            const uint32_t d = 16 * m + 4 * f.g + r;
            const int64_t hh = a0[r], mid = a1[r], ll = a2[r];
            if (f.mine) put(&part[f.c16][d], hh * 65536 + mid * 256 + ll);
            else if (f.c16 == kFewRows) put(&v[d], I8 ? hh : hh * 256 + ll);
        }
    }
    template <bool I8>
    __device__ __forceinline__ int64_t sum(uint32_t r, uint32_t d) const {
        return part[r][d] + (I8 ? v[d] * (128 * 65793) : v[d] * 32896 + 128 * w[r]);
    }
    template <bool I8>
    __device__ __forceinline__ void store(const Attn& a, const Tile<kFewRows>& tl, uint32_t head) const {
        const uint32_t rows = min(kFewRows, tl.rows - tl.row0);
        for (uint32_t i = threadIdx.x; i < rows * (HD / 2); i += blockDim.x) {
            const uint32_t r = i / (HD / 2), d = 2 * (i % (HD / 2)), rw = tl.row0 + r;
            const Divide q(w[r], a.fp);
            const uint32_t y0 = (uint32_t)q(sum<I8>(r, d)), y1 = (uint32_t)q(sum<I8>(r, d + 1));
            *reinterpret_cast<uint32_t*>(a.o + (uint64_t)(tl.q0 + rw / a.G) * a.o_ld + (uint64_t)(head * a.G + rw % a.G) * HD + d) =
                (y0 & 0xFFFFu) | y1 << 16;
        }
    }
};

// Caches of at most kShort keys in one launch of 16 wavefronts a tile.  For the scores a wavefront takes steps w, w + 16;
// the weights go through LDS (16 steps a round), and for P.V a wavefront takes 16 columns of V over 4 of the round's
// steps (8 at 128 d): its sums are 12 registers, and 4 (2) of them meet in LDS instead of 16.  V's first round is read
// beside K: one memory latency for both.  16 sequences of 1024 rows, 15 heads: 10.2 us
// (V's columns undivided 11.5, with the three kernels of long caches 14.3), on 80 CUs: a CU reads 262 KB in 4 us, the
// rest is the chain of launch, batch, page ids, K, maxima, V.  At 128 int16 columns 8 of the 128 registers that 16
// wavefronts leave a lane spill.
constexpr uint32_t kShort = 2048;

template <uint32_t HD, bool I8>
__global__ __launch_bounds__(1024) void paged_short_kernel(Cache c, Batch bt, Attn a, const int32_t* __restrict__ tab) {
    typedef Few<HD, I8> F;
    typedef Block<HD, I8> B;
    constexpr uint32_t NW = 16, NS = kShort / 64 / NW, DB = HD / 16, KG = NW / DB, SP = NW / KG;   // SP steps a wavefront and round
    __shared__ __attribute__((aligned(16))) int32_t stab[4096];
    __shared__ __attribute__((aligned(16))) uint4 wts[NW][2][64];
    __shared__ int32_t redm[NW][16];
    __shared__ FewSums<HD> sums;
    const Tile<kFewRows> tl(bt, a, blockIdx.x);
    if (!tl.on) return;
    const F f(c, bt, a, tl, blockIdx.y);
    __builtin_amdgcn_global_load_lds(tab + 4 * threadIdx.x, (__attribute__((address_space(3))) void*)(stab + 256 * f.w), 16, 0, 0);
    sums.clear();
    const uint32_t vm = f.w % DB, vk = f.w / DB;     // the wavefront's columns of V, and its steps vk, vk + KG, .. of a round
    constexpr uint32_t PF = HD == 64 || I8 ? 4 : 2;    // steps of V read ahead: 32 registers at most
    uint32_t idr[NS], ido[NS], sw[NS][8], idv[PF];
#pragma unroll
    for (uint32_t k = 0; k < NS; k++) {
        idr[k] = f.id_row(f.w + NW * k, tl.nt);
        ido[k] = f.id_own(f.w + NW * k, tl.nt);
    }
#pragma unroll
    for (uint32_t k = 0; k < PF; k++) idv[k] = f.id_own(vk + KG * k, tl.nt);
    struct VCols {
        v4i h, l, es;
    } v[PF];
    auto load_v = [&](uint32_t i, uint32_t id, VCols& x) {
        const uint32_t in = (tl.lo + 64 * i + 16 * f.g) & (c.page - 1);
        const uint8_t *vb = f.block(id), *vp = vb + B::v(c.page, 0) + (16 * vm + f.c16) * c.page + in;
        x.h = *reinterpret_cast<const v4i*>(vp);
        if constexpr (!I8) x.l = *reinterpret_cast<const v4i*>(vp + HD * c.page);
        if constexpr (I8) x.es = *reinterpret_cast<const v4i*>(vb + B::ve(c.page) + in);
        else x.es = v4i{0, 0, 0, 0};
    };
    const typename F::Query q = f.query(a);
#pragma unroll
    for (uint32_t k = 0; k < PF; k++)
        if (vk + KG * k < tl.nt) load_v(vk + KG * k, idv[k], v[k]);
    int mx = kNone;
#pragma unroll
    for (uint32_t k = 0; k < NS; k++)
        if (f.w + NW * k < tl.nt) f.scores(f.w + NW * k, idr[k], ido[k], q, sw[k], mx);
    mx = max(mx, __shfl_xor(mx, 16, 64));
    mx = max(mx, __shfl_xor(mx, 32, 64));
    if (f.g == 0) redm[f.w][f.c16] = mx;
    __builtin_amdgcn_s_waitcnt(0x0070);               // the TAB's copies
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < NW; k++) mx = max(mx, redm[k][f.c16]);
    const uint32_t m2 = twice((uint32_t)sat16i(mx >> 8)), dl2 = twice(a.smx.dlim);
    v4i acc[3] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
    uint32_t wsum = 0;
#pragma unroll
    for (uint32_t k = 0; k < NS; k++) {
        if (k && NW * k >= tl.nt) break;
        if (k) __syncthreads();                        // the round before read
        if (f.w + NW * k < tl.nt) {
            uint32_t wp[8];
            f.weights(f.w + NW * k, ido[k], sw[k], m2, dl2, a.smx, stab, wp, wsum);
            wts[f.w][0][f.lane] = make_uint4(wp[0], wp[1], wp[2], wp[3]);
            wts[f.w][1][f.lane] = make_uint4(wp[4], wp[5], wp[6], wp[7]);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < SP; j++) {
            const uint32_t st = vk + KG * j, i = st + NW * k;
            if (i >= tl.nt) break;
            if (k || j >= PF) load_v(i, f.id_own(i, tl.nt), v[j % PF]);
            const uint4 w0 = wts[st][0][f.lane], w1 = wts[st][1][f.lane];
            const uint32_t wp[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
            v4i p[I8 ? 3 : 2];
            f.operands(wp, v[j % PF].es, p);
            F::pv(v[j % PF].h, v[j % PF].l, p, acc[0], acc[1], acc[2]);
        }
    }
    if (f.w < tl.nt) sums.template add_w<I8>(f, wsum);
    if (vk < tl.nt) sums.template add_v<I8>(f, vm, acc[0], acc[1], acc[2]);
    __syncthreads();
    sums.template store<I8>(a, tl, blockIdx.y);
}

// Long caches.  A workgroup takes `per_s` steps, its four wavefronts in turn.  24 sequences of 300 .. 8192 rows, 8 x 128
// in 8 bits: 20 us for 64 MB (3.2 TB/s; 22 with the first, cold call among ten), the weights and V 22.5 (23) for as much;
// two steps' rows in flight a wavefront 29 (fewer wavefronts), 4 or 16 steps a workgroup 21.5.
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_scores_kernel(Cache c, Batch bt, Attn a, Work wk) {
    typedef Few<HD, I8> F;
    __shared__ int32_t redm[4][16];
    const uint32_t z = blockIdx.z;
    const Tile<kFewRows> tl(bt, a, blockIdx.x);
    if (!tl.on || z >= tl.parts(wk.per_s)) return;
    const F f(c, bt, a, tl, blockIdx.y);
    const uint32_t beg = z * wk.per_s + f.w, end = min((z + 1) * wk.per_s, tl.nt);
    uint32_t idr = f.id_row(beg, end), ido = f.id_own(beg, end);
    const typename F::Query q = f.query(a);
    int mx = kNone;
    for (uint32_t i = beg; i < end; i += 4) {
        const uint32_t nr = f.id_row(i + 4, end), no = f.id_own(i + 4, end), kg = tl.lo + 64 * i + 16 * f.g;
        uint32_t out[8];
        f.scores(i, idr, ido, q, out, mx);
        if (f.mine && kg < bt.cap) {                  // cap is a multiple of 16
            uint4* sp = reinterpret_cast<uint4*>(wk.sc + f.wrow * bt.cap + kg);
            sp[0] = make_uint4(out[0], out[1], out[2], out[3]);
            sp[1] = make_uint4(out[4], out[5], out[6], out[7]);
        }
        idr = nr;
        ido = no;
    }
    mx = max(mx, __shfl_xor(mx, 16, 64));
    mx = max(mx, __shfl_xor(mx, 32, 64));
    if (f.g == 0) redm[f.w][f.c16] = mx;
    __syncthreads();
    if (threadIdx.x < 16 && f.mine)
        wk.mx[f.wrow * wk.splits_s + z] = max(max(redm[0][f.c16], redm[1][f.c16]), max(redm[2][f.c16], redm[3][f.c16]));
}

// the maximum score of a row over its parts: the four lanes of a row (groups g) take every fourth, loads in fours
__device__ __forceinline__ int row_max(const Work& wk, uint64_t wrow, uint32_t parts, uint32_t g) {
    const int32_t* p = wk.mx + wrow * wk.splits_s;
    int m = kNone;
    for (uint32_t i = g; i < parts; i += 16) {
        int x[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = p[min(i + 4 * k, parts - 1)];
        m = max(max(m, max(x[0], x[1])), max(x[2], x[3]));
    }
    m = max(m, __shfl_xor(m, 16, 64));
    m = max(m, __shfl_xor(m, 32, 64));
    return sat16i(m >> 8);
}

// A round is four steps: each wavefront makes one step's weights (its byte operands meet in LDS, two rounds deep), then
// takes a quarter of V's columns over all four, so that no sums meet and a part ends in its lanes' stores (a step a
// wavefront, all columns, the sums joined by LDS atomics: 24.5; 16 sequences of 4096 rows in int16 47 us a call for 39).
// Parts of about eight workgroups a compute unit: four 30, six 24, twelve 23.6.
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_few_kernel(Cache c, Batch bt, Attn a, Work wk, const int32_t* __restrict__ tab) {
    typedef Few<HD, I8> F;
    typedef Block<HD, I8> B;
    constexpr uint32_t NB = HD / 64, NP = I8 ? 3 : 2;          // column blocks a wavefront; byte operands of the weights
    __shared__ __attribute__((aligned(16))) int32_t stab[4096];
    __shared__ v4i ops[2][4][NP][64];
    __shared__ int64_t wsum[4][16];
    const uint32_t z = blockIdx.z;
    const Tile<kFewRows> tl(bt, a, blockIdx.x);
    const uint32_t parts = tl.parts(wk.per);
    if (!tl.on || z >= parts) return;
    stage_tab(stab, tab);
    const F f(c, bt, a, tl, blockIdx.y);
    const uint32_t beg = z * wk.per, end = min((z + 1) * wk.per, tl.nt), g = f.g, w = f.w;
    auto load = [&](uint32_t i, uint32_t (&x)[8]) {
        const uint32_t kg = tl.lo + 64 * i + 16 * g;
        uint4 s0 = make_uint4(0, 0, 0, 0), s1 = s0;
        if (f.mine && i < end && kg < bt.cap) {
            const uint4* sp = reinterpret_cast<const uint4*>(wk.sc + f.wrow * bt.cap + kg);
            s0 = sp[0];
            s1 = sp[1];
        }
        x[0] = s0.x; x[1] = s0.y; x[2] = s0.z; x[3] = s0.w;
        x[4] = s1.x; x[5] = s1.y; x[6] = s1.z; x[7] = s1.w;
    };
    v4i vh[4][NB], vl[4][I8 ? 1 : NB], es = {0, 0, 0, 0};
    auto load_v = [&](uint32_t i, const uint32_t (&id)[4]) {   // past the end: block 0, not used
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t in = (tl.lo + 64 * (i + j) + 16 * g) & (c.page - 1);
            const uint8_t *vb = f.block(id[j]), *vp = vb + B::v(c.page, 0) + (16 * NB * w + f.c16) * c.page + in;
#pragma unroll
            for (uint32_t m = 0; m < NB; m++) {
                vh[j][m] = *reinterpret_cast<const v4i*>(vp + 16 * m * c.page);
                if constexpr (!I8) vl[j][m] = *reinterpret_cast<const v4i*>(vp + (HD + 16 * m) * c.page);
            }
        }
    };
    auto load_e = [&](uint32_t i, uint32_t id) {               // the shifts of the wavefront's own step's keys
        if constexpr (I8) es = *reinterpret_cast<const v4i*>(f.block(id) + B::ve(c.page) + ((tl.lo + 64 * i + 16 * g) & (c.page - 1)));
    };
    uint32_t id[4], sw[8];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) id[j] = f.id_own(beg + j, end);
    uint32_t ido = f.id_own(beg + w, end);
    load(beg + w, sw);
    load_e(beg + w, ido);
    load_v(beg, id);
    const uint32_t m2 = twice((uint32_t)row_max(wk, f.wrow, tl.parts(wk.per_s), g)), dl2 = twice(a.smx.dlim);
    __builtin_amdgcn_s_waitcnt(0x0070);               // the TAB's copies
    __syncthreads();
    v4i acc[3][NB];
#pragma unroll
    for (uint32_t m = 0; m < NB; m++) acc[0][m] = acc[1][m] = acc[2][m] = v4i{0, 0, 0, 0};
    uint32_t sum = 0;
    for (uint32_t i = beg, buf = 0; i < end; i += 4, buf ^= 1) {
        if (i + w < end) {
            uint32_t wp[8];
            f.weights(i + w, ido, sw, m2, dl2, a.smx, stab, wp, sum);
            v4i p[NP];
            f.operands(wp, es, p);
#pragma unroll
            for (uint32_t x = 0; x < NP; x++) ops[buf][w][x][f.lane] = p[x];
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) id[j] = f.id_own(i + 4 + j, end);
        ido = f.id_own(i + 4 + w, end);
        load(i + 4 + w, sw);
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            if (i + j >= end) break;
            v4i p[NP];
#pragma unroll
            for (uint32_t x = 0; x < NP; x++) p[x] = ops[buf][j][x][f.lane];
#pragma unroll
            for (uint32_t m = 0; m < NB; m++) F::pv(vh[j][m], vl[j][I8 ? 0 : m], p, acc[0][m], acc[1][m], acc[2][m]);
        }
        if (i + 4 < end) {
            load_e(i + 4 + w, ido);
            load_v(i + 4, id);
        }
    }
    int64_t ws = sum;
    ws += (int64_t)ro::shfl64((uint64_t)ws, 16);
    ws += (int64_t)ro::shfl64((uint64_t)ws, 32);
    if (g == 0) wsum[w][f.c16] = ws;
    __syncthreads();
    const int64_t total = wsum[0][f.c16] + wsum[1][f.c16] + wsum[2][f.c16] + wsum[3][f.c16];
    const Divide quot(total, a.fp);
    int64_t* pp = wk.part + (f.wrow * wk.splits + z) * (HD + 2);
#pragma unroll
    for (uint32_t m = 0; m < NB; m++) {
        const uint32_t d = 16 * (NB * w + m) + 4 * g;
        int64_t x[4];
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) {
            // in lane 15 V's sum, below 2^30
            const int vs = I8 ? acc[0][m][r] : (int)((uint32_t)acc[0][m][r] * 256u + (uint32_t)acc[2][m][r]);
            const int64_t v = __shfl(vs, 16 * g + kFewRows, 64);
            x[r] = (int64_t)acc[0][m][r] * 65536 + (int64_t)acc[1][m][r] * 256 + acc[2][m][r] +
                   (I8 ? v * (128 * 65793) : v * 32896 + 128 * total);
        }
        if (!f.mine) continue;
        if (parts == 1) {
            store_out(a.o + (uint64_t)(tl.q0 + f.row / a.G) * a.o_ld + (uint64_t)(f.head * a.G + f.row % a.G) * HD + d, quot, x);
        } else {
            *reinterpret_cast<longlong2*>(pp + d) = make_longlong2(x[0], x[1]);
            *reinterpret_cast<longlong2*>(pp + d + 2) = make_longlong2(x[2], x[3]);
        }
    }
    if (parts > 1 && f.mine && w == 0 && g == 0) pp[HD] = total;
}

// The parts' sums of a row added and divided: a wavefront per row, loads of four parts in flight.
template <uint32_t HD>
__global__ __launch_bounds__(256) void paged_join_kernel(Batch bt, Attn a, Work wk) {
    const uint32_t lane = threadIdx.x & 63, head = blockIdx.y;
    const uint32_t at = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));   // row of (token, i)
    const uint32_t tok = at / a.G;
    if (tok >= bt.start(bt.batch)) return;
    const uint32_t b = find_le(bt.batch, tok, [&](uint32_t i) { return bt.start(i); });
    const uint32_t row = at - bt.start(b) * a.G;
    const Tile<kFewRows> tl(bt, a, (uint32_t)((uint64_t)bt.start(b) * a.G / kFewRows) + b + row / kFewRows);
    const uint32_t parts = tl.parts(wk.per);
    if (!tl.on || parts == 1) return;
    const int64_t* pp = wk.part + ((uint64_t)head * bt.tokens * a.G + at) * wk.splits * (HD + 2);
    int64_t x[HD / 64], S = 0;
#pragma unroll
    for (uint32_t k = 0; k < HD / 64; k++) x[k] = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < parts; i++) {
        const int64_t* p = pp + (uint64_t)i * (HD + 2);
#pragma unroll
        for (uint32_t k = 0; k < HD / 64; k++) x[k] += p[lane * (HD / 64) + k];
        S += p[HD];
    }
    int16_t* op = a.o + (uint64_t)tok * a.o_ld + (uint64_t)(head * a.G + at % a.G) * HD + lane * (HD / 64);
    const Divide q(S, a.fp);
#pragma unroll
    for (uint32_t k = 0; k < HD / 64; k++) op[k] = (int16_t)q(x[k]);
}

// ---------------------------------------------------------------- attention of many rows
// Tiles of 64 QB rows, 16 QB a wavefront; the keys go by in steps of 64 through two LDS stages that all four
// wavefronts read, copied straight into LDS a step ahead.  One kernel for the rows' maxima (q.K^T alone), one for the
// weights and P.V with the scores computed again: a weight needs the final maximum (its shift drops bits, so a sum
// over another maximum cannot be rescaled), and the scores of many rows are dearer to keep than to compute twice.
//
// Two wavefronts a SIMD (the accumulators' registers; the second kernel takes all 256 and spills 18 of them with int16
// rows of 64, 12 with int16 rows of 128, 2 with int8 rows of 64, and 42 .. 50 SGPRs).  A prompt of 4096 tokens of 15 + 5
// heads of 64 takes 45 us for the maxima, 121 for the weights and P.V and 14 for the join of the pieces; the byte products
// of the first two are 13 and 26 at the matrix rate.  What the 121 lose, a part taken out at a time: the exponentials'
// arithmetic 31, their table reads 9, the sums of the score limbs 10, the weights' sum 4, the weights' bytes 3, V's sums 3,
// one of P.V's four products 6, the copies into LDS 5: 71 in all, the other seven products and the spilled registers not
// among them; they have not been taken apart.  Tiles of 64 rows at three wavefronts a SIMD: 123.  256 tokens on 4096 rows:
// 11 + 27 + 9, half of it the pieces' first loads and 33 MB of partial sums.
//
// LDS layouts.  K: row = key, its 16-byte chunks XORed by the key's place so that the 16 rows of a fragment (keys
// 16 a + 4 kb + i) fall on 16 bank groups.  V: [plane][16-key group][d][16 bytes], a fragment's lanes consecutive.
// Wavefront w copies the step's 16-key group w, of one page: a direct copy moves 1 KiB, lane l to 16 l (16 key rows,
// 8 at 128 d; or 64 d).
template <uint32_t HD, bool I8, bool V>
struct Stage {
    static constexpr uint32_t KBYTES = (I8 ? 1 : 2) * 64 * HD;
    static constexpr uint32_t TERM = V ? 2 * KBYTES : KBYTES, BYTES = TERM + 256 + (I8 ? 128 : 0);   // K, V, terms, shifts
};

template <uint32_t HD, bool I8, uint32_t QB, bool V>
struct Rows {
    static constexpr uint32_t KS = HD / 64, NP = I8 ? 1 : 2, R = 64 * QB;
    typedef Block<HD, I8> B;
    typedef Stage<HD, I8, V> S;
    const Cache& c;
    const Batch& bt;
    const Tile<R>& tl;
    uint32_t head, lane, c16, g, w;
    v4i qh[QB][KS], ql[QB][KS];
    int qterm[QB];
    uint32_t vend[QB], vbeg[QB];

    __device__ __forceinline__ Rows(const Cache& c_, const Batch& bt_, const Attn& a, const Tile<R>& tl_, uint32_t head_)
        : c(c_), bt(bt_), tl(tl_), head(head_) {
        lane = threadIdx.x & 63;
        c16 = lane & 15;
        g = lane >> 4;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    }
    __device__ __forceinline__ void queries(const Attn& a) {
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
            const uint32_t row = row_of(qb), rr = min(row, tl.rows - 1), tok = rr / a.G;
            vend[qb] = row < tl.rows ? tl.seen(bt, tok) : 0u;
            vbeg[qb] = tl.begin(a, tok);
            const int16_t* qp = a.q + (uint64_t)(tl.q0 + tok) * a.q_ld + (uint64_t)(head * a.G + rr % a.G) * HD + 16 * g;
            int qs = 0;
#pragma unroll
            for (uint32_t s = 0; s < KS; s++) limbs16(qp + 64 * s, qh[qb][s], ql[qb][s], qs);
            qs += __shfl_xor(qs, 16, 64);
            qs += __shfl_xor(qs, 32, 64);
            qterm[qb] = I8 ? 0 : 128 * qs;
        }
    }
    __device__ __forceinline__ uint32_t row_of(uint32_t qb) const { return tl.row0 + 16 * QB * w + 16 * qb + c16; }
    // the page ids of step i's four 16-key groups, one a lane group (~0: no page)
    __device__ __forceinline__ uint32_t ids(uint32_t i, uint32_t end) const {
        const uint32_t key = tl.lo + 64 * i + 16 * g;
        const uint32_t id = i < end && key < bt.cap ? (uint32_t)tl.tb[key >> c.lg] : ~0u;
        return id < c.pages ? id : ~0u;
    }
    static __device__ __forceinline__ void copy(const uint8_t* src, uint8_t* dst) {
        __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
    }
    __device__ __forceinline__ void stage(uint8_t* sm, uint32_t i, uint32_t id4) const {
        const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)id4, 16 * w);
        const uint8_t* blk = c.data + ((uint64_t)(id == ~0u ? 0u : id) * c.kv + head) * c.block;
        const uint32_t in = (tl.lo + 64 * i + 16 * w) & (c.page - 1);
        constexpr uint32_t CH = HD / 16, RPC = 64 / CH;               // chunks a row, rows a copy
#pragma unroll
        for (uint32_t pl = 0; pl < NP; pl++)
#pragma unroll
            for (uint32_t s = 0; s < KS; s++) {
                const uint32_t row = RPC * s + lane / CH, f = KS == 1 ? w : ((row >> 1) & 1) | w << 1;
                copy(blk + B::k(c.page, pl) + in * HD + row * HD + 16 * ((lane % CH) ^ f), sm + pl * 64 * HD + (16 * w + RPC * s) * HD);
            }
        if constexpr (V) {
#pragma unroll
            for (uint32_t pl = 0; pl < NP; pl++)
#pragma unroll
                for (uint32_t s = 0; s < KS; s++)
                    copy(blk + B::v(c.page, pl) + in + (64 * s + lane) * c.page, sm + S::KBYTES + ((pl * 4 + w) * HD + 64 * s) * 16);
        }
        if (lane < 4) copy(blk + B::term(c.page) + 4 * in + 16 * lane, sm + S::TERM + 64 * w);
        if constexpr (I8) {
            if (lane == 0) {
                copy(blk + B::ke(c.page) + in, sm + S::TERM + 256 + 16 * w);
                if constexpr (V) copy(blk + B::ve(c.page) + in, sm + S::TERM + 320 + 16 * w);
            }
        }
    }
    // the K operands of keys 16 g + 4 kb + r, r < 4, their terms and shifts
    struct Frag {
        v4i kh[KS], kl[KS], term;
        uint32_t es;
    };
    __device__ __forceinline__ void load(const uint8_t* sm, uint32_t kb, Frag& f) const {
        const uint32_t row = 16 * (c16 >> 2) + 4 * kb + (c16 & 3);
        f.term = *reinterpret_cast<const v4i*>(sm + S::TERM + 4 * (16 * g + 4 * kb));
#pragma unroll
        for (uint32_t s = 0; s < KS; s++) {
            const uint32_t x = KS == 1 ? c16 >> 2 : ((c16 >> 1) & 1) | (c16 >> 2) << 1;
            const uint8_t* kp = sm + row * HD + 16 * ((4 * s + g) ^ x);
            f.kh[s] = *reinterpret_cast<const v4i*>(kp);
            if constexpr (!I8) f.kl[s] = *reinterpret_cast<const v4i*>(kp + 64 * HD);
            else f.kl[s] = v4i{0, 0, 0, 0};
        }
        if constexpr (I8) f.es = *reinterpret_cast<const uint32_t*>(sm + S::TERM + 256 + 16 * g + 4 * kb);
        else f.es = 0;
    }
    __device__ __forceinline__ void products(const Frag& f, uint32_t qb, v4i& hh, v4i& mid, v4i& ll) const {
        hh = mid = v4i{0, 0, 0, 0};
        ll = f.term;
#pragma unroll
        for (uint32_t s = 0; s < KS; s++) qk<I8>(f.kh[s], f.kl[s], qh[qb][s], ql[qb][s], hh, mid, ll);
    }
    // whether every row sees all 64 keys of a step, its pages all there
    __device__ __forceinline__ bool whole(uint32_t i, uint32_t id4) const {
        const uint32_t k0 = tl.lo + 64 * i;
        return k0 >= tl.all_lo && k0 + 64 <= tl.all_hi && __ballot(id4 == ~0u) == 0;
    }
    // body(stage, step, ids) for the steps [i, end), two stages deep; an odd count is made even by a step without pages
    // (a loop that may end between its halves has the accumulators moved from registers to registers)
    // id0, id1: ids of the first two steps, loaded by the caller ahead of the queries
    template <class F>
    __device__ __forceinline__ void run(uint8_t* sm0, uint8_t* sm1, uint32_t i, uint32_t end, uint32_t id0, uint32_t id1,
                                        F body) const {
        if (i >= end) return;
        stage(sm0, i, id0);
        for (; i < end; i += 2) {
            __builtin_amdgcn_s_waitcnt(0x0070);        // this wavefront's copies
            __syncthreads();                           // every wavefront's; the other stage read
            const uint32_t id2 = ids(i + 2, end);
            stage(sm1, i + 1, id1);
            body(sm0, i, id0);
            __builtin_amdgcn_s_waitcnt(0x0070);
            __syncthreads();
            const uint32_t id3 = ids(i + 3, end);
            if (i + 2 < end) stage(sm0, i + 2, id2);
            body(sm1, i + 1, id1);
            id0 = id2;
            id1 = id3;
        }
    }
};

// ---- the work of many rows.  The 64-key steps of all tiles, one KV head after the other, are one list that is divided
// evenly over the workgroups (shares): a causal prompt's tiles differ by the length of the prompt, and a share per tile
// leaves the chip half empty behind the long ones.  A share covers the end of a tile, whole tiles, and the beginning of
// one; sums of a tile that crosses shares are joined by a last kernel.  Up to kPlan tiles of up to 64 sequences each
// workgroup sums the tiles' steps for itself (1 us of LDS work in place of a launch and its wait, 5.5 us); more have
// them from a kernel of their own.
constexpr uint32_t kPlan = 256;
struct Queue {
    uint32_t* cum;                         // [slots + 1] steps before each tile of a KV head; null: each workgroup's own
    int32_t* mx;                           // [max_shares + KV heads slots][R] raw maxima, a piece's at share + tile
    int64_t* part;                         // [shares][2][R HD + R], in the lanes' order
    uint32_t slots, max_shares, shares;    // shares at most, both multiples of 8
};
constexpr uint32_t kMaxMin = 4, kRowsMin = 4;   // steps of a share, at least: 6, 8, 12 for 4 in 256 tokens on 4096 rows
                                                // 52, 49, 55 us for 47

template <uint32_t R>
struct PlanLds {                           // one workgroup's
    typename Tile<R>::Seqs seqs[64];
    uint32_t cum[kPlan + 1], wave[4];
};

template <uint32_t R>
__device__ __forceinline__ uint32_t wave_scan(uint32_t n) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint32_t x = (uint32_t)__shfl_up((int)n, o, 64);
        n += lane >= o ? x : 0u;
    }
    return n;
}

// cum of at most kPlan slots by 256 threads; the sequences for Tile (every wavefront writes the same, and reads its own)
template <uint32_t R>
__device__ __forceinline__ void plan(PlanLds<R>& sm, const Batch& bt, const Attn& a, const Queue& q) {
    const uint32_t t = threadIdx.x, lane = t & 63, w = t >> 6;
    sm.seqs[lane] = typename Tile<R>::Seqs(bt);
    if (q.cum != nullptr) return;
    const uint32_t n = t < q.slots ? Tile<R>::lane_steps(bt, a, t, sm.seqs) : 0u, sum = wave_scan<R>(n);
    if (lane == 63) sm.wave[w] = sum;
    __syncthreads();
    uint32_t off = sum;
    for (uint32_t i = 0; i < w; i++) off += sm.wave[i];
    sm.cum[t + 1] = off;
    if (t == 0) sm.cum[0] = 0;
    __syncthreads();
}

// The shares of at most `most`
template <uint32_t R>
struct Shares {
    const uint32_t* cum;
    const PlanLds<R>& sm;
    uint64_t all;                          // positions of every KV head
    uint32_t slots, head, n;               // tiles and positions of one, shares
    __device__ __forceinline__ Shares(const Queue& q, const PlanLds<R>& sm_, uint32_t kv, uint32_t most, uint32_t least)
        : cum(q.cum), sm(sm_), slots(q.slots) {
        head = __builtin_amdgcn_readfirstlane(at(slots));
        all = (uint64_t)head * kv;
        n = all ? (uint32_t)min((uint64_t)most, max(all / least, (uint64_t)1)) : 0u;
    }
    __device__ __forceinline__ uint32_t at(uint32_t slot) const { return cum ? cum[slot] : sm.cum[slot]; }
    // the last slot with cum <= y, its cum and the next one's: a round of loads, one more from 64 and from 4032 slots on
    __device__ __forceinline__ uint32_t find(uint32_t y, uint32_t& c0, uint32_t& c1) const {
        const uint32_t lane = threadIdx.x & 63, stride = slots / 64 + 1;
        uint32_t v = at(min(lane * stride, slots)), base = 0;
        uint32_t k = max((uint32_t)__popcll(__ballot(lane * stride < slots && v <= y)), 1u) - 1;
        if (stride > 1) {
            base = k * stride;
            uint32_t m = min(stride, slots - base);
            if (stride > 63) {
                base += find_le(m, y, [&](uint32_t i) { return cum[base + i]; });
                m = 1;
            }
            v = at(min(base + lane, slots));
            k = max((uint32_t)__popcll(__ballot(lane < m && v <= y)), 1u) - 1;
        }
        c0 = (uint32_t)__builtin_amdgcn_readlane((int)v, k);
        c1 = (uint32_t)__builtin_amdgcn_readlane((int)v, k + 1);
        return base + k;
    }
    __device__ __forceinline__ uint64_t first(uint32_t i) const { return (uint64_t)i * all / n; }
    __device__ __forceinline__ uint32_t owner(uint64_t pos) const { return (uint32_t)(((pos + 1) * n - 1) / all); }
    // workgroups are dealt round-robin to the 8 XCDs: each takes a contiguous run of the list (its keys in its L2);
    // ~0: none (a grid of a multiple of 8 and of n or more)
    __device__ __forceinline__ uint32_t order(uint32_t i) const {
        const uint32_t lo = (uint32_t)((uint64_t)(i & 7) * n >> 3), hi = (uint32_t)((uint64_t)((i & 7) + 1) * n >> 3);
        return lo + (i >> 3) < hi ? lo + (i >> 3) : ~0u;
    }
};

// The part of a tile from position `at` of the list to `stop` at most: a tile has kTileCost positions, then its steps
struct Piece {
    uint32_t head, slot, beg, end, steps;  // steps [beg, end) of the tile's
    uint64_t next;                         // the list's position behind the piece
    uint64_t tile;                         // the position of the tile's first step
    bool whole;
    // a piece's maxima: along the list either the share or the tile grows from piece to piece
    static __device__ __forceinline__ uint64_t maxima(const Queue& q, uint32_t share, uint32_t head, uint32_t slot) {
        return share + (uint64_t)head * q.slots + slot;
    }
    template <uint32_t R>
    __device__ __forceinline__ Piece(const Shares<R>& sh, uint64_t at, uint64_t stop) {
        head = (uint32_t)(at / sh.head);
        uint32_t c0, c1;
        slot = sh.find((uint32_t)(at - (uint64_t)head * sh.head), c0, c1);
        steps = c1 - c0 - kTileCost;
        tile = (uint64_t)head * sh.head + c0 + kTileCost;
        next = min(stop, tile + steps);
        beg = (uint32_t)(max(at, tile) - tile);
        end = (uint32_t)(max(next, tile) - tile);
        whole = beg == 0 && end == steps;
    }
};

template <uint32_t R>
__global__ __launch_bounds__(1024) void paged_plan_kernel(Batch bt, Attn a, Queue qu) {
    const uint32_t t = threadIdx.x, lane = t & 63, w = t >> 6;
    __shared__ uint32_t wave[16];
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < qu.slots; s0 += 1024) {
        const uint32_t n = s0 + t < qu.slots ? Tile<R>::lane_steps(bt, a, s0 + t, nullptr) : 0u, sum = wave_scan<R>(n);
        if (lane == 63) wave[w] = sum;
        __syncthreads();
        uint32_t off = before, all = 0;
        for (uint32_t i = 0; i < 16; i++) {
            off += i < w ? wave[i] : 0u;
            all += wave[i];
        }
        if (s0 + t < qu.slots) qu.cum[s0 + t] = off + sum - n;
        before += all;
        __syncthreads();
    }
    if (t == 0) qu.cum[qu.slots] = before;
}

template <uint32_t HD, bool I8, uint32_t QB>
__global__ __launch_bounds__(256, 2) void paged_max_kernel(Cache c, Batch bt, Attn a, Queue qu) {
    typedef Rows<HD, I8, QB, false> RW;
    __shared__ __attribute__((aligned(1024))) uint8_t sm0[RW::S::BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t sm1[RW::S::BYTES];
    __shared__ PlanLds<RW::R> spl;
    plan(spl, bt, a, qu);
    const Shares<RW::R> sh(qu, spl, c.kv, qu.max_shares, kMaxMin);
    const uint32_t id = sh.order(blockIdx.x);
    if (id == ~0u) return;
    for (uint64_t at = sh.first(id), stop = sh.first(id + 1); at < stop;) {
        const Piece pc(sh, at, stop);
        at = pc.next;
        if (pc.beg == pc.end) continue;            // a tile's first positions alone
        const uint32_t head = pc.head;
        const Tile<RW::R> tl(bt, a, pc.slot, spl.seqs[threadIdx.x & 63]);
        if (!tl.on) continue;
        RW rw(c, bt, a, tl, head);
        int mx[QB];
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) mx[qb] = kNone;
        const uint32_t id0 = rw.ids(pc.beg, pc.end), id1 = rw.ids(pc.beg + 1, pc.end);
        rw.queries(a);
        rw.run(sm0, sm1, pc.beg, pc.end, id0, id1, [&](const uint8_t* sm, uint32_t i, uint32_t ids) {
            const uint32_t kg = tl.lo + 64 * i + 16 * rw.g;
            constexpr uint32_t NB = 4 * QB;
            auto maxima = [&](auto masked) {
                typename RW::Frag f;
                v4i h[2], md[2], l[2];
                uint32_t es[2];
                rw.load(sm, 0, f);
#pragma unroll
                for (uint32_t j = 0; j < NB + 1; j++) {
                    if (j < NB) {
                        rw.products(f, j % QB, h[j & 1], md[j & 1], l[j & 1]);
                        es[j & 1] = f.es;
                        if (j % QB == QB - 1 && j / QB + 1 < 4) rw.load(sm, j / QB + 1, f);
                    }
                    if (j >= 1) {
                        const uint32_t y = j - 1, qb = y % QB;
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++) {
                            int z = raw_sum<I8>(h[y & 1][r], md[y & 1][r], l[y & 1][r], es[y & 1], r, rw.qterm[qb]);
                            if constexpr (masked) {
                                const uint32_t key = kg + 4 * (y / QB) + r;
                                z = ids != ~0u && key >= rw.vbeg[qb] && key < rw.vend[qb] ? z : kNone;
                            }
                            mx[qb] = max(mx[qb], z);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if (rw.whole(i, ids)) maxima(std::false_type{});
            else maxima(std::true_type{});
        });
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
            int m = mx[qb];
            m = max(m, __shfl_xor(m, 16, 64));
            m = max(m, __shfl_xor(m, 32, 64));
            if (rw.g == 0) qu.mx[Piece::maxima(qu, id, head, pc.slot) * RW::R + rw.row_of(qb) - tl.row0] = m;
        }
    }
}

template <uint32_t HD, bool I8, uint32_t QB>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(Cache c, Batch bt, Attn a, Queue qu, const int32_t* __restrict__ tab) {
    constexpr uint32_t DB = HD / 16, NP = I8 ? 1 : 2, MW = DB / 4;
    typedef Rows<HD, I8, QB, true> RW;
    typedef typename RW::S S;
    __shared__ __attribute__((aligned(1024))) uint8_t sm0[S::BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t sm1[S::BYTES];
    // int16 rows of 128 take 66 KB of stages: with TAB in 16 bits two workgroups fit a CU
    constexpr bool HALF = HD == 128 && !I8;
    __shared__ __attribute__((aligned(16))) int32_t stab[HALF ? 2048 : 4096];
    __shared__ int32_t vsum[NP][HD];
    __shared__ PlanLds<RW::R> spl;
    plan(spl, bt, a, qu);
    const Shares<RW::R> sh(qu, spl, c.kv, qu.shares, kRowsMin);
    const uint32_t id = sh.order(blockIdx.x);
    if (id == ~0u) return;
    if constexpr (HALF) stage_tab_half(stab, tab);
    else stage_tab(stab, tab);
    for (uint64_t at = sh.first(id), stop = sh.first(id + 1); at < stop;) {
        const Piece pc(sh, at, stop);
        at = pc.next;
        if (pc.beg == pc.end) continue;            // a tile's first positions alone
        const uint32_t head = pc.head;
        const Tile<RW::R> tl(bt, a, pc.slot, spl.seqs[threadIdx.x & 63]);
        if (!tl.on) continue;
        RW rw(c, bt, a, tl, head);
        int64_t* part = qu.part + (uint64_t)(2 * id + (pc.beg == 0 ? 1 : 0)) * (RW::R * HD + RW::R);
        const uint32_t g = rw.g, c16 = rw.c16, w = rw.w;
        const v4i zero = {0, 0, 0, 0}, ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
        uint32_t id0 = rw.ids(pc.beg, pc.end), id1 = rw.ids(pc.beg + 1, pc.end);
        uint32_t m2[QB];
        const uint32_t dl2 = twice(a.smx.dlim);
        int64_t total[QB];
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
            m2[qb] = (uint32_t)kNone;
            total[qb] = 0;
        }
        {                                          // the tile's maxima: its pieces' in the list of paged_max_kernel
            const Shares<RW::R> shm(qu, spl, c.kv, qu.max_shares, kMaxMin);
            const uint32_t i0 = shm.owner(pc.tile), i1 = shm.owner(pc.tile + pc.steps - 1);
#pragma unroll 4
            for (uint32_t i = i0 + g; i <= i1; i += 4) {
                const int32_t* mp = qu.mx + Piece::maxima(qu, i, head, pc.slot) * RW::R + rw.row_of(0) - tl.row0;
#pragma unroll
                for (uint32_t qb = 0; qb < QB; qb++) m2[qb] = (uint32_t)max((int)m2[qb], mp[16 * qb]);
            }
        }
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
            int m = max((int)m2[qb], __shfl_xor((int)m2[qb], 16, 64));
            m = max(m, __shfl_xor(m, 32, 64));
            m2[qb] = twice((uint32_t)sat16i(m >> 8));
        }
        rw.queries(a);
        // at most kMaxPart keys in the int32 limb sums (a product is below 2^14, two a key in the middle ones): a longer
        // piece adds to its partial sums
        for (uint32_t beg = pc.beg; beg < pc.end;) {
        const uint32_t end = min(pc.end, beg + kMaxPart / 64);
        v4i acc[3][DB][QB], vs[NP][MW];
        uint32_t wsum[QB];                         // the lane's keys' weights: below 2^16 * 16 * kMaxPart / 64
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
#pragma unroll
            for (uint32_t m = 0; m < DB; m++) acc[0][m][qb] = acc[1][m][qb] = acc[2][m][qb] = zero;
            wsum[qb] = 0;
        }
#pragma unroll
        for (uint32_t m = 0; m < MW; m++) vs[0][m] = vs[NP - 1][m] = zero;
        rw.run(sm0, sm1, beg, end, id0, id1, [&](const uint8_t* sm, uint32_t i, uint32_t ids) {
            const uint32_t kg = tl.lo + 64 * i + 16 * g;
            v4i p[QB][I8 ? 3 : 2];
            // the step's blocks (16 keys x 16 rows) in three stages, a block's products under the exponentials of the one
            // before and the packing of the one before that
            constexpr uint32_t NB = 4 * QB;
            auto weights = [&](auto masked) {
                typename RW::Frag f;
                v4i h[2], md[2], l[2];
                uint32_t es[2];
                Exp2 x[2][2];
                rw.load(sm, 0, f);
#pragma unroll
                for (uint32_t j = 0; j < NB + 2; j++) {
                    if (j < NB) {
                        rw.products(f, j % QB, h[j & 1], md[j & 1], l[j & 1]);
                        es[j & 1] = f.es;
                        if (j % QB == QB - 1 && j / QB + 1 < 4) rw.load(sm, j / QB + 1, f);
                    }
                    if (j >= 1 && j <= NB) {
                        const uint32_t y = j - 1, qb = y % QB;
                        int z[4];
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            z[r] = raw_sum<I8>(h[y & 1][r], md[y & 1][r], l[y & 1][r], es[y & 1], r, rw.qterm[qb]) >> 8;
                        x[y & 1][0] = exps<HALF>(z[0], z[1], m2[qb], dl2, a.smx, stab);
                        x[y & 1][1] = exps<HALF>(z[2], z[3], m2[qb], dl2, a.smx, stab);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (j >= 2) {
                        const uint32_t y = j - 2, kb = y / QB, qb = y % QB;
                        const Exp2 *e = x[y & 1];
                        uint32_t v[4] = {e[0].e0(), e[0].e1(), e[1].e0(), e[1].e1()};
                        if constexpr (masked) {
#pragma unroll
                            for (uint32_t r = 0; r < 4; r++) {
                                const uint32_t key = kg + 4 * kb + r;
                                v[r] = ids != ~0u && key >= rw.vbeg[qb] && key < rw.vend[qb] ? v[r] : 0u;
                            }
                        }
                        const uint32_t w01 = pair16(v[0], v[1]), w23 = pair16(v[2], v[3]);
                        wsum[qb] = add16(w01, add16(w23, wsum[qb]));
                        uint32_t ve = 0;
                        if constexpr (I8) ve = *reinterpret_cast<const uint32_t*>(sm + S::TERM + 320 + 16 * g + 4 * kb);
                        weight_bytes<I8>(w01, w23, ve, p[qb], kb);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if (rw.whole(i, ids)) weights(std::false_type{});
            else weights(std::true_type{});
#pragma unroll
            for (uint32_t m = 0; m < DB; m++) {
                const uint8_t* vp = sm + S::KBYTES + (g * HD + 16 * m + c16) * 16;
                const v4i vh = *reinterpret_cast<const v4i*>(vp);
                v4i vl = zero;
                if constexpr (!I8) vl = *reinterpret_cast<const v4i*>(vp + 64 * HD);
#pragma unroll
                for (uint32_t qb = 0; qb < QB; qb++) {
                    if constexpr (I8) {
                        acc[0][m][qb] = mfma(vh, p[qb][I8 ? 2 : 0], acc[0][m][qb]);
                        acc[1][m][qb] = mfma(vh, p[qb][1], acc[1][m][qb]);
                        acc[2][m][qb] = mfma(vh, p[qb][0], acc[2][m][qb]);
                    } else {
                        acc[0][m][qb] = mfma(vh, p[qb][1], acc[0][m][qb]);
                        acc[1][m][qb] = mfma(vh, p[qb][0], acc[1][m][qb]);
                        acc[2][m][qb] = mfma(vl, p[qb][0], acc[2][m][qb]);
                        acc[1][m][qb] = mfma(vl, p[qb][1], acc[1][m][qb]);
                    }
                }
            }
#pragma unroll
            for (uint32_t m = 0; m < MW; m++) {    // V's sums: each wavefront its share of d
                const uint8_t* vp = sm + S::KBYTES + (g * HD + 16 * (w + 4 * m) + c16) * 16;
                vs[0][m] = mfma(*reinterpret_cast<const v4i*>(vp), ones, vs[0][m]);
                if constexpr (!I8) vs[NP - 1][m] = mfma(*reinterpret_cast<const v4i*>(vp + 64 * HD), ones, vs[NP - 1][m]);
            }
        });
        if (c16 == 0) {
#pragma unroll
            for (uint32_t m = 0; m < MW; m++)
#pragma unroll
                for (uint32_t pl = 0; pl < NP; pl++)
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) vsum[pl][16 * (w + 4 * m) + 4 * g + r] = vs[pl][m][r];
        }
        __syncthreads();
        const bool last = end == pc.end;
#pragma unroll
        for (uint32_t qb = 0; qb < QB; qb++) {
            int64_t sum = wsum[qb];
            sum += (int64_t)ro::shfl64((uint64_t)sum, 16);
            sum += (int64_t)ro::shfl64((uint64_t)sum, 32);
            total[qb] += sum;
            const uint32_t row = rw.row_of(qb);
            const bool on = row < tl.rows;
            int16_t* op = a.o + (uint64_t)(tl.q0 + row / a.G) * a.o_ld + (uint64_t)(head * a.G + row % a.G) * HD;
            const Divide quot(total[qb], a.fp);
#pragma unroll
            for (uint32_t m = 0; m < DB; m++) {
                int64_t x[4];
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    const uint32_t d = 16 * m + 4 * g + r;
                    x[r] = whole_sum<I8>(acc[0][m][qb][r], acc[1][m][qb][r], acc[2][m][qb][r], vsum[0][d], vsum[NP - 1][d], sum);
                }
                longlong2* pp = reinterpret_cast<longlong2*>(part) + (((w * QB + qb) * DB + m) * 2) * 64 + rw.lane;
                if (beg != pc.beg) {
                    const longlong2 u = pp[0], v = pp[64];
                    x[0] += u.x;
                    x[1] += u.y;
                    x[2] += v.x;
                    x[3] += v.y;
                }
                if (!last || !pc.whole) {
                    pp[0] = make_longlong2(x[0], x[1]);
                    pp[64] = make_longlong2(x[2], x[3]);
                } else if (on) {
                    store_out(op + 16 * m + 4 * g, quot, x);
                }
            }
            if (last && !pc.whole && g == 0) part[RW::R * HD + 16 * (w * QB + qb) + c16] = total[qb];
        }
        beg = end;
        if (beg < pc.end) {
            id0 = rw.ids(beg, pc.end);
            id1 = rw.ids(beg + 1, pc.end);
        }
        }
    }
}

// The pieces' sums of a tile added and divided, in the lanes' order of paged_rows_kernel: a workgroup per tile, 64 rows
// and 16 columns; loads of four pieces in flight.
template <uint32_t HD, uint32_t QB>
__global__ __launch_bounds__(256) void paged_rows_join_kernel(Cache c, Batch bt, Attn a, Queue qu) {
    constexpr uint32_t DB = HD / 16, R = 64 * QB;
    __shared__ PlanLds<R> spl;
    plan(spl, bt, a, qu);
    const Shares<R> sh(qu, spl, c.kv, qu.shares, kRowsMin);
    const uint32_t slot = blockIdx.x, head = blockIdx.y, m = blockIdx.z % DB, qb = blockIdx.z / DB;
    const uint32_t c0 = __builtin_amdgcn_readfirstlane(sh.at(slot)), c1 = __builtin_amdgcn_readfirstlane(sh.at(slot + 1));
    if (c0 == c1) return;
    const uint64_t tile = (uint64_t)head * sh.head + c0 + kTileCost;
    const uint32_t i0 = sh.owner(tile), i1 = sh.owner(tile + (c1 - c0 - kTileCost) - 1);
    if (i0 == i1) return;                      // one piece: written
    const uint32_t lane = threadIdx.x & 63, c16 = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Tile<R> tl(bt, a, slot, spl.seqs[lane]);
    const uint32_t wq = w * QB + qb, row = tl.row0 + 16 * wq + c16;
    if (tl.row0 + 16 * wq >= tl.rows) return;
    int64_t x[4] = {0, 0, 0, 0}, S = 0;
#pragma unroll 4
    for (uint32_t i = i0; i <= i1; i++) {
        const int64_t* p = qu.part + (uint64_t)(2 * i + (i == i0 ? 1 : 0)) * (R * HD + R);
        const longlong2* pp = reinterpret_cast<const longlong2*>(p) + (wq * DB + m) * 128 + lane;
        const longlong2 u = pp[0], v = pp[64];
        S += p[R * HD + 16 * wq + c16];
        x[0] += u.x;
        x[1] += u.y;
        x[2] += v.x;
        x[3] += v.y;
    }
    if (row >= tl.rows) return;
    const Divide quot(S, a.fp);
    store_out(a.o + (uint64_t)(tl.q0 + row / a.G) * a.o_ld + (uint64_t)(head * a.G + row % a.G) * HD + 16 * m + 4 * g, quot, x);
}

// ---------------------------------------------------------------- the host's checks
constexpr uint32_t kMaxKeys = 1u << 20;
constexpr uint64_t kMaxScores = 1ull << 28;    // bytes of scores that a call keeps

int view(const cm_paged_cache* cache, const cm_paged_batch* batch, Cache* c, Batch* b) {
    if (cache == nullptr || batch == nullptr) return fail(CM_EINVAL, "paged: a null cache or batch");
    const cm_paged_cache& k = *cache;
    if (k.head_dim != 64 && k.head_dim != 128) return fail(CM_EINVAL, "paged: head_dim %u (64 or 128)", k.head_dim);
    if (k.page < 16 || k.page > 4096 || (k.page & (k.page - 1)))
        return fail(CM_EINVAL, "paged: pages of %u rows (a power of two, 16 .. 4096)", k.page);
    if (k.pages == 0 || k.pages > 0x7FFFFFFFu || k.kv_heads == 0 || k.kv_heads > 1024)
        return fail(CM_EINVAL, "paged: %u pages of %u heads", k.pages, k.kv_heads);
    if (k.int8 > 1) return fail(CM_EINVAL, "paged: int8 %u", k.int8);
    if (batch->batch > (1u << 20) || batch->tokens > (1u << 24))
        return fail(CM_EINVAL, "paged: %u sequences, %u tokens", batch->batch, batch->tokens);
    if (batch->max_pages == 0 || (uint64_t)batch->max_pages * k.page > kMaxKeys)
        return fail(CM_EINVAL, "paged: %u pages of %u rows a sequence (1 .. 2^20 rows)", batch->max_pages, k.page);
    if (k.data == nullptr || batch->q_start == nullptr || batch->kv_len == nullptr || batch->table == nullptr)
        return fail(CM_EINVAL, "paged: a null pool, q_start, kv_len or table");
    if (!aligned16(k.data)) return fail(CM_EALIGN, "paged: the pool must be 16-byte aligned");
    *c = Cache{static_cast<uint8_t*>(k.data), block_bytes(k.page, k.head_dim, k.int8 != 0), k.pages, k.page,
               (uint32_t)__builtin_ctz(k.page), k.kv_heads};
    *b = Batch{batch->q_start, batch->kv_len, batch->table, batch->batch, batch->tokens, batch->max_pages,
               batch->max_pages * k.page, batch->table_ld};
    return CM_OK;
}

int run_prep(const cm_paged_cache* cache, const cm_paged_batch* batch, const cm_paged_prep_args* args, hipStream_t s) {
    Cache c;
    Batch b;
    int rc = view(cache, batch, &c, &b);
    if (rc) return rc;
    if (args == nullptr) return fail(CM_EINVAL, "paged prep: null arguments");
    const cm_paged_prep_args& p = *args;
    if (p.heads == 0 || p.heads > 4096) return fail(CM_EINVAL, "paged prep: %u heads", p.heads);
    if (b.batch == 0 || b.tokens == 0) return CM_OK;
    if (p.q == nullptr || p.k == nullptr || p.v == nullptr || p.qr == nullptr || p.rope == nullptr ||
        p.rope_q == nullptr || p.rope_k == nullptr)
        return fail(CM_EINVAL, "paged prep: a null operand, table or rotation parameter block");
    if (p.rotary == 0 || p.rotary % 16 || p.rotary > cache->head_dim || p.rope_rows == 0)
        return fail(CM_EINVAL, "paged prep: %u rotated columns of %u (a multiple of 16), %u table rows", p.rotary,
                    cache->head_dim, p.rope_rows);
    if (p.eps_q < 0 || p.eps_k < 0 || p.eps_q > ((int64_t)1 << 61) || p.eps_k > ((int64_t)1 << 61))
        return fail(CM_EINVAL, "paged prep: eps outside 0 .. 2^61");
    if (!aligned16(p.q) || !aligned16(p.k) || !aligned16(p.v) || !aligned16(p.qr) || !aligned16(p.rope) ||
        !aligned16(p.rope_q) || !aligned16(p.rope_k) || !aligned16(p.norm_q) || !aligned16(p.norm_k) ||
        ((p.q_ld | p.k_ld | p.v_ld | p.qr_ld) & 7))
        return fail(CM_EALIGN, "paged prep: rows, tables and parameter blocks must be 16-byte aligned");
    const uint64_t qw = (uint64_t)p.heads * cache->head_dim, kw = (uint64_t)c.kv * cache->head_dim;
    if (b.tokens > 1 && (p.q_ld < qw || p.qr_ld < qw || p.k_ld < kw || p.v_ld < kw))
        return fail(CM_EINVAL, "paged prep: rows of %llu and %llu columns overlap at their strides",
                    (unsigned long long)qw, (unsigned long long)kw);
    DeviceState* st;
    if ((rc = state(&st))) return rc;
    const Prep a{p.q, p.k, p.v, p.qr, p.q_ld, p.k_ld, p.v_ld, p.qr_ld, p.heads, p.rope_rows, p.rotary, p.interleaved,
                 p.rope, static_cast<const uint8_t*>(p.rope_q), static_cast<const uint8_t*>(p.rope_k),
                 static_cast<const uint8_t*>(p.norm_q), static_cast<const uint8_t*>(p.norm_k), p.rope_q_cols,
                 p.rope_k_cols, p.eps_q, p.eps_k, st->ro_tables};
    // q and k: a pass of a token a wavefront until those are 4096 wavefronts (16 decode tokens 3.8 us, in groups 6.0),
    // then kPrepGroup passes and `tpw` tokens (1610 packed tokens of 12 + 4 heads of 128: 11.7 us, a pass alone 14.6;
    // 8192 tokens of 15 + 5 heads of 64: 31 either way).  V: a workgroup a chunk and head.
    const uint32_t rw = 64 / (cache->head_dim / 8), passes = (p.heads + c.kv + rw - 1) / rw;
    const bool grouped = (uint64_t)b.tokens * passes > 4096u;
    const uint32_t groups = grouped ? (passes + kPrepGroup - 1) / kPrepGroup : passes;
    const uint32_t tpw = grouped ? (uint32_t)std::min<uint64_t>(std::max<uint64_t>((uint64_t)b.tokens * groups / 2048, 1), 8) : 1;
    const uint64_t waves = (uint64_t)((b.tokens + tpw - 1) / tpw) * groups, qk = (waves + 3) / 4, vb = chunk_slots(b) * c.kv;
    if (qk + vb > 0x7FFFFFFFu) return fail(CM_EINVAL, "paged prep: %u tokens of %u heads", b.tokens, p.heads);
    const dim3 grid((unsigned)(qk + vb));
#define CM_PREP(HD, I8)                                                                                               \
    if (grouped) {                                                                                                    \
        CM_LAUNCH("paged_prep_kernel", (paged_prep_kernel<HD, I8, kPrepGroup>), grid, dim3(256), 0, s, c, b, a,       \
                  (uint32_t)qk, passes, tpw);                                                                         \
    } else {                                                                                                          \
        CM_LAUNCH("paged_prep_kernel", (paged_prep_kernel<HD, I8, 1>), grid, dim3(256), 0, s, c, b, a, (uint32_t)qk,  \
                  passes, tpw);                                                                                       \
    }
    if (cache->head_dim == 64) {
        if (cache->int8) { CM_PREP(64, true) } else { CM_PREP(64, false) }
    } else {
        if (cache->int8) { CM_PREP(128, true) } else { CM_PREP(128, false) }
    }
#undef CM_PREP
    return CM_OK;
}

int run_read(const cm_paged_cache* cache, const cm_paged_batch* batch, int16_t* k, int16_t* v, uint64_t k_ld,
             uint64_t v_ld, hipStream_t s) {
    Cache c;
    Batch b;
    int rc = view(cache, batch, &c, &b);
    if (rc) return rc;
    if (b.batch == 0 || b.tokens == 0) return CM_OK;
    if (k == nullptr || v == nullptr) return fail(CM_EINVAL, "paged read: a null output");
    if (!aligned16(k) || !aligned16(v) || ((k_ld | v_ld) & 7)) return fail(CM_EALIGN, "paged read: rows must be 16-byte aligned");
    const uint64_t kw = (uint64_t)c.kv * cache->head_dim;
    if (b.tokens > 1 && (k_ld < kw || v_ld < kw))
        return fail(CM_EINVAL, "paged read: rows of %llu columns overlap at their strides", (unsigned long long)kw);
    DeviceState* st;
    if ((rc = state(&st))) return rc;
    const dim3 grid((unsigned)chunk_slots(b), c.kv);
#define CM_READ(HD, I8) \
    CM_LAUNCH("paged_read_kernel", (paged_read_kernel<HD, I8>), grid, dim3(256), 0, s, c, b, k, v, k_ld, v_ld)
    if (cache->head_dim == 64) {
        if (cache->int8) { CM_READ(64, true); } else { CM_READ(64, false); }
    } else {
        if (cache->int8) { CM_READ(128, true); } else { CM_READ(128, false); }
    }
#undef CM_READ
    return CM_OK;
}

int run_attention(const cm_paged_cache* cache, const cm_paged_batch* batch, const int16_t* q, int16_t* o, uint64_t q_ld,
                  uint64_t o_ld, uint32_t heads, uint32_t window, uint32_t smx_cm, uint32_t smx_cfg, hipStream_t s) {
    Cache c;
    Batch b;
    int rc = view(cache, batch, &c, &b);
    if (rc) return rc;
    if (heads == 0 || heads % c.kv || heads / c.kv > 1024)
        return fail(CM_EINVAL, "paged attention: %u heads over %u KV heads", heads, c.kv);
    const uint32_t fp = (smx_cfg >> 8) & 31u;
    if (fp < 1 || fp > 15) return fail(CM_EINVAL, "paged attention: softmax output bits %u (1 .. 15)", fp);
    if (window > 0x3FFFFFFFu) return fail(CM_EINVAL, "paged attention: a window of %u keys", window);
    Smx smx;
    if (!smx_of(smx_cm & 0xFFFFFFu, smx_cfg & 63u, &smx))
        return fail(CM_EINVAL, "paged attention: softmax scale %u 2^-%u (65535 steps within 1/128 octave)", smx_cm & 0xFFFFFFu, smx_cfg & 63u);
    if (b.batch == 0 || b.tokens == 0) return CM_OK;
    if (q == nullptr || o == nullptr) return fail(CM_EINVAL, "paged attention: a null q or o");
    if (!aligned16(q) || !aligned16(o) || ((q_ld | o_ld) & 7))
        return fail(CM_EALIGN, "paged attention: rows must be 16-byte aligned");
    const uint64_t qw = (uint64_t)heads * cache->head_dim;
    if (b.tokens > 1 && (q_ld < qw || o_ld < qw))
        return fail(CM_EINVAL, "paged attention: rows of %llu columns overlap at their strides", (unsigned long long)qw);
    DeviceState* st;
    if ((rc = state(&st))) return rc;
    const uint32_t G = heads / c.kv;
    if ((uint64_t)b.tokens * G > 0x7FFFFFFFu)
        return fail(CM_EINVAL, "paged attention: %u tokens of %u heads", b.tokens, heads);
    const Attn a{q, o, q_ld, o_ld, G, window, fp, smx};
    // Tiles of 15 rows in one launch (tables of at most kShort rows), tiles of 15 rows whose scores are kept (where those
    // fit kMaxScores), or tiles of 64 or 128 rows that compute the scores twice: the least of three estimates in ns, from
    // the tiles' count for sequences of equal rows.  They decide as the present kernels' times do, within 3 % (15 + 5 heads
    // of 64, us of few and of many): 16 sequences of 1024 rows, 1 / 16 / 32 tokens each 11.5 / 29.5 / 45 and 38 / 41 / 43;
    // of 4096, 8 / 12 / 16 tokens 47 / 65 / 81 and 74 / 74 / 73; one of 1000, 40 tokens 12.3 and 27; one of 200, 100 tokens
    // 8.3 and 31; one of 4000, 20 tokens 18 and 36.  (16 + 4 heads of 128, int16 / int8) 16 of 4096, 8 tokens 83 / 62 and
    // 68 / 55; 1 token 38 / 33 and 66 / 52.  All of it counts the table's width (cap), the lengths being on the device: 16
    // sequences of 1024 rows, a token each, take 11.4 us under tables of 2048 rows, 16.6 of 8192 and 19.4 of 16384.
    const uint64_t rows = (uint64_t)b.tokens * heads, packed = (uint64_t)b.tokens * G, each = (packed + b.batch - 1) / b.batch;
    const uint32_t steps = (b.cap + 63) / 64, big = cache->head_dim == 64 ? 128 : 64, wide = cache->head_dim / 64;
    auto tiles_of = [&](uint32_t r) { return (each + r - 1) / r * b.batch * c.kv; };
    const uint64_t many_ns = 31000 + tiles_of(big) * steps * (cache->int8 ? 55 : 85) / 10;
    const uint64_t rounds = ((packed / kFewRows + b.batch) * c.kv + st->cus - 1) / st->cus;
    const uint64_t few_ns = b.cap <= kShort ? rounds * (6500 + 8 * b.cap) * (wide + 1) / 2
                                            : wide == 1 ? 12000 + tiles_of(kFewRows) * steps * (cache->int8 ? 26 : 35) / 10
                                                        : 18000 + tiles_of(kFewRows) * steps * (cache->int8 ? 37 : 50) / 10;
    const bool few = few_ns <= many_ns && (b.cap <= kShort || rows * b.cap * 2 <= kMaxScores);
    const uint32_t R = few ? kFewRows : big;
    const uint64_t slots = packed / R + b.batch;
    if (slots > 0x7FFFFFFFu) return fail(CM_EINVAL, "paged attention: %u tokens of %u heads", b.tokens, heads);
    const dim3 tiles((unsigned)slots, c.kv);
    if (few && b.cap <= kShort) {
#define CM_SHORT(HD, I8) \
    CM_LAUNCH("paged_short_kernel", (paged_short_kernel<HD, I8>), tiles, dim3(1024), 0, s, c, b, a, st->smx_tab)
        if (cache->head_dim == 64) {
            if (cache->int8) { CM_SHORT(64, true); } else { CM_SHORT(64, false); }
        } else {
            if (cache->int8) { CM_SHORT(128, true); } else { CM_SHORT(128, false); }
        }
#undef CM_SHORT
        return CM_OK;
    }
    if (few) {
        // parts of equal steps: about eight workgroups a compute unit, two steps a wavefront for the scores; a part of at
        // most kMaxPart keys (the int32 limb sums)
        const uint32_t wgs = (uint32_t)std::min<uint64_t>(slots * c.kv, 1u << 20), want = std::max(8u * (uint32_t)st->cus / wgs, 1u);
        const uint32_t per = std::min(std::max((steps + want - 1) / want, 4u), kMaxPart / 64), splits = (steps + per - 1) / per;
        const uint32_t per_s = std::min(per, 8u), splits_s = (steps + per_s - 1) / per_s;
        if (splits_s > 65535u) return fail(CM_EINVAL, "paged attention: %u parts", splits_s);
        const size_t mx_bytes = round_up(rows * splits_s * 4, 256), sc_bytes = round_up(rows * b.cap * 2, 256);
        const size_t part_bytes = splits > 1 ? rows * splits * (cache->head_dim + 2) * 8 : 0;
        void* ws;
        if ((rc = workspace(st, mx_bytes + sc_bytes + part_bytes, &ws, s))) return rc;
        uint8_t* p = static_cast<uint8_t*>(ws);
        const Work wk{reinterpret_cast<int32_t*>(p), reinterpret_cast<int16_t*>(p + mx_bytes),
                      reinterpret_cast<int64_t*>(p + mx_bytes + sc_bytes), splits, per, splits_s, per_s};
        const dim3 grid((unsigned)slots, c.kv, splits), sgrid((unsigned)slots, c.kv, splits_s), jgrid((unsigned)(((uint64_t)b.tokens * G + 3) / 4), c.kv);
#define CM_FEW(HD, I8)                                                                                              \
    CM_LAUNCH("paged_scores_kernel", (paged_scores_kernel<HD, I8>), sgrid, dim3(256), 0, s, c, b, a, wk);           \
    CM_LAUNCH("paged_few_kernel", (paged_few_kernel<HD, I8>), grid, dim3(256), 0, s, c, b, a, wk, st->smx_tab);     \
    if (splits > 1) { CM_LAUNCH("paged_join_kernel", paged_join_kernel<HD>, jgrid, dim3(256), 0, s, b, a, wk); }
        if (cache->head_dim == 64) {
            if (cache->int8) { CM_FEW(64, true) } else { CM_FEW(64, false) }
        } else {
            if (cache->int8) { CM_FEW(128, true) } else { CM_FEW(128, false) }
        }
#undef CM_FEW
        return CM_OK;
    }
    if (slots * (steps + kTileCost) > 0xFFFFFFFFu)
        return fail(CM_EINVAL, "paged attention: %u tokens over %u rows", b.tokens, b.cap);
    const bool planned = slots > kPlan || b.batch > 64;
    const uint32_t shares = 2 * (uint32_t)st->cus / 8 * 8, max_shares = 2 * shares;
    const size_t cum_bytes = planned ? round_up((slots + 1) * 4, 256) : 0, mx_bytes = (max_shares + slots * c.kv) * R * 4;
    void* ws;
    if ((rc = workspace(st, cum_bytes + mx_bytes + (size_t)shares * 2 * R * (cache->head_dim + 1) * 8, &ws, s))) return rc;
    uint8_t* p = static_cast<uint8_t*>(ws);
    const Queue qu{planned ? reinterpret_cast<uint32_t*>(p) : nullptr, reinterpret_cast<int32_t*>(p + cum_bytes),
                   reinterpret_cast<int64_t*>(p + cum_bytes + mx_bytes), (uint32_t)slots, max_shares, shares};
    const dim3 jgrid((unsigned)slots, c.kv, cache->head_dim / 16 * (R / 64));
#define CM_ROWS(HD, I8, QB)                                                                                         \
    if (planned) { CM_LAUNCH("paged_plan_kernel", paged_plan_kernel<64 * QB>, dim3(1), dim3(1024), 0, s, b, a, qu); } \
    CM_LAUNCH("paged_max_kernel", (paged_max_kernel<HD, I8, QB>), dim3(max_shares), dim3(256), 0, s, c, b, a, qu);  \
    CM_LAUNCH("paged_rows_kernel", (paged_rows_kernel<HD, I8, QB>), dim3(shares), dim3(256), 0, s, c, b, a, qu,     \
              st->smx_tab);                                                                                         \
    CM_LAUNCH("paged_join_kernel", (paged_rows_join_kernel<HD, QB>), jgrid, dim3(256), 0, s, c, b, a, qu);
    if (cache->head_dim == 64) {
        if (cache->int8) { CM_ROWS(64, true, 2) } else { CM_ROWS(64, false, 2) }
    } else {
        if (cache->int8) { CM_ROWS(128, true, 1) } else { CM_ROWS(128, false, 1) }
    }
#undef CM_ROWS
    return CM_OK;
}

}  // namespace
}  // namespace cm

extern "C" size_t cm_paged_block_bytes(uint32_t page, uint32_t head_dim, uint32_t int8) {
    return cm::block_bytes(page, head_dim, int8 != 0);
}

extern "C" int cm_paged_prep(const cm_paged_cache* cache, const cm_paged_batch* batch, const cm_paged_prep_args* args,
                             void* stream) {
    return cm::run_prep(cache, batch, args, cm::as_stream(stream));
}

extern "C" int cm_paged_attention(const cm_paged_cache* cache, const cm_paged_batch* batch, const int16_t* q, int16_t* o,
                                  uint64_t q_ld, uint64_t o_ld, uint32_t heads, uint32_t window, uint32_t smx_cm,
                                  uint32_t smx_cfg, void* stream) {
    return cm::run_attention(cache, batch, q, o, q_ld, o_ld, heads, window, smx_cm, smx_cfg, cm::as_stream(stream));
}

extern "C" int cm_paged_read(const cm_paged_cache* cache, const cm_paged_batch* batch, int16_t* k, int16_t* v,
                             uint64_t k_ld, uint64_t v_ld, void* stream) {
    return cm::run_read(cache, batch, k, v, k_ld, v_ld, cm::as_stream(stream));
}
