// cm_paged.hip -- the paged K / V cache: the step's rows into it (cm_paged_prep), the attention over
// it (cm_paged_attention) and its rows back (cm_paged_read).
//
// A page holds K rows as the byte planes that an MFMA operand lane reads 16 bytes of (d contiguous for
// q.K^T) and V transposed (keys contiguous for P.V), so the attention neither splits nor transposes
// what it reads: an int16 x is 256 h + l + 128 (h = x >> 8, l = (x & 255) - 128).
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

// rsqrt_bf (cm_rowops_math.h) for D below 2^63
__device__ __forceinline__ void rsqrt64(uint64_t D, uint64_t& Rm, int& sh, const uint8_t* tab) {
    const int e = 64 - __clzll((long long)D);
    int d = e - 32;
    d += d & 1;
    const uint32_t Dm = (uint32_t)(d >= 0 ? D >> d : D << -d);
    const uint32_t y0 = *reinterpret_cast<const uint32_t*>(tab + 32768 + 4 * ((Dm >> 19) & 8191u));
    const uint32_t u = __umulhi(__umulhi(Dm, y0), y0);
    const __int128 y1 = (__int128)y0 + (((__int128)y0 * (((int64_t)1 << 30) - (int64_t)u)) >> 31);
    const __int128 lo = (__int128)1 << 31, hi = ((__int128)1 << 32) - 1;
    Rm = (uint64_t)(y1 < lo ? lo : y1 > hi ? hi : y1);
    sh = 47 + d / 2;
}

__device__ __forceinline__ int rne_sat(int64_t v, uint32_t sc) {
    return (int)(sc <= 61 ? ro::sat16(ro::rne_shr_fast(v, sc)) : ro::sat16(ro::rne_shr((__int128)v, (int)sc)));
}

template <uint32_t L>
__device__ __forceinline__ int64_t row_sum64(int64_t x) {     // over the L lanes of a row
#pragma unroll
    for (uint32_t o = 1; o < L; o <<= 1) x += (int64_t)ro::shfl64((uint64_t)x, (int)o);
    return x;
}

// HD / 8 lanes a head row, 8 columns a lane; a wavefront takes consecutive rows of
// [token][q heads, k heads, v heads].
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_prep_kernel(Cache c, Batch bt, Prep a) {
    constexpr uint32_t L = HD / 8, RW = 64 / L;
    const uint32_t lane = threadIdx.x & 63, u = lane % L, d0 = 8 * u;
    const uint32_t per = a.heads + 2 * c.kv;
    const uint64_t item = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * RW + lane / L;
    const uint64_t items = (uint64_t)bt.start(bt.batch) * per;
    if (((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * RW >= items) return;
    const bool on = item < items;
    const uint32_t tok = on ? (uint32_t)(item / per) : 0u, head = on ? (uint32_t)(item - (uint64_t)tok * per) : 0u;
    // the wavefront's tokens lie in a few sequences: the first by search, then the rows after it one by one
    const uint32_t tok0 = __builtin_amdgcn_readfirstlane(tok);
    uint32_t b = find_le(bt.batch, tok0, [&](uint32_t i) { return bt.start(i); });
    while (b + 1 < bt.batch && bt.start(b + 1) <= tok) b++;
    const int n = (int)bt.start(b + 1) - (int)bt.start(b);
    const int64_t pos = (int64_t)bt.len(b) - n + (int)(tok - bt.start(b));
    const bool isq = head < a.heads, isv = head >= a.heads + c.kv;
    const uint32_t g = isq ? head : isv ? head - a.heads - c.kv : head - a.heads;
    const int16_t* src = isq ? a.q + tok * a.q_ld : isv ? a.v + tok * a.v_ld : a.k + tok * a.k_ld;
    const int4 xw = on ? *reinterpret_cast<const int4*>(src + g * HD + d0) : make_int4(0, 0, 0, 0);
    int x[8];
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) x[l] = (int)reinterpret_cast<const int16_t*>(&xw)[l];

    const uint8_t* np = isq ? a.norm_q : isv ? nullptr : a.norm_k;
    int64_t s2 = 0;
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) s2 += (int64_t)x[l] * x[l];
    s2 = row_sum64<L>(s2);
    if (np != nullptr) {
        const int64_t D = s2 + (isq ? a.eps_q : a.eps_k);
        uint64_t Rm;
        int sh;
        rsqrt64((uint64_t)(D > 0 ? D : 1), Rm, sh, a.tab);
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) {
            const ro::Param p = ro::ld_param(np, d0 + l, false);
            const int64_t P1 = ((int64_t)x[l] * (int64_t)Rm) >> (sh - 24);
            x[l] = rne_sat(P1 * p.g + p.bq, (uint32_t)p.sc);
        }
    }
    // rotation: the partner column's value from this or another lane of the row
    const uint32_t half = a.rotary / 2;
    const uint32_t row = (uint32_t)min(max(pos, (int64_t)0), (int64_t)a.rope_rows - 1);
    const int32_t* cs = a.rope + (uint64_t)row * 2 * a.rotary;
    const bool rot = d0 < a.rotary;
    const uint32_t pl = a.interleaved ? lane : d0 < half ? lane + half / 8 : lane - half / 8;
    int y[8];
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) {
        const int other = __shfl(x[l], (int)(rot ? pl : lane), 64);
        y[l] = a.interleaved ? (l & 1 ? x[l - 1] : -x[l + 1]) : d0 < half ? -other : other;
    }
    if (!isv) {
        const uint8_t* rp = isq ? a.rope_q : a.rope_k;
        const bool cols = (isq ? a.rope_q_cols : a.rope_k_cols) != 0;
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) {
            const ro::Param p = ro::ld_param(rp, g * HD + d0 + l, !cols);
            const int co = rot ? cs[d0 + l] : 1 << 23, si = rot ? cs[a.rotary + d0 + l] : 0;
            x[l] = ro::rope_elem(x[l], rot ? y[l] : 0, co, si, p);
        }
    }
    if (isq) {
        if (on) *reinterpret_cast<int4*>(a.qr + tok * a.qr_ld + g * HD + d0) = ro::pack16(x);
        // fall through: the lanes of other rows of this wavefront share the shuffles below
    }
    // the int8 form's shift and codes, and the key's term
    uint32_t e = 0;
    if constexpr (I8) {
        int m = 0;
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) m = max(m, x[l] ^ (x[l] >> 31));
#pragma unroll
        for (uint32_t o = 1; o < L; o <<= 1) m = max(m, __shfl_xor(m, (int)o, 64));
        e = (uint32_t)max(0, 32 - __clz(m) - 7);
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) x[l] = min(127, (int)ro::rne_shr_fast(x[l], e));
    }
    int s = 0;
#pragma unroll
    for (uint32_t l = 0; l < 8; l++) s += x[l];
#pragma unroll
    for (uint32_t o = 1; o < L; o <<= 1) s += __shfl_xor(s, (int)o, 64);
    if (isq || !on || pos < 0 || pos >= (int64_t)bt.cap) return;
    const uint32_t id = (uint32_t)bt.table[b * bt.table_ld + (uint32_t)(pos >> c.lg)], slot = (uint32_t)pos & (c.page - 1);
    if (id >= c.pages) return;
    uint8_t* blk = c.data + ((uint64_t)id * c.kv + g) * c.block;
    typedef Block<HD, I8> B;
    uint32_t h[2], lo[2];                  // bytes of the two planes (the codes alone in int8)
#pragma unroll
    for (uint32_t w = 0; w < 2; w++) {
        h[w] = lo[w] = 0;
#pragma unroll
        for (uint32_t l = 0; l < 4; l++) {
            const uint32_t z = (uint32_t)x[4 * w + l];
            h[w] |= ((I8 ? z : z >> 8) & 255u) << (8 * l);
            lo[w] |= ((z & 255u) ^ 128u) << (8 * l);
        }
    }
    if (!isv) {
        *reinterpret_cast<uint2*>(blk + B::k(c.page, 0) + slot * HD + d0) = make_uint2(h[0], h[1]);
        if constexpr (!I8) *reinterpret_cast<uint2*>(blk + B::k(c.page, 1) + slot * HD + d0) = make_uint2(lo[0], lo[1]);
        if (u == 0) {
            reinterpret_cast<int32_t*>(blk + B::term(c.page))[slot] = 128 * s - (I8 ? 0 : 16384 * (int)HD);
            if constexpr (I8) blk[B::ke(c.page) + slot] = (uint8_t)e;
        }
    } else {
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) {
            blk[B::v(c.page, 0) + (d0 + l) * c.page + slot] = (uint8_t)(h[l / 4] >> (8 * (l & 3)));
            if constexpr (!I8) blk[B::v(c.page, 1) + (d0 + l) * c.page + slot] = (uint8_t)(lo[l / 4] >> (8 * (l & 3)));
        }
        if constexpr (I8)
            if (u == 0) blk[B::ve(c.page) + slot] = (uint8_t)e;
    }
}

// ---------------------------------------------------------------- read
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_read_kernel(Cache c, Batch bt, int16_t* k, int16_t* v, uint64_t k_ld,
                                                         uint64_t v_ld) {
    constexpr uint32_t L = HD / 8, RW = 64 / L;
    const uint32_t lane = threadIdx.x & 63, d0 = 8 * (lane % L);
    const uint64_t first = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * RW;
    const uint64_t items = (uint64_t)bt.start(bt.batch) * c.kv;
    if (first >= items) return;
    const uint64_t item = min(first + lane / L, items - 1);
    const uint32_t tok = (uint32_t)(item / c.kv), g = (uint32_t)(item - (uint64_t)tok * c.kv);
    uint32_t b = find_le(bt.batch, __builtin_amdgcn_readfirstlane(tok), [&](uint32_t i) { return bt.start(i); });
    while (b + 1 < bt.batch && bt.start(b + 1) <= tok) b++;
    const int n = (int)bt.start(b + 1) - (int)bt.start(b);
    const int64_t pos = (int64_t)bt.len(b) - n + (int)(tok - bt.start(b));
    const bool in = pos >= 0 && pos < (int64_t)bt.cap;
    const uint32_t id = in ? (uint32_t)bt.table[b * bt.table_ld + (uint32_t)(pos >> c.lg)] : 0xFFFFFFFFu;
    int kx[8] = {0, 0, 0, 0, 0, 0, 0, 0}, vx[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (id < c.pages) {
        const uint32_t slot = (uint32_t)pos & (c.page - 1);
        const uint8_t* blk = c.data + ((uint64_t)id * c.kv + g) * c.block;
        typedef Block<HD, I8> B;
        const int8_t *kp = reinterpret_cast<const int8_t*>(blk + B::k(c.page, 0) + slot * HD + d0),
                     *vp = reinterpret_cast<const int8_t*>(blk + B::v(c.page, 0) + d0 * c.page + slot);
#pragma unroll
        for (uint32_t l = 0; l < 8; l++) {
            if constexpr (I8) {
                kx[l] = kp[l] << blk[B::ke(c.page) + slot];
                vx[l] = vp[l * c.page] << blk[B::ve(c.page) + slot];
            } else {
                kx[l] = kp[l] * 256 + kp[c.page * HD + l] + 128;
                vx[l] = vp[l * c.page] * 256 + vp[(HD + l) * c.page] + 128;
            }
        }
    }
    *reinterpret_cast<int4*>(k + tok * k_ld + g * HD + d0) = ro::pack16(kx);
    *reinterpret_cast<int4*>(v + tok * v_ld + g * HD + d0) = ro::pack16(vx);
}

// ---------------------------------------------------------------- attention
struct Attn {
    const int16_t* q;
    int16_t* o;
    uint64_t q_ld, o_ld;
    uint32_t G, window, cm, cs, fp, dlim;
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

// floor(2^(fp - 8) A / S + 1/2) saturated to int16: the quotient estimated in double (2 |A| 2^7 < 2^60, S <
// 2^37), put right by the int64 remainder
__device__ __forceinline__ int finish(int64_t A, int64_t S, uint32_t fp) {
    if (S == 0) return 0;
    const int64_t num = fp >= 8 ? 2 * (A * ((int64_t)1 << (fp - 8))) + S : 2 * A + (S << (8 - fp));
    const int64_t den = 2 * (fp >= 8 ? S : S << (8 - fp));
    int64_t f = (int64_t)floor((double)num / (double)den);
    const int64_t r = num - f * den;
    f += r >= den ? 1 : r < 0 ? -1 : 0;
    return (int)(f > 32767 ? 32767 : f < -32768 ? -32768 : f);
}

// A workgroup takes 16 rows (token, head of the group) of one sequence and KV head; its wavefronts take
// the 64-key steps of the keys that any row sees, w, w + 4, ..; first the rows' maxima, then weights and
// P.V with the scores computed again.
template <uint32_t HD, bool I8>
__global__ __launch_bounds__(256) void paged_attention_kernel(Cache c, Batch bt, Attn a, const int32_t* __restrict__ tab) {
    constexpr uint32_t KS = HD / 64, DB = HD / 16;
    typedef Block<HD, I8> B;
    __shared__ __attribute__((aligned(16))) int32_t stab[4096];
    __shared__ int32_t redm[4][16];
    __shared__ int64_t reds[4][16];
    __shared__ int64_t part[16][HD + 1];
    const uint32_t t = threadIdx.x, lane = t & 63, c16 = lane & 15, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t slot = blockIdx.x, head = blockIdx.y;
    // sequence b's tiles have the slots from floor(start(b) G / 16) + b on
    auto first = [&](uint32_t b) { return (uint32_t)((uint64_t)bt.start(b) * a.G / 16) + b; };
    const uint32_t b = find_le(bt.batch, slot, first);
    const uint32_t q0 = bt.start(b), n = (uint32_t)max((int)bt.start(b + 1) - (int)q0, 0);
    const uint32_t tile = slot - first(b), rows = n * a.G;
    if (tile * 16 >= rows) return;
    const int base = bt.len(b) - (int)n;                    // position of the sequence's first new token
    const uint32_t row = tile * 16 + c16;
    const bool on = row < rows;
    const uint32_t tok = row / a.G, hh = head * a.G + row % a.G;
    auto seen = [&](uint32_t tk) { return (uint32_t)min(max(base + (int)tk + 1, 0), (int)bt.cap); };
    auto begin = [&](uint32_t tk) { return a.window ? (uint32_t)max(base + (int)tk + 1 - (int)a.window, 0) : 0u; };
    const uint32_t vend = on ? seen(tok) : 0u, vbeg = on ? begin(tok) : 0u;
    const uint32_t lo = begin(tile * 16 / a.G) & ~63u, hi = seen(min((tile * 16 + 15) / a.G, n - 1));
    const int32_t* tb = bt.table + b * bt.table_ld;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) *reinterpret_cast<int4*>(stab + 4 * (t + 256 * i)) = *reinterpret_cast<const int4*>(tab + 4 * (t + 256 * i));
    for (uint32_t i = t; i < 16 * (HD + 1); i += 256) (&part[0][0])[i] = 0;

    v4i qh[KS], ql[KS];
    int qsum = 0;
    const int16_t* qp = a.q + (uint64_t)(q0 + (on ? tok : 0)) * a.q_ld + (uint64_t)(on ? hh : 0) * HD + 16 * g;
#pragma unroll
    for (uint32_t s = 0; s < KS; s++) limbs16(qp + 64 * s, qh[s], ql[s], qsum);
    qsum += __shfl_xor(qsum, 16, 64);
    qsum += __shfl_xor(qsum, 32, 64);
    const int qterm = I8 ? 0 : 128 * qsum;
    const v4i zero = {0, 0, 0, 0}, ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};

    // a key's page: outside the pool its rows are masked (and block 0 read in their place)
    auto page_of = [&](uint32_t key) { return key < bt.cap ? (uint32_t)tb[key >> c.lg] : 0xFFFFFFFFu; };
    auto block_of = [&](uint32_t id) { return c.data + ((uint64_t)(id < c.pages ? id : 0) * c.kv + head) * c.block; };
    // the scores of 64 keys: the lane's are k0 + 16 g + 4 kb + r of query c16 (row i of block kb is key
    // 16 (i / 4) + 4 kb + i % 4, so that the lane's keys are the 16 consecutive ones of its V operand)
    auto scores = [&](uint32_t k0, const uint8_t* vb, bool ok, int (&sv)[16]) {
        const uint32_t kr = k0 + 16 * (c16 >> 2) + (c16 & 3), kg = k0 + 16 * g;
        const uint8_t* kb0 = block_of(page_of(kr)) + 16 * g;
#pragma unroll
        for (uint32_t kb = 0; kb < 4; kb++) {
            const uint8_t* kp = kb0 + ((kr + 4 * kb) & (c.page - 1)) * HD;
            v4i hh4 = zero, mid = zero, ll = *reinterpret_cast<const v4i*>(vb + B::term(c.page) + 4 * ((kg + 4 * kb) & (c.page - 1)));
#pragma unroll
            for (uint32_t s = 0; s < KS; s++) {
                const v4i kh = *reinterpret_cast<const v4i*>(kp + 64 * s);
                if constexpr (I8) {
                    mid = mfma(kh, qh[s], mid);
                    ll = mfma(kh, ql[s], ll);
                } else {
                    const v4i kl = *reinterpret_cast<const v4i*>(kp + B::k(c.page, 1) + 64 * s);
                    hh4 = mfma(kh, qh[s], hh4);
                    mid = mfma(kh, ql[s], mid);
                    mid = mfma(kl, qh[s], mid);
                    ll = mfma(kl, ql[s], ll);
                }
            }
            uint32_t es = 0;
            if constexpr (I8) es = *reinterpret_cast<const uint32_t*>(vb + B::ke(c.page) + ((kg + 4 * kb) & (c.page - 1)));
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                uint32_t acc = ((uint32_t)mid[r] << 8) + (uint32_t)ll[r];
                if constexpr (I8) acc <<= (es >> (8 * r)) & 31u;
                else acc += ((uint32_t)hh4[r] << 16) + (uint32_t)qterm;
                const uint32_t key = kg + 4 * kb + r;
                sv[4 * kb + r] = ok && key >= vbeg && key < vend ? sat16i((int)acc >> 8) : -0x10000;
            }
        }
    };

    int mx = -0x10000;
    for (uint32_t k0 = lo + 64 * w; k0 < hi; k0 += 256) {
        const uint32_t id = page_of(k0 + 16 * g);
        int sv[16];
        scores(k0, block_of(id), id < c.pages, sv);
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) mx = max(mx, sv[i]);
    }
    mx = max(mx, __shfl_xor(mx, 16, 64));
    mx = max(mx, __shfl_xor(mx, 32, 64));
    if (g == 0) redm[w][c16] = mx;
    __syncthreads();
    mx = max(max(redm[0][c16], redm[1][c16]), max(redm[2][c16], redm[3][c16]));

    constexpr uint32_t NA = 3;             // limb products: int16 hh, mid, ll; int8 the weight's three bytes
    v4i acc[NA][DB], vs[I8 ? 1 : 2][DB];
#pragma unroll
    for (uint32_t m = 0; m < DB; m++) {
        acc[0][m] = acc[1][m] = acc[2][m] = zero;
        vs[0][m] = vs[I8 ? 0 : 1][m] = zero;
    }
    int64_t wsum = 0;
    for (uint32_t k0 = lo + 64 * w; k0 < hi; k0 += 256) {
        const uint32_t id = page_of(k0 + 16 * g);
        const uint8_t* vb = block_of(id);
        int sv[16];
        scores(k0, vb, id < c.pages, sv);
        uint32_t part32 = 0;
        const uint32_t in = (k0 + 16 * g) & (c.page - 1);
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) {
            const bool ok = sv[i] != -0x10000;
            const uint32_t d = ok ? (uint32_t)(mx - sv[i]) : 0u;
            const uint32_t y = (uint32_t)(((uint64_t)d * a.cm) >> a.cs);
            const uint32_t e = ok && d < a.dlim ? min((uint32_t)stab[y & 4095] >> ((y >> 12) & 31), 65535u) : 0u;
            part32 += e;
            sv[i] = (int)e;
        }
        wsum += part32;
        v4i p[3];
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
            uint32_t e4[4], by[3] = {0, 0, 0};
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                e4[r] = (uint32_t)sv[4 * q + r];
                if constexpr (I8) e4[r] <<= vb[B::ve(c.page) + in + 4 * q + r] & 15u;
#pragma unroll
                for (uint32_t z = 0; z < 3; z++) by[z] |= (((e4[r] >> (8 * z)) & 255u) ^ 128u) << (8 * r);
            }
            p[0][q] = (int)by[0];
            p[1][q] = (int)by[1];
            p[2][q] = (int)by[2];
        }
#pragma unroll
        for (uint32_t m = 0; m < DB; m++) {
            const uint8_t* vp = vb + B::v(c.page, 0) + (16 * m + c16) * c.page + in;
            const v4i vh = *reinterpret_cast<const v4i*>(vp);
            if constexpr (I8) {
                acc[0][m] = mfma(vh, p[2], acc[0][m]);
                acc[1][m] = mfma(vh, p[1], acc[1][m]);
                acc[2][m] = mfma(vh, p[0], acc[2][m]);
                vs[0][m] = mfma(vh, ones, vs[0][m]);
            } else {
                const v4i vl = *reinterpret_cast<const v4i*>(vp + HD * c.page);
                acc[0][m] = mfma(vh, p[1], acc[0][m]);
                acc[1][m] = mfma(vh, p[0], acc[1][m]);
                acc[1][m] = mfma(vl, p[1], acc[1][m]);
                acc[2][m] = mfma(vl, p[0], acc[2][m]);
                vs[0][m] = mfma(vh, ones, vs[0][m]);
                vs[1][m] = mfma(vl, ones, vs[1][m]);
            }
        }
    }
    wsum += (int64_t)ro::shfl64((uint64_t)wsum, 16);
    wsum += (int64_t)ro::shfl64((uint64_t)wsum, 32);
    if (g == 0) reds[w][c16] = wsum;
#pragma unroll
    for (uint32_t m = 0; m < DB; m++)
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) {
            int64_t x = (int64_t)acc[0][m][r] * 65536 + (int64_t)acc[1][m][r] * 256 + acc[2][m][r];
            x += I8 ? (int64_t)vs[0][m][r] * (128 * 65793)
                    : ((int64_t)vs[0][m][r] * 256 + vs[I8 ? 0 : 1][m][r]) * 32896 + 128 * wsum;
            atomicAdd(reinterpret_cast<unsigned long long*>(&part[c16][16 * m + 4 * g + r]), (unsigned long long)x);
        }
    __syncthreads();
    for (uint32_t i = t; i < 16 * HD / 2; i += 256) {
        const uint32_t r = i / (HD / 2), d = 2 * (i % (HD / 2)), rw = tile * 16 + r;
        if (rw >= rows) break;
        const int64_t S = reds[0][r] + reds[1][r] + reds[2][r] + reds[3][r];
        const int o0 = finish(part[r][d], S, a.fp), o1 = finish(part[r][d + 1], S, a.fp);
        *reinterpret_cast<uint32_t*>(a.o + (uint64_t)(q0 + rw / a.G) * a.o_ld + (uint64_t)(head * a.G + rw % a.G) * HD + d) =
            (uint32_t)(uint16_t)o0 | ((uint32_t)(uint16_t)o1 << 16);
    }
}

// ---------------------------------------------------------------- the host's checks
constexpr uint32_t kMaxKeys = 1u << 20;

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
    const uint64_t items = (uint64_t)b.tokens * (p.heads + 2 * c.kv), per = 4 * (64 / (cache->head_dim / 8));
    const dim3 grid((unsigned)((items + per - 1) / per));
#define CM_PREP(HD, I8)                                                                                     \
    CM_LAUNCH("paged_prep_kernel", (paged_prep_kernel<HD, I8>), grid, dim3(256), 0, s, c, b, a)
    if (cache->head_dim == 64) {
        if (cache->int8) { CM_PREP(64, true); } else { CM_PREP(64, false); }
    } else {
        if (cache->int8) { CM_PREP(128, true); } else { CM_PREP(128, false); }
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
    const uint64_t items = (uint64_t)b.tokens * c.kv, per = 4 * (64 / (cache->head_dim / 8));
    const dim3 grid((unsigned)((items + per - 1) / per));
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
    if (b.batch == 0 || b.tokens == 0) return CM_OK;
    if (q == nullptr || o == nullptr) return fail(CM_EINVAL, "paged attention: a null q or o");
    if (!aligned16(q) || !aligned16(o) || ((q_ld | o_ld) & 7))
        return fail(CM_EALIGN, "paged attention: rows must be 16-byte aligned");
    const uint64_t qw = (uint64_t)heads * cache->head_dim;
    if (b.tokens > 1 && (q_ld < qw || o_ld < qw))
        return fail(CM_EINVAL, "paged attention: rows of %llu columns overlap at their strides", (unsigned long long)qw);
    DeviceState* st;
    if ((rc = state(&st))) return rc;
    const uint32_t cm24 = smx_cm & 0xFFFFFFu, cs = smx_cfg & 63u, G = heads / c.kv;
    const Attn a{q, o, q_ld, o_ld, G, window, cm24, cs, fp, smx_dlim(cm24, cs)};
    const uint64_t slots = (uint64_t)b.tokens * G / 16 + b.batch;
    if (slots > 0x7FFFFFFFu) return fail(CM_EINVAL, "paged attention: %u tokens of %u heads", b.tokens, heads);
    const dim3 grid((unsigned)slots, c.kv);
#define CM_ATTN(HD, I8) \
    CM_LAUNCH("paged_attention_kernel", (paged_attention_kernel<HD, I8>), grid, dim3(256), 0, s, c, b, a, st->smx_tab)
    if (cache->head_dim == 64) {
        if (cache->int8) { CM_ATTN(64, true); } else { CM_ATTN(64, false); }
    } else {
        if (cache->int8) { CM_ATTN(128, true); } else { CM_ATTN(128, false); }
    }
#undef CM_ATTN
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
