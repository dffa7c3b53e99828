// cm_linear8.hip -- the 8-bit linear layers: int16 rows quantised a token at a time, their product with
// 8-bit weights on CDNA4 i8 MFMA, and what a decoder does with it: a bias and int16 rows, the add
// into the int32 residual stream, or a feed-forward block's gate (activation of one product times another).
//
// Arithmetic.  A row's codes are c = (x R + 2^23) >> 24 with R = floor((127 2^24 + (a >> 1)) / a), a = max |x|
// (|x R| <= 127 2^24 + 2^14: 32 bits).  acc = sum c w is exact in int32 (k <= 32768: |acc| <= 2^29).
// The output is rne(acc a mu + b), mu the channel's multiplier, a double: acc a < 2^45 is exact in a
// double, and one fused multiply-add onto 1.5 2^52 + b rounds the exact value once, to the nearest whole
// number, ties to even, which then stands in the low word.  |mu| <= 64 keeps the sum below 2^52.
//
// Layout.  Codes and weights are held as the matrix units read them: blocks of 32 lines (rows of
// x, columns of w) by 64 k, 2 KiB each, in it 16-byte pieces of 16 consecutive k, [k / 16 % 4][line % 32].
// A 32 x 32 x 32 operand is then 1 KiB in lane order, a 16 x 16 x 64 operand four runs of 256 bytes.  A gated
// weight alternates blocks of 32 gate columns and the same 32 up columns.
#include "cm_common.h"

#include <algorithm>
#include <type_traits>

namespace cm {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr uint32_t kLine = 32, kStep = 64, kPiece = kLine * kStep;      // lines and k of a block, its bytes
constexpr uint32_t kMaxK = 32768, kMaxM = 1u << 20, kMaxN = 1u << 22;
constexpr double kMagic = 6755399441055744.0;                           // 1.5 2^52: a whole number added to it is its low word

// What a product becomes: int16 rows, the int32 residual with them, or a gate by the sigmoid's pieces or a byte table.
enum : uint32_t { kOut16 = 0, kOut32 = 1, kSiluGate = 2, kTableGate = 3 };
constexpr bool gated(uint32_t mode) { return mode >= kSiluGate; }
enum : uint32_t { kSilu = 0, kGelu = 1, kGeluTanh = 2 };             // cm_linear8_weight's act
constexpr double kMagic70 = 0x1.8p70;
constexpr uint32_t kPieces = 4096;                                    // of the sigmoid, 8 bytes each, and one behind them
static_assert(kSigmoidBytes >= 8 * (kPieces + 1) && kSigmoidBytes % 4096 == 0, "whole copies of four wavefronts");

inline uint32_t steps_of(uint32_t k) { return ceil_div(k, kStep); }
inline uint32_t blocks_of(uint32_t lines) { return ceil_div(lines, kLine); }

// Bytes of a block of lines; where a rows image's maxima and a weight image's channel parameters start (behind the blocks).  An
// odd number of pieces between blocks, for k of powers of two, measured the same (8192 x 4096 x 8192).
__host__ __device__ inline uint32_t pitch_of(uint32_t steps) { return steps * kPiece; }
inline size_t codes_bytes(uint32_t blocks, uint32_t k) { return (size_t)blocks * pitch_of(steps_of(k)); }
inline size_t rows_bytes(uint32_t n, uint32_t k) { return codes_bytes(blocks_of(n), k) + (size_t)blocks_of(n) * kLine * 4; }
inline size_t image_bytes(uint32_t k, uint32_t m, bool gated) {
    const uint32_t b = blocks_of(m) * (gated ? 2 : 1);
    return codes_bytes(b, k) + (size_t)b * kLine * sizeof(double2);
}

// One product: x's image, the weight's image, and the output.
struct Prod {
    const int8_t* a;
    const int32_t* amax;
    const int8_t* w;
    const double2* cols;             // [32 blocks]: mu, 1.5 2^52 + bias
    uint32_t n, m, steps, rblocks, cblocks;
    void* out;
    uint64_t out_ld;
    const int32_t* res;              // kOut32
    uint64_t res_ld;
    uint32_t shift;
    const uint8_t* tab;              // a gate's: the sigmoid's pieces, or the activation's bytes (`len` of them)
    uint32_t len;
    double gscale, gneg, scale;      // SiLU: 2^sa, 2^(sa + 24), 2^(-18 - sc); a byte table: scale 2^-sc
};

// 1.5 2^52 + sat16(rne(acc a mu + b)): the low word is the result.
__device__ __forceinline__ double scaled(int32_t acc, double a, double2 c) {
    const double z = __builtin_fma((double)acc * a, c.x, c.y);
    return __builtin_fmin(__builtin_fmax(z, kMagic - 32768.0), kMagic + 32767.0);
}

// sat32(h + (o << shift)), o of 16 bits and shift at most 16.
__device__ __forceinline__ int32_t add_res(int32_t h, int32_t o, uint32_t shift) {
    return __builtin_elementwise_add_sat(h, (int32_t)((uint32_t)o << shift));
}

// act(g) u 2^-sc, rounded to even and saturated, of the two products zg, zu as `scaled` gives them.  SiLU by the row-ops
// rule (MULACT): s = sigma(|g|) at 2^-24 from the piece of m = |g| at 2^-14, silu(g) = rne(m s 2^-18) at 2^-20, for a negative
// g of s - 2^24.  m s and m 2^24 are exact in a double (2^29 2^26), and one fused multiply-add of both onto 1.5 2^70, whose
// last place is 2^18, is that rounding; so is the product with u (2^37 2^15) and its own rounding onto 1.5 2^52.
template <uint32_t MODE, class Tab>
__device__ __forceinline__ int32_t gate16(double zg, double zu, Tab tab, const Prod& p) {
    double f;
    if (MODE == kSiluGate) {
        const double g = zg - kMagic, m = __builtin_fabs(g) * p.gscale;
        const uint32_t av = (uint32_t)m, at = min(av, kPieces << 6);
        const uint2 e = *reinterpret_cast<const uint2*>(tab + ((at >> 3) & ~7u));     // {64 value, step to the next} of 64 pieces
        const uint32_t s = (e.x + __umul24(e.y, av & 63)) >> 6;
        f = __builtin_fma(m, (double)s, __builtin_fma(__builtin_fmin(g, 0.0), p.gneg, kMagic70)) - kMagic70;
    } else {
        const int32_t g = __double2loint(zg), a = max(g, -g);
        f = (double)(max(g, 0) - ((uint32_t)a < p.len ? (int32_t)tab[a] : 0));
    }
    const double z = __builtin_fma(f * (zu - kMagic), p.scale, kMagic);
    return __double2loint(__builtin_fmin(__builtin_fmax(z, kMagic - 32768.0), kMagic + 32767.0));
}

// ---------------------------------------------------------------- a weight's image
// The blocks of w (element (kk, j) at kk ks + j js), and the channels' parameters; a block of `part` 1 / 2 is
// every second one (gate, up).  Once a weight: a thread a 16-byte piece.
__global__ __launch_bounds__(256) void linear8_pack_kernel(const int8_t* __restrict__ w, uint64_t ks, uint64_t js,
                                                           const double* __restrict__ mult, const int32_t* __restrict__ bias,
                                                           int8_t* __restrict__ codes, double2* __restrict__ cols, uint32_t k,
                                                           uint32_t m, uint32_t steps, uint32_t blocks, uint32_t part) {
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;           // (block, step, piece, line)
    const uint64_t total = (uint64_t)blocks * steps * 128;
    if (id >= total) return;
    const uint32_t line = id & 31, kg = (uint32_t)(id >> 5) & 3;
    const uint64_t bs = id >> 7;
    const uint32_t st = (uint32_t)(bs % steps), b = (uint32_t)(bs / steps), j = b * kLine + line;
    const uint32_t to = part ? 2 * b + part - 1 : b;
    int8_t v[16];
    for (uint32_t e = 0; e < 16; e++) {
        const uint32_t kk = st * kStep + kg * 16 + e;
        v[e] = kk < k && j < m ? w[kk * ks + j * js] : (int8_t)0;
    }
    *reinterpret_cast<int4*>(codes + (uint64_t)to * pitch_of(steps) + st * kPiece + kg * 512 + line * 16) = *reinterpret_cast<const int4*>(v);
    if (st == 0 && kg == 0)
        cols[(uint64_t)to * kLine + line] = j < m ? make_double2(mult[j], kMagic + (bias ? (double)bias[j] : 0.0)) : make_double2(0.0, kMagic);
}

// ---------------------------------------------------------------- a row's codes
__device__ __forceinline__ uint32_t recip(uint32_t a) { return a ? (127u * (1u << 24) + (a >> 1)) / a : 0u; }

typedef short v2s __attribute__((ext_vector_type(2)));

// A row, or with ODD the element before one that starts between two 4-byte words: then loads are of the words that hold the row's
// elements, the first and the last of which may hold another's beside them (in the word of one of the row's, so no load leaves its
// page; shifted out before it counts), and `settle` moves them into place once they are there.  16 bytes a lane between two
// words take 1.4 us more: 16 rows of 1001 x 960 5.6 us, 4.6 with ODD; 4.2 at even strides, 4.4 with ODD.
template <bool ODD>
struct Row {
    const int16_t* p;
    uint32_t shift;                  // 0, or 16 bits for an element
};
template <bool ODD>
__device__ __forceinline__ Row<ODD> row_of(const int16_t* row) {
    const uint32_t m = ODD ? (uint32_t)(reinterpret_cast<uintptr_t>(row) >> 1) & 1u : 0;
    return Row<ODD>{row - m, 16 * m};
}

// 16 elements from k0 of a row of k (zeros past its end); with ODD as they come from memory, until `settle`.
template <bool ODD>
struct Piece {
    int4 v[2];
};
template <>
struct Piece<true> {
    int4 v[2];
    uint32_t last;
};
__device__ __forceinline__ int4 load8(const int16_t* p) {                   // 8 elements at any alignment
    int4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <bool ODD>
__device__ __forceinline__ Piece<ODD> load_piece(const Row<ODD>& r, uint32_t k0, uint32_t k) {
    constexpr uint32_t N = ODD ? 18 : 16;
    Piece<ODD> p;
    if (k0 + 16 <= k) {
        p.v[0] = load8(r.p + k0);
        p.v[1] = load8(r.p + k0 + 8);
        if constexpr (ODD) __builtin_memcpy(&p.last, r.p + k0 + (r.shift ? 16 : 14), 4);     // a word that holds one of them
    } else if (k0 < k) {
        int16_t e[N];                                      // the row's last elements, one by one
        const uint32_t m = ODD ? r.shift >> 4 : 0;
#pragma unroll
        for (uint32_t q = 0; q < N; q++) e[q] = k0 + q < k + m ? r.p[k0 + q] : (int16_t)0;
        __builtin_memcpy(p.v, e, 32);
        if constexpr (ODD) __builtin_memcpy(&p.last, e + 16, 4);
    } else {
        p.v[0] = p.v[1] = int4{0, 0, 0, 0};
        if constexpr (ODD) p.last = 0;
    }
    return p;
}
template <bool ODD>
__device__ __forceinline__ void settle(Piece<ODD>& p, const Row<ODD>& r) {
    if constexpr (ODD) {
        uint32_t w[9];
        __builtin_memcpy(w, p.v, 32);
        w[8] = p.last;
#pragma unroll
        for (int q = 0; q < 8; q++) w[q] = __builtin_amdgcn_alignbit(w[q + 1], w[q], r.shift);
        __builtin_memcpy(p.v, w, 32);
    }
}

// The largest and the smallest elements so far, two lanes of 16 bits each: |-32768| has no int16.
struct Range {
    v2s hi{0, 0}, lo{0, 0};
    template <bool ODD>
    __device__ __forceinline__ void add(const Piece<ODD>& p) {
        const v2s* e = reinterpret_cast<const v2s*>(p.v);
#pragma unroll
        for (int q = 0; q < 8; q++) {
            hi = __builtin_elementwise_max(hi, e[q]);
            lo = __builtin_elementwise_min(lo, e[q]);
        }
    }
    __device__ __forceinline__ int32_t top() const {
        return max(max((int32_t)hi[0], (int32_t)hi[1]), -min((int32_t)lo[0], (int32_t)lo[1]));
    }
};

// The largest of N maxima (N a multiple of 4, 16-byte aligned).
template <uint32_t N>
__device__ __forceinline__ int32_t top_of(const int32_t* part) {
    int32_t t = 0;
#pragma unroll
    for (uint32_t i = 0; i < N / 4; i++) {
        const int4 v = reinterpret_cast<const int4*>(part)[i];
        t = max(max(max(t, v.x), max(v.y, v.z)), v.w);
    }
    return t;
}

// The 16 codes of a piece: the top bytes of x R + 2^23.  `small`: every R of the wavefront is below 2^23 (maxima from 255 on),
// so that a 24-bit multiply-add does (full rate; a 32-bit product a quarter of it).
template <bool ODD>
__device__ __forceinline__ v4i codes_of(const Piece<ODD>& p, int32_t r, bool small) {
    const v2s* e = reinterpret_cast<const v2s*>(p.v);
    v4i out;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        int32_t t[4];
#pragma unroll
        for (int h = 0; h < 4; h++) {
            const int32_t x = e[2 * q + (h >> 1)][h & 1];
            t[h] = (small ? __mul24(x, r) : x * r) + (1 << 23);
        }
        const uint32_t a = __builtin_amdgcn_perm((uint32_t)t[1], (uint32_t)t[0], 0x0C0C0703u);
        const uint32_t b = __builtin_amdgcn_perm((uint32_t)t[3], (uint32_t)t[2], 0x0C0C0703u);
        out[q] = (int)(a | b << 16);
    }
    return out;
}

// RW rows a workgroup, a wavefront a row: its maximum, then its codes, 16 elements a lane and pass of 1024; rows of up to 1024 U
// elements stay in registers, U = 0: longer ones are read twice.  A pass's codes go through LDS, so that RW lanes
// write 16 RW consecutive bytes of a block.  Bound by memory for many rows (16 a workgroup: 8192 x 4096 19.0 us; a wavefront's
// own stores of 16 bytes a line 27), by latency for few (4 a workgroup: 512 x 2560 4.7 us, 16: 6.8).
template <int U, uint32_t RW>
__global__ __launch_bounds__(64 * RW) void linear8_rows_kernel(const int16_t* __restrict__ x, uint64_t ld, uint32_t n, uint32_t k,
                                                           int8_t* __restrict__ codes, int32_t* __restrict__ amax, uint32_t steps) {
    constexpr uint32_t PL = 16 * RW + 16;                  // bytes of a piece of RW rows in LDS: pieces in different banks
    __shared__ __attribute__((aligned(16))) int8_t sm[2][64 * PL];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row0 = blockIdx.x * RW, row = row0 + wave;
    const Row<false> r = row_of<false>(x + (uint64_t)min(row, n - 1) * ld);
    Range range;
    Piece<false> e[U ? U : 1];
    if constexpr (U != 0) {
#pragma unroll
        for (int i = 0; i < U; i++) e[i] = load_piece(r, 16 * lane + 1024 * i, k);
#pragma unroll
        for (int i = 0; i < U; i++) range.add(e[i]);
    } else {
        for (uint32_t k0 = 16 * lane; k0 < k; k0 += 1024) range.add(load_piece(r, k0, k));
    }
    int32_t top = range.top();
    for (int off = 32; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
    top = __builtin_amdgcn_readfirstlane(top);
    if (lane == 0 && row < n) amax[row] = top;
    const int32_t rc = (int32_t)recip((uint32_t)top);
    int8_t* to = codes + (uint64_t)(row0 >> 5) * pitch_of(steps) + (row0 & 31) * 16;
    const uint32_t piece = threadIdx.x / RW, line = threadIdx.x % RW;
    auto pass = [&](int i, const Piece<false>& p) {
        *reinterpret_cast<v4i*>(&sm[i & 1][lane * PL + wave * 16]) = codes_of(p, rc, rc < 1 << 23);
        lds_barrier();                                     // two buffers: one barrier a pass
        const uint32_t q = 64 * i + piece;
        if (q < 4 * steps && row0 + line < n)
            *reinterpret_cast<v4i*>(to + q * 512 + line * 16) = *reinterpret_cast<const v4i*>(&sm[i & 1][piece * PL + line * 16]);
    };
    if constexpr (U != 0) {
#pragma unroll
        for (int i = 0; i < U; i++)
            if (1024 * i < (int)k) pass(i, e[i]);          // the same for the whole workgroup
    } else {
        for (int i = 0; 1024 * i < (int)k; i++) pass(i, load_piece(r, 16 * lane + 1024 * i, k));
    }
}

// A row a workgroup, N pieces a lane: few rows, where the time is one row's latency.
template <uint32_t N>
__global__ __launch_bounds__(1024) void linear8_row_kernel(const int16_t* __restrict__ x, uint64_t ld, uint32_t k,
                                                          int8_t* __restrict__ codes, int32_t* __restrict__ amax, uint32_t steps) {
    __shared__ __attribute__((aligned(16))) int32_t part[16];
    const uint32_t row = blockIdx.x, W = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Row<false> r = row_of<false>(x + (uint64_t)row * ld);
    Piece<false> e[N];
    Range range;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) e[i] = load_piece(r, 16 * (threadIdx.x + i * blockDim.x), k);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) range.add(e[i]);
    int32_t top = range.top();
    for (int off = 32; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
    if (W > 1) {
        if (lane == 0)
            for (uint32_t i = wave; i < 16; i += W) part[i] = top;         // absent wavefronts' places too
        lds_barrier();
        top = top_of<16>(part);
    }
    top = __builtin_amdgcn_readfirstlane(top);
    if (threadIdx.x == 0) amax[row] = top;
    const int32_t rc = (int32_t)recip((uint32_t)top);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        const uint32_t q = threadIdx.x + i * blockDim.x;
        if (q < 4 * steps)
            *reinterpret_cast<v4i*>(codes + (uint64_t)(row >> 5) * pitch_of(steps) + (row & 31) * 16 + q * 512) = codes_of(e[i], rc, rc < 1 << 23);
    }
}

// ---------------------------------------------------------------- products
// What an output element needs besides its sums, loaded before them: its column's parameters and its residual.
struct Elem {
    double2 c0{}, c1{};
    int32_t h = 0;
};
template <uint32_t MODE>
__device__ __forceinline__ Elem element(const Prod& p, uint32_t row, uint32_t col) {
    Elem e;
    if (row >= p.n || col >= p.m) return e;
    const double2* c = p.cols + (gated(MODE) ? (col >> 5) * 64 + (col & 31) : col);
    e.c0 = c[0];
    if (gated(MODE)) e.c1 = c[32];
    if (MODE == kOut32) e.h = p.res[row * p.res_ld + col];
    return e;
}

// One output element from the sums of its column (a gate: of both).
template <uint32_t MODE>
__device__ __forceinline__ void store(const Prod& p, uint32_t row, uint32_t col, int32_t acc0, int32_t acc1, double a, const Elem& e) {
    if (row >= p.n || col >= p.m) return;
    const double z = scaled(acc0, a, e.c0);
    if (MODE == kOut32) {
        static_cast<int32_t*>(p.out)[row * p.out_ld + col] = add_res(e.h, __double2loint(z), p.shift);
    } else {
        const int32_t o = gated(MODE) ? gate16<MODE>(z, scaled(acc1, a, e.c1), p.tab, p) : __double2loint(z);
        static_cast<int16_t*>(p.out)[row * p.out_ld + col] = (int16_t)o;
    }
}

// ---------------------------------------------------------------- many rows
// LDS reads, LDS copies and vector memory each move 64 bytes a cycle and compute unit (measured), an i8 MFMA of 32 x
// 32 x 32 takes 32 cycles: what bounds a product is how often its operands pass through those two ports.  So a
// wavefront takes 64 rows by 128 columns, four of them side by side over the same columns: x's fragments, which no other
// wavefront reads, go from memory straight into registers, D steps ahead; the weight's columns go through a ring of
// D LDS stages, copied D steps ahead.  A 64-k step of two such workgroups on a compute unit is 1024 cycles of MFMA
// on each SIMD, 64 KiB of LDS reads, 16 KiB of copies and 32 KiB of loads.  Operand pieces lie in memory, in LDS and in the
// registers in one order (a lane's 16 bytes at 16 lane): whole lines, no bank conflict.  Fewer rows take a wavefront of 32
// rows by 128 or 64 columns (RB, CB: blocks of a wavefront): half or a quarter of a workgroup's work, for a chip with fewer
// tiles than it holds.  D is 3 where the registers hold no more (RB 2), else 4: operands past the L2 come too late for 3
// (512 x 8192 x 1024 in 128 x 64 tiles 25.4 us, 4 stages 19.4, 6 19.3; 128 x 2560 x 960 6.8 / 6.8 / 7.0).
// Buffer accesses: a block's base in scalar registers, the lane's 16 bytes in one vector register, the step's offset
// scalar.  Copies to LDS go this way and not as global_load_lds, which the compiler counts as a flat access: every wait
// for a register load or an LDS read behind one becomes a wait for all (8192 x 4096 x 8192: 268 us, 260 this way).
// Both are marked volatile: a wait below counts the accesses behind a copy, so none of them may move over another.
typedef __amdgpu_buffer_rsrc_t Buf;
constexpr int kVolatile = (int)0x80000000;
__device__ __forceinline__ Buf buffer_of(const int8_t* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ void lds_copy16(Buf b, uint32_t lane_at, uint32_t at, int8_t* lds_wave_base) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void*)lds_wave_base, 16, (int)lane_at, (int)at, 0, kVolatile);
}
__device__ __forceinline__ v4i load16(Buf b, uint32_t lane_at, uint32_t at) {
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(b, (int)lane_at, (int)at, kVolatile));
}

template <int N>
__device__ __forceinline__ void wait_copies() {            // at most N of this wavefront's copies outstanding, LDS reads done
    static_assert(N >= 0 && N < 64, "vmcnt is six bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
}

// The output tile of workgroup x: the workgroups of an XCD (one residue mod 8) take a contiguous run of an order that
// walks strips of xw tile columns row by row, so that its L2 holds the operands of a block of tiles.
struct Tile {
    uint32_t r, c;
};
__device__ __forceinline__ Tile tile_of(uint32_t x, uint32_t tiles_r, uint32_t tiles_c, uint32_t xw) {
    const uint32_t tiles = tiles_r * tiles_c, q = tiles >> 3, res = x & 7;
    const uint32_t at = res * q + min(res, tiles & 7) + (x >> 3);
    const uint32_t strip = at / (tiles_r * xw), in = at - strip * tiles_r * xw;
    const uint32_t w = min(xw, tiles_c - strip * xw), row = in / w;
    return Tile{row, strip * xw + in - row * w};
}

// The outputs of a wavefront's RB x CB blocks: a lane holds column l32 of a block, its rows 8 (r / 4) + 4 lh + r % 4.  Through
// buffer accesses, which drop what lies past the last row and, at an offset past every row, past the last column.
template <uint32_t MODE, int RB, int CB, class Tab>
__device__ __forceinline__ void epilogue(const Prod& p, const v16i (&acc)[RB][CB], uint32_t rb0, uint32_t cb0, uint32_t l32,
                                         uint32_t lh, Tab tab) {
    constexpr uint32_t E = MODE == kOut32 ? 4 : 2;
    constexpr int ST = gated(MODE) ? 2 : 1;
    const uint32_t ld = (uint32_t)p.out_ld, rld = (uint32_t)p.res_ld;
#pragma unroll
    for (int i = 0; i < RB; i++) {
        const uint32_t row0 = (rb0 + i) * kLine;
        if (row0 >= p.n) break;
        const uint32_t rows = min(p.n - row0, kLine);
        const Buf ob = buffer_of(static_cast<int8_t*>(p.out) + (uint64_t)row0 * p.out_ld * E, ((rows - 1) * ld + p.m) * E);
        Buf hb;
        if constexpr (MODE == kOut32)
            hb = buffer_of(reinterpret_cast<const int8_t*>(p.res) + (uint64_t)row0 * p.res_ld * E, ((rows - 1) * rld + p.m) * E);
        double am[16];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int4 v = *reinterpret_cast<const int4*>(p.amax + row0 + 8 * q + 4 * lh);
            am[4 * q] = v.x, am[4 * q + 1] = v.y, am[4 * q + 2] = v.z, am[4 * q + 3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < CB; j += ST) {
            const uint32_t blk = cb0 + j, col = (gated(MODE) ? blk >> 1 : blk) * kLine + l32;
            const double2 c0 = p.cols[min(blk, p.cblocks - 1) * kLine + l32];
            const double2 c1 = gated(MODE) ? p.cols[min(blk + 1, p.cblocks - 1) * kLine + l32] : double2{};
            const uint32_t at = col < p.m ? (4 * lh * ld + col) * E : 0x80000000u;
            int32_t h[16];
            if constexpr (MODE == kOut32) {
                const uint32_t rat = col < p.m ? (4 * lh * rld + col) * E : 0x80000000u;
#pragma unroll
                for (int r = 0; r < 16; r++)
                    h[r] = __builtin_amdgcn_raw_buffer_load_b32(hb, (int)(rat + (8 * (r >> 2) + (r & 3)) * rld * E), 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const double z = scaled(acc[i][j][r], am[r], c0);
                const int to = (int)(at + (8 * (r >> 2) + (r & 3)) * ld * E);
                if constexpr (MODE == kOut32) {
                    __builtin_amdgcn_raw_buffer_store_b32(add_res(h[r], __double2loint(z), p.shift), ob, to, 0, 0);
                } else {
                    int32_t o = __double2loint(z);
                    if constexpr (gated(MODE)) o = gate16<MODE>(z, scaled(acc[i][j + 1][r], am[r], c1), tab, p);
                    __builtin_amdgcn_raw_buffer_store_b16((short)o, ob, to, 0, 0);
                }
            }
            if constexpr (MODE == kOut32) __builtin_amdgcn_sched_barrier(0);     // a block's residuals in registers at a time
        }
    }
}

template <uint32_t MODE, int RB, int CB>
__global__ __launch_bounds__(256, 2) void linear8_ring_kernel(Prod p, uint32_t tiles_r, uint32_t tiles_c, uint32_t xw) {
    constexpr int WR = 4, NC = 2 * CB / WR;                // wavefronts; copies a wavefront and step
    constexpr int D = RB == 1 ? 4 : 3;                     // stages
    __shared__ __attribute__((aligned(1024))) int8_t sm0[2 * CB * 1024];
    __shared__ __attribute__((aligned(1024))) int8_t sm1[2 * CB * 1024];
    __shared__ __attribute__((aligned(1024))) int8_t sm2[2 * CB * 1024];
    __shared__ __attribute__((aligned(1024))) int8_t sm3[D > 3 ? 2 * CB * 1024 : 16];
    // a gate's table, for gathers of 64 lanes; it lands before the ring's first copies
    constexpr int TAB = MODE == kSiluGate ? kSigmoidBytes : MODE == kTableGate ? kActTabBytes : 16;
    __shared__ __attribute__((aligned(1024))) int8_t tab[TAB];
    const Tile t = tile_of(blockIdx.x, tiles_r, tiles_c, xw);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t l32 = lane & 31, lh = lane >> 5;
    const uint32_t rb0 = (t.r * WR + wave) * RB, cb0 = t.c * CB;
    // blocks past the last: any, never stored
    const uint32_t line = pitch_of(p.steps);               // bytes of a block of lines
    Buf xa[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) xa[i] = buffer_of(p.a + (uint64_t)min(rb0 + i, p.rblocks - 1) * line, line);
    const Buf wb = buffer_of(p.w + (uint64_t)cb0 * line, min(p.cblocks - cb0, (uint32_t)CB) * line);
    uint32_t wq[NC];
#pragma unroll
    for (int i = 0; i < NC; i++) {                         // piece q of a stage: block q / 2, substep q % 2
        const uint32_t q = wave * NC + i;
        wq[i] = min(q >> 1, p.cblocks - 1 - cb0) * line + (q & 1) * 1024;
    }
    const uint32_t l16 = lane * 16;
    v16i acc[RB][CB];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int j = 0; j < CB; j++) acc[i][j] = v16i{};
    v4i a[D][2][RB], b[2][CB];
    auto at = [&](uint32_t step) { return min(step, p.steps - 1) * kPiece; };       // past the last step: any, never used
    auto issue = [&](int8_t* sm, uint32_t step) {
#pragma unroll
        for (int i = 0; i < NC; i++) lds_copy16(wb, l16, wq[i] + at(step), sm + (wave * NC + i) * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load = [&](int slot, int s, uint32_t step) {
#pragma unroll
        for (int i = 0; i < RB; i++) a[slot][s][i] = load16(xa[i], l16, at(step) + s * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto fragments = [&](const int8_t* sm, int s) {
#pragma unroll
        for (int j = 0; j < CB; j++) b[s][j] = *reinterpret_cast<const v4i*>(sm + (2 * j + s) * 1024 + l16);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto products = [&](int slot, int s) {
#pragma unroll
        for (int j = 0; j < CB; j++)
#pragma unroll
            for (int i = 0; i < RB; i++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[slot][s][i], b[s][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // Step kt + slot, its first weight fragments read: the second ones are read under the first products, the next step's
    // first ones under the second, behind the barrier that frees its stage for D steps later and says that the next
    // step has landed.  Behind that one's copies this wavefront has copied D - 2 times more (NC each) and, in the loop,
    // loaded x 2 (D - 1) times (RB each: the loads of a later step that feed no product may be left out by the compiler, so the
    // steps behind the loop count none).  No copy is conditional: with a path that skips one the compiler waits for
    // every copy in flight before it reads a stage.
    auto stage = [&](auto i) -> int8_t* {
        if constexpr (i.value % D == 0) return sm0;
        else if constexpr (i.value % D == 1) return sm1;
        else if constexpr (i.value % D == 2) return sm2;
        else return sm3;
    };
    uint32_t kt = 0;
    auto step = [&](auto slot, auto loads) {
        int8_t* const cur = stage(slot);
        const int8_t* const next = stage(std::integral_constant<int, slot.value + 1>{});
        const uint32_t to = kt + slot.value + D;
        fragments(cur, 1);
        products(slot.value, 0);
        wait_copies<(D - 2) * NC + loads.value>();
        __builtin_amdgcn_s_barrier();
        issue(cur, to);
        load(slot.value, 0, to);
        fragments(next, 0);
        products(slot.value, 1);
        load(slot.value, 1, to);
    };
    constexpr std::integral_constant<int, 2 * (D - 1) * RB> in_loop{};
    constexpr std::integral_constant<int, 0> behind{};
    if constexpr (gated(MODE)) {
        const Buf tb = buffer_of(reinterpret_cast<const int8_t*>(p.tab), TAB);
#pragma unroll
        for (int i = 0; i < TAB / 1024 / WR; i++) lds_copy16(tb, l16, (wave * (TAB / 1024 / WR) + i) * 1024, tab + (wave * (TAB / 1024 / WR) + i) * 1024);
        __builtin_amdgcn_sched_barrier(0);
    }
    auto first = [&](auto slot) {
        issue(stage(slot), slot.value);
        load(slot.value, 0, slot.value);
        load(slot.value, 1, slot.value);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto each = [&](auto f) {                        // f of 0 .. D - 1
        f(std::integral_constant<int, 0>{}), f(std::integral_constant<int, 1>{}), f(std::integral_constant<int, 2>{});
        if constexpr (D > 3) f(std::integral_constant<int, 3>{});
    };
    each(first);
    wait_copies<(D - 1) * NC>();                     // x's first loads may have moved behind the copies
    __builtin_amdgcn_s_barrier();
    fragments(sm0, 0);
    for (; kt + D <= p.steps; kt += D) each([&](auto i) { step(i, in_loop); });
    each([&](auto i) {
        if constexpr (i.value < D - 1)
            if (kt + i.value < p.steps) step(i, behind);
    });
    wait_copies<0>();                                // no copy may land after the workgroup ends

    epilogue<MODE, RB, CB>(p, acc, rb0, cb0, l32, lh, (const uint8_t*)tab);
}

// ---------------------------------------------------------------- a few tiles
// Products of too few rows to fill the chip with the tiles above: a workgroup computes 32 RB x 32 CB outputs, its wavefronts
// taking the 64-k steps in turn with operands straight from memory (nothing waits on another wavefront, two steps in flight), and
// adds their sums in LDS (integer adds: any order).  Bound by the latency of the few steps a wavefront has.
constexpr uint32_t kMidWaves = 4;

template <uint32_t MODE, int CB>
__global__ __launch_bounds__(64 * kMidWaves) void linear8_mid_kernel(Prod p, uint32_t tiles_r, uint32_t tiles_c, uint32_t xw) {
    constexpr uint32_t R = 32, COLS = 32 * CB, OUT = gated(MODE) ? COLS / 2 : COLS;
    constexpr uint32_t LD = COLS + 8;                // rows four apart 32 banks apart
    static_assert(!gated(MODE) || CB % 2 == 0, "gate beside up");
    __shared__ int32_t red[R * LD];
    const Tile t = tile_of(blockIdx.x, tiles_r, tiles_c, xw);
    const uint32_t W = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t l32 = lane & 31, lh = lane >> 5, l16 = lane * 16, row0 = t.r * R, cb0 = t.c * CB;
    const uint32_t line = pitch_of(p.steps);
    const Buf xa = buffer_of(p.a + (uint64_t)t.r * line, line);
    Buf wb[CB];                                      // blocks past the last: any, never stored
#pragma unroll
    for (int j = 0; j < CB; j++) wb[j] = buffer_of(p.w + (uint64_t)min(cb0 + j, p.cblocks - 1) * line, line);
    v4i a[2][2], b[2][2][CB];
    auto load = [&](int slot, uint32_t step) {
        const uint32_t at = min(step, p.steps - 1) * kPiece;       // past the last step: any, never used
#pragma unroll
        for (int s = 0; s < 2; s++) {
            a[slot][s] = load16(xa, l16, at + s * 1024);
#pragma unroll
            for (int j = 0; j < CB; j++) b[slot][s][j] = load16(wb[j], l16, at + s * 1024);
        }
    };
    v16i acc[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) acc[j] = v16i{};
    auto products = [&](int slot) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < CB; j++) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[slot][s], b[slot][s][j], acc[j], 0, 0, 0);
    };
    load(0, wave);
    load(1, wave + W);
    const uint32_t col0 = (gated(MODE) ? cb0 / 2 : cb0) * kLine;
    const Elem el = element<MODE>(p, row0 + threadIdx.x / OUT, col0 + threadIdx.x % OUT);
    for (uint32_t e = threadIdx.x; e < R * LD; e += blockDim.x) red[e] = 0;
    for (uint32_t st = wave; st < p.steps; st += 2 * W) {
        products(0);
        load(0, st + 2 * W);
        if (st + W < p.steps) products(1);
        load(1, st + 3 * W);
    }
    lds_barrier();                                   // red is zeros
#pragma unroll
    for (int j = 0; j < CB; j++)
#pragma unroll
        for (int r = 0; r < 16; r++)
            __hip_atomic_fetch_add(&red[(8 * (r >> 2) + 4 * lh + (r & 3)) * LD + 32 * j + l32], acc[j][r], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_WORKGROUP);
    lds_barrier();
    auto put = [&](uint32_t e, const Elem& x) {
        const uint32_t rl = e / OUT, cl = e % OUT, row = row0 + rl;
        const uint32_t at = gated(MODE) ? (cl >> 5) * 64 + (cl & 31) : cl;
        const int32_t s0 = red[rl * LD + at], s1 = gated(MODE) ? red[rl * LD + at + 32] : 0;
        store<MODE>(p, row, col0 + cl, s0, s1, (double)p.amax[min(row, p.n - 1)], x);
    };
    put(threadIdx.x, el);
    for (uint32_t e = threadIdx.x + blockDim.x; e < R * OUT; e += blockDim.x)
        put(e, element<MODE>(p, row0 + e / OUT, col0 + e % OUT));
}

// The same from x: 32 rows by 32 CB columns, S steps a wavefront; the rows' pieces stay in registers while their maxima meet in
// LDS and become codes there, as in the kernel of few rows: one launch instead of two.
constexpr uint32_t kDirectWaves = 8, kDirectSteps = 3;

template <uint32_t MODE, int CB, int S, bool ODD>
__global__ __launch_bounds__(64 * kDirectWaves) void linear8_mid_direct_kernel(Prod p, const int16_t* __restrict__ x, uint64_t ld, uint32_t k,
                                                                      uint32_t tiles_r, uint32_t tiles_c, uint32_t xw) {
    constexpr uint32_t R = 32, COLS = 32 * CB, OUT = gated(MODE) ? COLS / 2 : COLS, MW = kDirectWaves;
    constexpr uint32_t LD = COLS + 8;                // rows four apart 32 banks apart
    static_assert(!gated(MODE) || CB % 2 == 0, "gate beside up");
    __shared__ int32_t red[R * LD];
    __shared__ __attribute__((aligned(16))) int32_t part[R * MW];
    __shared__ int32_t top[R];
    const Tile t = tile_of(blockIdx.x, tiles_r, tiles_c, xw);
    const uint32_t W = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t l32 = lane & 31, lh = lane >> 5, l16 = lane * 16, row0 = t.r * R, cb0 = t.c * CB;
    const uint32_t line = pitch_of(p.steps);
    Buf wb[CB];                                      // blocks past the last: any, never stored
#pragma unroll
    for (int j = 0; j < CB; j++) wb[j] = buffer_of(p.w + (uint64_t)min(cb0 + j, p.cblocks - 1) * line, line);
    v4i a[S][2], b[S][2][CB];
    auto load = [&](int slot, uint32_t step) {
        const uint32_t at = min(step, p.steps - 1) * kPiece;       // past the last step: any, its codes are zeros
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < CB; j++) b[slot][s][j] = load16(wb[j], l16, at + s * 1024);
    };
    const Row<ODD> xr = row_of<ODD>(x + (uint64_t)min(row0 + l32, p.n - 1) * ld);
    Piece<ODD> xv[S][2];
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) xv[i][s] = load_piece(xr, (wave + i * W) * kStep + 32 * s + 16 * lh, k);
#pragma unroll
    for (int i = 0; i < S; i++) load(i, wave + i * W);
    const uint32_t col0 = (gated(MODE) ? cb0 / 2 : cb0) * kLine;
    const Elem el = element<MODE>(p, row0 + threadIdx.x / OUT, col0 + threadIdx.x % OUT);
    for (uint32_t e = threadIdx.x; e < R * LD; e += blockDim.x) red[e] = 0;
    Range range;
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            settle(xv[i][s], xr);
            range.add(xv[i][s]);
        }
    int32_t am = range.top();
    am = max(am, __shfl_xor(am, 32, 64));
    if (lh == 0)
        for (uint32_t i = wave; i < MW; i += W) part[l32 * MW + i] = am;       // the places of absent wavefronts too
    lds_barrier();
    am = top_of<MW>(part + l32 * MW);
    if (wave == 0 && lh == 0) top[l32] = am;
    const int32_t rc = (int32_t)recip((uint32_t)am);
    const bool small = __all(rc < 1 << 23);
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) a[i][s] = codes_of(xv[i][s], rc, small);
    v16i acc[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) acc[j] = v16i{};
#pragma unroll
    for (int i = 0; i < S; i++)
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < CB; j++) acc[j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i][s], b[i][s][j], acc[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < CB; j++)
#pragma unroll
        for (int r = 0; r < 16; r++)
            __hip_atomic_fetch_add(&red[(8 * (r >> 2) + 4 * lh + (r & 3)) * LD + 32 * j + l32], acc[j][r], __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_WORKGROUP);
    lds_barrier();
    auto put = [&](uint32_t e, const Elem& x) {
        const uint32_t rl = e / OUT, cl = e % OUT;
        const uint32_t at = gated(MODE) ? (cl >> 5) * 64 + (cl & 31) : cl;
        const int32_t s0 = red[rl * LD + at], s1 = gated(MODE) ? red[rl * LD + at + 32] : 0;
        store<MODE>(p, row0 + rl, col0 + cl, s0, s1, (double)top[rl], x);
    };
    if (threadIdx.x < R * OUT) put(threadIdx.x, el);
    for (uint32_t e = threadIdx.x + blockDim.x; e < R * OUT; e += blockDim.x)
        put(e, element<MODE>(p, row0 + e / OUT, col0 + e % OUT));
}

// ---------------------------------------------------------------- few rows
// At most 16 RF rows: the weight is read once and the time is the latency of a launch, of x and of a
// weight's bytes.  A workgroup of W wavefronts takes NF fragments of 16 columns (a gate: half gate, half up) at
// all of k, the wavefronts its 64-k steps in turn; their sums meet in LDS (integer adds: any order).  With
// x (DIRECT) a wavefront loads its own steps' pieces of the rows in the operand's layout, keeps them
// in registers while the rows' maxima meet in LDS, and turns them into codes there: x is read once, no launch
// and no memory between (S steps a wavefront, all of k).  Without, the codes are read, S steps at a time.
// Further units of columns reuse a direct call's codes.
constexpr uint32_t kFewWaves = 16, kFewSteps = 4;

template <uint32_t NF>
__device__ __forceinline__ void load_weights(v4i (&b)[NF], const int8_t* const (&w)[NF], uint32_t step) {
#pragma unroll
    for (uint32_t f = 0; f < NF; f++) b[f] = *reinterpret_cast<const v4i*>(w[f] + (uint64_t)step * kPiece);
}

template <uint32_t MODE, uint32_t RF, uint32_t NF, uint32_t S, bool DIRECT, bool ODD>
__global__ __launch_bounds__(64 * kFewWaves) void linear8_few_kernel(Prod p, const int16_t* __restrict__ x, uint64_t ld, uint32_t k) {
    constexpr uint32_t R = 16 * RF, COLS = 16 * NF, OUT = gated(MODE) ? COLS / 2 : COLS;
    constexpr uint32_t LD = COLS + 4;                // the four k groups' rows in different banks
    __shared__ int32_t red[R * LD];                  // the unit's sums, zeros between units
    __shared__ __attribute__((aligned(16))) int32_t part[R * kFewWaves];       // the rows' maxima: of a wavefront's pieces,
    __shared__ int32_t top[R];                                                 // and all
    const uint32_t W = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint32_t units = (p.m + OUT - 1) / OUT;
    const int8_t* w[NF];
    // fragment f of unit u: its column block and half (a gate's blocks alternate)
    auto weights_of = [&](uint32_t u) {
#pragma unroll
        for (uint32_t f = 0; f < NF; f++) {
            constexpr uint32_t per = gated(MODE) ? NF / 2 : NF;
            const uint32_t q = u * per + f % per;
            const uint32_t blk = gated(MODE) ? 2 * (q >> 1) + f / per : q >> 1;
            // columns past the last block: any, never stored
            w[f] = p.w + (uint64_t)min(blk, p.cblocks - 1) * pitch_of(p.steps) + g * 512 + (q & 1) * 256 + c * 16;
        }
    };
    uint32_t u = blockIdx.x;
    weights_of(u);
    v4i a[S][RF], b[S][NF];
    Elem el = element<MODE>(p, threadIdx.x / OUT, u * OUT + threadIdx.x % OUT);
    for (uint32_t e = threadIdx.x; e < R * LD; e += blockDim.x) red[e] = 0;
    if constexpr (DIRECT) {
        Piece<ODD> xv[S][RF];
        Row<ODD> xr[RF];
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) xr[f] = row_of<ODD>(x + (uint64_t)min(16 * f + c, p.n - 1) * ld);
#pragma unroll
        for (uint32_t i = 0; i < S; i++)
#pragma unroll
            for (uint32_t f = 0; f < RF; f++) xv[i][f] = load_piece(xr[f], (wave + i * W) * kStep + 16 * g, k);
#pragma unroll
        for (uint32_t i = 0; i < S; i++)
            if (wave + i * W < p.steps) load_weights<NF>(b[i], w, wave + i * W);
        // the rows' maxima: this wavefront's pieces, its four k groups, then the wavefronts
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) {
            Range range;
#pragma unroll
            for (uint32_t i = 0; i < S; i++) {
                settle(xv[i][f], xr[f]);
                range.add(xv[i][f]);
            }
            int32_t t = range.top();
            t = max(t, __shfl_xor(t, 16, 64));
            t = max(t, __shfl_xor(t, 32, 64));
            if (g == 0)
                for (uint32_t i = wave; i < kFewWaves; i += W) part[(16 * f + c) * kFewWaves + i] = t;     // absent wavefronts' too
        }
        lds_barrier();
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) {
            const int32_t am = top_of<kFewWaves>(part + (16 * f + c) * kFewWaves);
            if (wave == 0 && g == 0) top[16 * f + c] = am;
            const int32_t rc = (int32_t)recip((uint32_t)am);
            const bool small = __all(rc < 1 << 23);
#pragma unroll
            for (uint32_t i = 0; i < S; i++) a[i][f] = codes_of(xv[i][f], rc, small);
        }
    } else {
        lds_barrier();                               // red is zeros
    }
    for (;;) {
        v4i sum[RF][NF];
#pragma unroll
        for (uint32_t f = 0; f < RF; f++)
#pragma unroll
            for (uint32_t q = 0; q < NF; q++) sum[f][q] = v4i{0, 0, 0, 0};
        // one round of S steps if direct, else as many as k takes
        for (uint32_t s0 = wave; s0 < p.steps; s0 += S * W) {
            if constexpr (!DIRECT) {
#pragma unroll
                for (uint32_t i = 0; i < S; i++) {
                    const uint32_t st = min(s0 + i * W, p.steps - 1);
                    load_weights<NF>(b[i], w, st);
#pragma unroll
                    for (uint32_t f = 0; f < RF; f++)
                        a[i][f] = *reinterpret_cast<const v4i*>(p.a + (uint64_t)st * kPiece + g * 512 + f * 256 + c * 16);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < S; i++) {
                if (s0 + i * W >= p.steps) break;
#pragma unroll
                for (uint32_t q = 0; q < NF; q++)
#pragma unroll
                    for (uint32_t f = 0; f < RF; f++)
                        sum[f][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i][f], b[i][q], sum[f][q], 0, 0, 0);
            }
        }
        const uint32_t next = u + gridDim.x;
        if (next < units) {                          // the next unit's weights travel while this one's sums meet
            weights_of(next);
            if constexpr (DIRECT) {
#pragma unroll
                for (uint32_t i = 0; i < S; i++)
                    if (wave + i * W < p.steps) load_weights<NF>(b[i], w, wave + i * W);
            }
        }
#pragma unroll
        for (uint32_t f = 0; f < RF; f++)
#pragma unroll
            for (uint32_t q = 0; q < NF; q++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    __hip_atomic_fetch_add(&red[(16 * f + 4 * g + i) * LD + 16 * q + c], sum[f][q][i], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_WORKGROUP);
        lds_barrier();
        auto put = [&](uint32_t e, const Elem& x) {
            const uint32_t row = e / OUT, cl = e % OUT;
            const int32_t s0 = red[row * LD + cl], s1 = gated(MODE) ? red[row * LD + OUT + cl] : 0;
            red[row * LD + cl] = 0;
            if (gated(MODE)) red[row * LD + OUT + cl] = 0;
            store<MODE>(p, row, u * OUT + cl, s0, s1, (double)(DIRECT ? top[row] : p.amax[min(row, p.n - 1)]), x);
        };
        if (threadIdx.x < R * OUT) put(threadIdx.x, el);
        for (uint32_t e = threadIdx.x + blockDim.x; e < R * OUT; e += blockDim.x)
            put(e, element<MODE>(p, e / OUT, u * OUT + e % OUT));
        if (next >= units) return;
        u = next;
        el = element<MODE>(p, threadIdx.x / OUT, u * OUT + threadIdx.x % OUT);
        lds_barrier();                               // red is zeros again
    }
}

// ---------------------------------------------------------------- calls
int check_weight(const char* what, const cm_linear8_weight* w, bool gated) {
    if (w == nullptr || w->image == nullptr) return fail(CM_EINVAL, "%s: a null weight", what);
    if (w->k == 0 || w->k > kMaxK || w->m == 0 || w->m > kMaxM)
        return fail(CM_EINVAL, "%s: a weight of %u x %u (up to %u x %u)", what, w->k, w->m, kMaxK, kMaxM);
    if ((w->gated != 0) != gated) return fail(CM_EINVAL, "%s: the weight is %sgated", what, gated ? "not " : "");
    if (reinterpret_cast<uintptr_t>(w->image) & 255u) return fail(CM_EALIGN, "%s: the image must be 256-byte aligned", what);
    if (gated && (w->act > kGeluTanh || w->gate_shift > 14 || w->out_shift > 63))
        return fail(CM_EINVAL, "%s: activation %u, shifts %u and %u", what, w->act, w->gate_shift, w->out_shift);
    return CM_OK;
}

template <uint32_t RW>
int quantise_at(const int16_t* x, uint64_t x_ld, int8_t* codes, int32_t* amax, uint32_t n, uint32_t k, hipStream_t s) {
#define CM_ROWS(U) \
    CM_LAUNCH("linear8_rows_kernel", (linear8_rows_kernel<U, RW>), dim3(ceil_div(n, RW)), dim3(64 * RW), 0, s, x, x_ld, n, k, codes, amax, steps_of(k))
    if (k <= 1024) { CM_ROWS(1); }
    else if (k <= 2048) { CM_ROWS(2); }
    else if (k <= 4096) { CM_ROWS(4); }
    else if (k <= 8192) { CM_ROWS(8); }
    else { CM_ROWS(0); }
#undef CM_ROWS
    return CM_OK;
}

int quantise(const DeviceState* st, const int16_t* x, uint64_t x_ld, void* rows, uint32_t n, uint32_t k, hipStream_t s) {
    int8_t* codes = static_cast<int8_t*>(rows);
    int32_t* amax = reinterpret_cast<int32_t*>(codes + codes_bytes(blocks_of(n), k));
    // A row a workgroup up to a row a compute unit, and up to 1024 rows of more than 8192, which no wavefront's registers hold
    // (rows x k, us a row / four rows a workgroup): 16 x 2560 2.9 / 3.3, 256 x 2560 3.4 / 3.5, 512 x 2560 4.0 / 3.5; 16 x
    // 16384 3.5 / 11.2, 512 x 16384 10.1 / 15.8, 2048 x 16384 33.9 / 26.4.
    if (n <= (k > 8192 ? 1024u : (uint32_t)st->cus)) {
        if (k <= 16384) {
            CM_LAUNCH("linear8_rows_kernel", linear8_row_kernel<1>, dim3(n), dim3(64 * ceil_div(k, 1024)), 0, s, x, x_ld, k, codes, amax, steps_of(k));
        } else {
            CM_LAUNCH("linear8_rows_kernel", linear8_row_kernel<2>, dim3(n), dim3(1024), 0, s, x, x_ld, k, codes, amax, steps_of(k));
        }
        return CM_OK;
    }
    return n <= 16 * (uint32_t)st->cus ? quantise_at<4>(x, x_ld, codes, amax, n, k, s) : quantise_at<16>(x, x_ld, codes, amax, n, k, s);
}

int check_rows(const char* what, const int16_t* x, uint64_t x_ld, const void* rows, uint32_t n, uint32_t k) {
    if (n > kMaxN) return fail(CM_EINVAL, "%s: %u rows (up to %u)", what, n, kMaxN);
    if (n == 0) return CM_OK;
    if ((x == nullptr) == (rows == nullptr)) return fail(CM_EINVAL, "%s: either x or its codes", what);
    if (reinterpret_cast<uintptr_t>(x) & 1u) return fail(CM_EALIGN, "%s: x is not 2-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(rows) & 255u) return fail(CM_EALIGN, "%s: the codes must be 256-byte aligned", what);
    if (x != nullptr && n > 1 && x_ld < k) return fail(CM_EINVAL, "%s: rows of %u columns overlap at a stride of %llu", what, k, (unsigned long long)x_ld);
    return CM_OK;
}

// May a row start between two 4-byte words?
bool odd_rows(const int16_t* x, uint64_t ld) { return (reinterpret_cast<uintptr_t>(x) & 2u) != 0 || (ld & 1u) != 0; }

// Few rows.  A workgroup takes 16 columns (a gate 16 of each), 32 where two workgroups of 16 a compute unit do not reach.
constexpr uint32_t kFewPerCu = 2;
uint32_t few_cap(const DeviceState* st) { return kFewPerCu * (uint32_t)st->cus; }
uint32_t few_steps(const Prod& p) { return ceil_div(p.steps, std::min(kFewWaves, p.steps)); }

// From x in one launch, or codes first?  What the one launch repeats in every workgroup is the quantisation: a wavefront's
// steps, twice for more than 16 rows, times the workgroups a compute unit runs.  Up to 3 of those cost less than the second
// launch (us, one / two; columns x rows): 960 x 4096 of 1 row 3.8 / 5.2, of 16 4.4 / 5.4, of 32 6.4 / 5.9; 2048 x 4096 of 16 5.9 /
// 6.2; 2560 x 960 of 16 7.1 / 6.6 (0.5 for a launch less on the host); 4096 x 4096 of 16 8.6 / 7.5, of 1 6.2 / 7.2; 2048 x 16384
// of 1 8.8 / 7.8, of 16 10.6 / 8.1; 960 x 49152 of 16 10.2 / 12.9.
bool few_direct(const DeviceState* st, const Prod& p) {
    const uint32_t cus = (uint32_t)st->cus, wgs = std::min(ceil_div(p.m, 16), few_cap(st)), per = few_steps(p);
    if (p.n > 16) return per == 1 && wgs <= cus;
    return per * std::max(wgs, cus) <= 3 * cus || (p.n <= 4 && per <= 4 && wgs <= cus);
}

template <uint32_t MODE>
int few_rows(const DeviceState* st, const Prod& p, const int16_t* x, uint64_t ld, uint32_t k, hipStream_t s) {
    constexpr uint32_t P = gated(MODE) ? 2 : 1;
    const uint32_t cap = few_cap(st), per = few_steps(p);
    const dim3 block(64 * std::min(kFewWaves, p.steps)), narrow(std::min(ceil_div(p.m, 16), cap)), wide(std::min(ceil_div(p.m, 32), cap));
    const bool odd = odd_rows(x, ld);
#define CM_FEW(RF, NF, S, D, G)                                                                                                 \
    if (D && odd) {                                                                                                             \
        CM_LAUNCH("linear8_few_kernel", (linear8_few_kernel<MODE, RF, NF, S, D, D>), G, block, 0, s, p, x, ld, k);              \
    } else {                                                                                                                    \
        CM_LAUNCH("linear8_few_kernel", (linear8_few_kernel<MODE, RF, NF, S, D, false>), G, block, 0, s, p, x, ld, k);          \
    }
    if (p.n > 16) {
        if (x != nullptr) { CM_FEW(2, P, 1, true, narrow); }
        else { CM_FEW(2, P, kFewSteps, false, narrow); }
    } else if (p.m > 16 * cap) {                     // columns again and again for a workgroup: a step a wavefront if from x
        if (x != nullptr) { CM_FEW(1, 2 * P, 1, true, wide); }
        else { CM_FEW(1, 2 * P, kFewSteps, false, wide); }
    } else {
        if (x == nullptr) { CM_FEW(1, P, kFewSteps, false, narrow); }
        else if (per == 1) { CM_FEW(1, P, 1, true, narrow); }
        else if (per == 2) { CM_FEW(1, P, 2, true, narrow); }
        else if (per == 3) { CM_FEW(1, P, 3, true, narrow); }
        else { CM_FEW(1, P, 4, true, narrow); }
    }
#undef CM_FEW
    return CM_OK;
}

// Tile columns of a strip of an XCD's run (tile_of).
uint32_t strip_of(uint64_t tiles, uint32_t tc) {
    const uint64_t run = (tiles + 7) / 8;
    uint32_t xw = 1;
    while ((uint64_t)xw * xw < run && xw < tc) xw++;
    return xw;
}

template <uint32_t MODE, int CB>
int mid_at(const Prod& p, hipStream_t s) {
    const uint32_t tr = p.rblocks, tc = ceil_div(p.cblocks, CB);
    CM_LAUNCH("linear8_mid_kernel", (linear8_mid_kernel<MODE, CB>), dim3(tr * tc), dim3(64 * std::min(kMidWaves, p.steps)), 0,
              s, p, tr, tc, strip_of((uint64_t)tr * tc, tc));
    return CM_OK;
}

// Rows of a few tiles from x in one launch: up to 1536 columns (the pieces of 3 steps in registers); each workgroup quantises
// its rows again.  Tiles of 32 columns up to one a compute unit, of 64 up to two (one of 3 steps); a gate's, of 32 + 32, up to 5 / 2
// steps of a wavefront a compute unit; else 0: codes first.  One launch of tiles of 32 / of 64 / two launches (us, 0.5 to 1 more for
// the second launch on the host): 64 x 256 x 1024 3.7 / 4.3 / 5.9, 512 x 256 x 1024 4.6 / 4.5 / 6.8, 2048 x 256 x 1024 8.8 / 7.7 / 7.4,
// 200 x 960 x 960 5.6 / 6.1 / 6.6, 333 x 960 x 960 7.6 / 6.2 / 7.4, 512 x 960 x 1600 12.5 / 9.0 / 8.9, 1024 x 960 x 960 12.1 / 8.7 / 9.1,
// 333 x 1000 x 4000 15.8 / 12.5 / 9.5, 128 x 1500 x 1600 6.6 / 7.3 / 7.6, 256 x 1500 x 1600 9.9 / 7.5 / 9.0, 512 x 1500 x 1600 17.3 /
// 11.4 / 10.7; a fourth step 128 x 2048 x 512 8.0 / 8.9 / 7.5; gates of 576 x 1536, 128 rows 5.8 / 7.4, 200 8.3 / 8.2, 512 11.9 / 8.6,
// of 256 x 1024, 512 rows 5.7 / 7.5, of 1500 x 1600, 128 rows 7.4 / 8.8, 256 11.2 / 10.5.
template <uint32_t MODE>
uint32_t mid_direct(const DeviceState* st, const Prod& p) {
    const uint32_t per = ceil_div(p.steps, kDirectWaves);
    if (per > kDirectSteps) return 0;
    auto tiles = [&](uint32_t columns) { return (uint64_t)p.rblocks * ceil_div(p.cblocks, columns); };
    const uint64_t cus = (uint64_t)st->cus;
    if (gated(MODE)) return 2 * per * tiles(2) <= 5 * cus ? 2 : 0;
    return tiles(1) <= cus ? 1 : tiles(2) <= (per < 3 ? 2 : 1) * cus ? 2 : 0;
}

template <uint32_t MODE, int CB>
int mid_direct_at(const Prod& p, const int16_t* x, uint64_t ld, uint32_t k, hipStream_t s) {
    const uint32_t tc = ceil_div(p.cblocks, CB), tiles = p.rblocks * tc, xw = strip_of(tiles, tc);
    const dim3 block(64 * std::min(kDirectWaves, p.steps));
    const bool odd = odd_rows(x, ld);
#define CM_MID(S, O) \
    CM_LAUNCH("linear8_mid_kernel", (linear8_mid_direct_kernel<MODE, CB, S, O>), dim3(tiles), block, 0, s, p, x, ld, k, p.rblocks, tc, xw)
    if (p.steps <= kDirectWaves) {
        if (odd) { CM_MID(1, true); } else { CM_MID(1, false); }
    } else if (p.steps <= 2 * kDirectWaves) {
        if (odd) { CM_MID(2, true); } else { CM_MID(2, false); }
    } else {
        if (odd) { CM_MID(3, true); } else { CM_MID(3, false); }
    }
#undef CM_MID
    return CM_OK;
}

template <uint32_t MODE, int RB, int CB>
int ring_at(const Prod& p, hipStream_t s) {
    const uint32_t tr = ceil_div(p.rblocks, 4 * RB), tc = ceil_div(p.cblocks, CB);
    CM_LAUNCH("linear8_ring_kernel", (linear8_ring_kernel<MODE, RB, CB>), dim3(tr * tc), dim3(256), 0, s, p, tr, tc,
              strip_of((uint64_t)tr * tc, tc));
    return CM_OK;
}

// The tile with the least of four estimates in ns, fitted to 150 measured products of 33 to 8192 rows (0.9 % behind the best
// tile of each, gates 0.6 %).  Among them (rows x k x columns: us of 256 x 128, 128 x 128, 128 x 64 and 32 x 32 tiles): 128 x 2560 x 960
// 17.2 / 10.6 / 6.8 / 4.4; 512 x 960 x 2560 10.3 / 6.8 / 5.0 / 7.9; 1000 x 1024 x 1024 10.4 / 6.9 / 5.0 / 6.9; 1024 x 2560 x 960 17.5 /
// 10.9 / 7.5 / 9.9; 512 x 8192 x 1024 - / 25.9 / 19.2 / 12.5; 2048 x 8192 x 2048 46.8 / 36.5 / 39.9 / 105; 4096 x 960 x 2560 20.4 /
// 18.7 / 17.7 / 44.0; 2048 x 4096 x 4096 35.2 / 35.3 / 41.7 / 99.7.  Gates (the smallest tile 32 x (32 + 32)): 300 x 960 x 2560
// 12.9 / 8.2 / 5.9 / 8.5; 777 x 768 x 2049 12.6 / 8.5 / 8.0 / 15.1; 2048 x 960 x 2560 22.3 / 20.7 / 18.3 / 39.5.  A compute unit holds
// two workgroups of 256 x 128, two or three of 128 x 128.  Up to a tile of 128 x 64 a compute unit, its own loads bound it (12 KiB
// a step at 64 bytes a cycle): eight wavefronts with k between them measured the same, 512 x 8192 x 1024 19.5 us.
template <uint32_t MODE>
int many_rows(const DeviceState* st, const Prod& p, hipStream_t s) {
    constexpr bool G = gated(MODE);
    constexpr int C0 = G ? 2 : 1;                          // the smallest tile's blocks of columns
    auto tiles = [&](uint32_t r, uint32_t c) { return (uint64_t)ceil_div(p.rblocks, r) * ceil_div(p.cblocks, c); };
    if (tiles(1, C0) > 0x7FFFFFFFu) return fail(CM_EINVAL, "linear8: %u rows of %u columns", p.n, p.m);
    const uint64_t cus = (uint64_t)st->cus, steps = p.steps;
    // quarters of a round of tiles: at least so many; whole rounds behind the first where a compute unit has one or two tiles at a time
    auto rounds = [&](uint64_t t) { return 4 * t <= 3 * cus ? 3 : (t + cus - 1) / cus * 4; };
    const uint64_t big = (G ? 6000 : 4000) + rounds(tiles(8, 4)) * (G ? 4800 + 310 * steps : 2800 + 430 * steps) / 4;
    const uint64_t square = (G ? 2800 : 2400) + rounds(tiles(4, 4)) * (G ? 3000 + 200 * steps : 1400 + 250 * steps) / 4;
    const uint64_t tall = 2400 + std::max(4 * tiles(4, 2), 3 * cus) * (G ? 1300 + 160 * steps : 700 + 150 * steps) / (4 * cus);
    const uint64_t small = 2500 + std::max(tiles(1, C0), cus) * (G ? 1500 + 60 * steps : 700 + 30 * steps) / cus;
    const uint64_t best = std::min(std::min(big, square), std::min(tall, small));
    if (best == small) return mid_at<MODE, C0>(p, s);
    if (best == tall) return ring_at<MODE, 1, 2>(p, s);
    return best == square ? ring_at<MODE, 1, 4>(p, s) : ring_at<MODE, 2, 4>(p, s);
}

// The product behind its checks: the rows' codes (the caller's, or made in the workspace), then the kernel.
template <uint32_t MODE>
int product(const cm_linear8_weight* w, const int16_t* x, uint64_t x_ld, const void* rows, Prod p, hipStream_t s) {
    DeviceState* st;
    int rc = state(&st);
    if (rc) return rc;
    p.m = w->m;
    p.steps = steps_of(w->k);
    p.rblocks = blocks_of(p.n);
    p.cblocks = blocks_of(w->m) * (gated(MODE) ? 2 : 1);
    const bool few = p.n <= 32;
    const uint32_t columns = rows == nullptr && !few ? mid_direct<MODE>(st, p) : 0;
    const bool direct = few ? rows == nullptr && few_direct(st, p) : columns != 0;
    if (rows == nullptr && !direct) {
        void* ws;
        if ((rc = workspace(st, rows_bytes(p.n, w->k), &ws, s))) return rc;
        if ((rc = quantise(st, x, x_ld, ws, p.n, w->k, s))) return rc;
        rows = ws;
    }
    if (!direct) {
        p.a = static_cast<const int8_t*>(rows);
        p.amax = reinterpret_cast<const int32_t*>(p.a + codes_bytes(p.rblocks, w->k));
    }
    p.w = static_cast<const int8_t*>(w->image);
    p.cols = reinterpret_cast<const double2*>(p.w + codes_bytes(p.cblocks, w->k));
    if (gated(MODE)) {
        p.gscale = __builtin_ldexp(1.0, (int)w->gate_shift);
        p.gneg = __builtin_ldexp(1.0, (int)w->gate_shift + 24);
        p.scale = __builtin_ldexp(1.0, -(int)w->out_shift - (w->act == kSilu ? 18 : 0));
        p.tab = w->act == kSilu ? st->sigmoid : st->act_tab + w->act * kActTabBytes;
        p.len = w->act == kSilu ? 0 : st->act_len[w->act];
    }
    if (few) {
        const int16_t* src = direct ? x : nullptr;
        return few_rows<MODE>(st, p, src, x_ld, w->k, s);
    }
    if constexpr (!gated(MODE))
        if (columns == 1) return mid_direct_at<MODE, 1>(p, x, x_ld, w->k, s);
    if (columns == 2) return mid_direct_at<MODE, 2>(p, x, x_ld, w->k, s);
    return many_rows<MODE>(st, p, s);
}

// n rows of some bytes, `pitch` bytes apart.
struct Extent {
    uintptr_t at;
    uint64_t pitch, bytes;
};

// Have two operands a byte in common?  Exact for equal pitches (columns of one buffer); others that reach into each other count as
// sharing one.
bool share(const Extent& a, const Extent& b, uint32_t n) {
    typedef unsigned __int128 Wide;
    const Wide ae = (Wide)a.at + (Wide)(n - 1) * a.pitch + a.bytes, be = (Wide)b.at + (Wide)(n - 1) * b.pitch + b.bytes;
    if (ae <= b.at || be <= a.at) return false;
    if (n == 1 || a.pitch != b.pitch) return true;
    const uint64_t d = a.at <= b.at ? (b.at - a.at) % a.pitch : a.pitch - 1 - (a.at - b.at - 1) % a.pitch;       // b's column behind a's
    return d < a.bytes || d + b.bytes > a.pitch;
}

Extent extent(const void* t, uint64_t ld, uint64_t columns, uint32_t bytes) {
    return Extent{reinterpret_cast<uintptr_t>(t), ld * bytes, columns * bytes};
}

// The output against x and the residual (another workgroup may still read what one has written), but for the residual's own rows.
int check_apart(const char* what, const cm_linear8_weight* w, const int16_t* x, uint64_t x_ld, uint32_t n, const Extent& out,
                const Extent* res) {
    if (x != nullptr && share(extent(x, x_ld, w->k, 2), out, n)) return fail(CM_EINVAL, "%s: the output overlaps x", what);
    if (res == nullptr || (res->at == out.at && (n == 1 || res->pitch == out.pitch))) return CM_OK;
    if (share(*res, out, n)) return fail(CM_EINVAL, "%s: the output overlaps the residual at another place or stride", what);
    return CM_OK;
}

int check_out(const char* what, const void* out, uint64_t ld, uint32_t n, uint32_t m, uint32_t bytes) {
    if (out == nullptr) return fail(CM_EINVAL, "%s: a null output", what);
    if (reinterpret_cast<uintptr_t>(out) & (bytes - 1)) return fail(CM_EALIGN, "%s: an operand is not aligned to its elements", what);
    if (n > 1 && ld < m) return fail(CM_EINVAL, "%s: rows of %u columns overlap at a stride of %llu", what, m, (unsigned long long)ld);
    if (n > 1 && ld >= 1u << 23) return fail(CM_EINVAL, "%s: a row stride of %llu (below 2^23)", what, (unsigned long long)ld);
    return CM_OK;
}

}  // namespace
}  // namespace cm

extern "C" size_t cm_linear8_image_bytes(uint32_t k, uint32_t m, uint32_t gated) { return cm::image_bytes(k, m, gated != 0); }

extern "C" size_t cm_linear8_rows_bytes(uint32_t n, uint32_t k) { return cm::rows_bytes(n, k); }

extern "C" int cm_linear8_pack(const int8_t* w, uint64_t k_stride, uint64_t m_stride, const double* mult, const int32_t* bias,
                               void* image, uint32_t k, uint32_t m, uint32_t part, void* stream) {
    using namespace cm;
    if (w == nullptr || mult == nullptr || image == nullptr) return fail(CM_EINVAL, "linear8 pack: a null operand");
    if (k == 0 || k > kMaxK || m == 0 || m > kMaxM)
        return fail(CM_EINVAL, "linear8 pack: a weight of %u x %u (up to %u x %u)", k, m, kMaxK, kMaxM);
    if (part > 2) return fail(CM_EINVAL, "linear8 pack: part %u (0: the weight, 1: gate, 2: up)", part);
    if ((reinterpret_cast<uintptr_t>(image) & 255u) || (reinterpret_cast<uintptr_t>(mult) & 7u) || (reinterpret_cast<uintptr_t>(bias) & 3u))
        return fail(CM_EALIGN, "linear8 pack: the image must be 256-byte aligned, the parameters to their elements");
    const uint32_t b = blocks_of(m), steps = steps_of(k);
    int8_t* codes = static_cast<int8_t*>(image);
    double2* cols = reinterpret_cast<double2*>(codes + codes_bytes(part ? 2 * b : b, k));
    const uint64_t pieces = (uint64_t)b * steps * 128;
    CM_LAUNCH("linear8_pack_kernel", linear8_pack_kernel, dim3(ceil_div(pieces, 256)), dim3(256), 0, as_stream(stream), w,
              k_stride, m_stride, mult, bias, codes, cols, k, m, steps, b, part);
    return CM_OK;
}

extern "C" int cm_linear8_rows(const int16_t* x, uint64_t x_ld, void* rows, uint32_t n, uint32_t k, void* stream) {
    using namespace cm;
    if (k == 0 || k > kMaxK) return fail(CM_EINVAL, "linear8 rows: rows of %u (up to %u)", k, kMaxK);
    int rc = check_rows("linear8 rows", x, x_ld, nullptr, n, k);
    if (rc || n == 0) return rc;
    if (rows == nullptr) return fail(CM_EINVAL, "linear8 rows: a null output");
    if (reinterpret_cast<uintptr_t>(rows) & 255u) return fail(CM_EALIGN, "linear8 rows: the codes must be 256-byte aligned");
    DeviceState* st;
    if ((rc = state(&st))) return rc;
    return quantise(st, x, x_ld, rows, n, k, as_stream(stream));
}

extern "C" int cm_linear8(const cm_linear8_weight* weight, const int16_t* x, uint64_t x_ld, const void* rows, uint32_t n,
                          void* out, uint64_t out_ld, const int32_t* residual, uint64_t residual_ld, uint32_t shift,
                          void* stream) {
    using namespace cm;
    int rc = check_weight("linear8", weight, false);
    if (rc || (rc = check_rows("linear8", x, x_ld, rows, n, weight->k)) || n == 0) return rc;
    const uint32_t bytes = residual ? 4 : 2;
    const Extent to = extent(out, out_ld, weight->m, bytes), from = extent(residual, residual_ld, weight->m, 4);
    if ((rc = check_out("linear8", out, out_ld, n, weight->m, bytes))) return rc;
    if (residual != nullptr && (rc = check_out("linear8", residual, residual_ld, n, weight->m, 4))) return rc;
    if ((rc = check_apart("linear8", weight, x, x_ld, n, to, residual ? &from : nullptr))) return rc;
    if (shift > 16) return fail(CM_EINVAL, "linear8: a residual shift of %u (up to 16)", shift);
    Prod p{};
    p.n = n;
    p.out = out;
    p.out_ld = out_ld;
    if (residual == nullptr) return product<kOut16>(weight, x, x_ld, rows, p, as_stream(stream));
    p.res = residual;
    p.res_ld = residual_ld;
    p.shift = shift;
    return product<kOut32>(weight, x, x_ld, rows, p, as_stream(stream));
}

extern "C" int cm_linear8_gated(const cm_linear8_weight* weight, const int16_t* x, uint64_t x_ld, const void* rows, uint32_t n,
                                int16_t* out, uint64_t out_ld, void* stream) {
    using namespace cm;
    int rc = check_weight("linear8 gated", weight, true);
    if (rc || (rc = check_rows("linear8 gated", x, x_ld, rows, n, weight->k)) || n == 0) return rc;
    if ((rc = check_out("linear8 gated", out, out_ld, n, weight->m, 2))) return rc;
    if ((rc = check_apart("linear8 gated", weight, x, x_ld, n, extent(out, out_ld, weight->m, 2), nullptr))) return rc;
    Prod p{};
    p.n = n;
    p.out = out;
    p.out_ld = out_ld;
    return weight->act == kSilu ? product<kSiluGate>(weight, x, x_ld, rows, p, as_stream(stream))
                                : product<kTableGate>(weight, x, x_ld, rows, p, as_stream(stream));
}
