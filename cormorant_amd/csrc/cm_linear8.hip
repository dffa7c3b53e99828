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
#include "cm_rowops_math.h"

namespace cm {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr uint32_t kLine = 32, kStep = 64, kPiece = kLine * kStep;      // lines and k of a block, its bytes
constexpr uint32_t kMaxK = 32768, kMaxM = 1u << 20, kMaxN = 1u << 22;
constexpr double kMagic = 6755399441055744.0;                           // 1.5 2^52: a whole number added to it is its low word

enum : uint32_t { kOut16 = 0, kOut32 = 1, kGated = 2 };
enum : uint32_t { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

inline uint32_t steps_of(uint32_t k) { return ceil_div(k, kStep); }
inline uint32_t blocks_of(uint32_t lines) { return ceil_div(lines, kLine); }

// Where a rows image's maxima and a weight image's channel parameters start (behind the blocks).
inline size_t codes_bytes(uint32_t blocks, uint32_t k) { return (size_t)blocks * steps_of(k) * kPiece; }
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
    const uint8_t* tab;              // kGated: the sigmoid's pieces, or the activation's bytes (`len` of them)
    uint32_t act, len, sa;
    double scale;                    // 2^-sc
};

// rne(acc a mu + b), saturated to int16.
__device__ __forceinline__ int32_t out16(int32_t acc, double a, double2 c) {
    const double z = __builtin_fma((double)acc * a, c.x, c.y);
    return __double2loint(__builtin_fmin(__builtin_fmax(z, kMagic - 32768.0), kMagic + 32767.0));
}

__device__ __forceinline__ int32_t add_res(int32_t h, int32_t o, uint32_t shift) {
    const int64_t s = (int64_t)h + ((int64_t)o << shift);
    return (int32_t)(s > 2147483647 ? 2147483647 : s < -2147483648ll ? -2147483648ll : s);
}

// act(g) u 2^-sc, rounded to even and saturated.  SiLU by the row-ops rule (MULACT): sigma at 2^-24 from the
// piece of |g| at 2^-14, silu at 2^-20.  gv sigma is exact in a double (below 2^18 2^26, or a power of two
// times g), so is silu u (2^35 2^15), and each sum onto 1.5 2^52 is its one rounding.
__device__ __forceinline__ int32_t gate16(int32_t g, int32_t u, const Prod& p) {
    double f;
    const uint32_t a = (uint32_t)(g < 0 ? -g : g);
    if (p.act == kSilu) {
        const uint32_t av = a << p.sa, ai = min(av, (1u << 18) - 1), fr = ai & 63;
        const uint64_t e = *reinterpret_cast<const uint64_t*>(p.tab + 8 * (ai >> 6));
        const uint32_t T = (uint32_t)e & 0x1FFFFFFu, D = (uint32_t)(e >> 25) & 0xFFFFFFu;
        int32_t sg = av >= (1u << 18) ? 1 << 24 : (int32_t)(T + ((D * fr) >> 6));
        if (g < 0) sg = (1 << 24) - sg;
        f = __builtin_fma((double)(g << p.sa), (double)sg * 0x1p-18, kMagic) - kMagic;
    } else {
        f = (double)(max(g, 0) - (a < p.len ? (int32_t)p.tab[a] : 0));
    }
    const double v = __builtin_fmin(__builtin_fmax(f * (double)u * p.scale, -65536.0), 65536.0);
    return min(max(__double2loint(v + kMagic), -32768), 32767);
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
    *reinterpret_cast<int4*>(codes + ((uint64_t)to * steps + st) * kPiece + kg * 512 + line * 16) = *reinterpret_cast<const int4*>(v);
    if (st == 0 && kg == 0)
        cols[(uint64_t)to * kLine + line] = j < m ? make_double2(mult[j], kMagic + (bias ? (double)bias[j] : 0.0)) : make_double2(0.0, kMagic);
}

// ---------------------------------------------------------------- a row's codes
__device__ __forceinline__ int4 load8(const int16_t* p) {                   // 8 elements at any alignment
    int4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

__device__ __forceinline__ uint32_t recip(uint32_t a) { return a ? (127u * (1u << 24) + (a >> 1)) / a : 0u; }
__device__ __forceinline__ int32_t code(int32_t x, uint32_t r) { return (x * (int32_t)r + (1 << 23)) >> 24; }

// A wavefront a row: its maximum, then its codes, 16 elements a lane.
__global__ __launch_bounds__(256) void linear8_rows_kernel(const int16_t* __restrict__ x, uint64_t ld, uint32_t n, uint32_t k,
                                                           int8_t* __restrict__ codes, int32_t* __restrict__ amax, uint32_t steps) {
    const uint32_t lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= n) return;
    const int16_t* r = x + (uint64_t)row * ld;
    const uint32_t kp = steps * kStep;
    auto load = [&](uint32_t k0, int16_t (&e)[16]) {
        if (k0 + 16 <= k) {
            const int4 v[2] = {load8(r + k0), load8(r + k0 + 8)};
            __builtin_memcpy(e, v, 32);
        } else {
            for (uint32_t q = 0; q < 16; q++) e[q] = k0 + q < k ? r[k0 + q] : (int16_t)0;
        }
    };
    int32_t top = 0;
    int16_t e[16];
    for (uint32_t k0 = 16 * lane; k0 < kp; k0 += 1024) {
        load(k0, e);
        for (int q = 0; q < 16; q++) top = max(top, abs((int32_t)e[q]));
    }
    for (int off = 32; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
    if (lane == 0) amax[row] = top;
    const uint32_t rc = recip((uint32_t)top);
    for (uint32_t k0 = 16 * lane; k0 < kp; k0 += 1024) {
        load(k0, e);
        int8_t c[16];
        for (int q = 0; q < 16; q++) c[q] = (int8_t)code(e[q], rc);
        const uint32_t st = k0 >> 6, kg = (k0 >> 4) & 3;
        *reinterpret_cast<int4*>(codes + ((uint64_t)(row >> 5) * steps + st) * kPiece + kg * 512 + (row & 31) * 16) =
            *reinterpret_cast<const int4*>(c);
    }
}

// ---------------------------------------------------------------- products
// The value of one output element from the sums of its columns (kGated: gate and up).
template <uint32_t MODE>
__device__ __forceinline__ void store(const Prod& p, uint32_t row, uint32_t col, int32_t acc0, int32_t acc1, double a,
                                      double2 c0, double2 c1) {
    if (row >= p.n || col >= p.m) return;
    const int32_t o = out16(acc0, a, c0);
    if (MODE == kOut16) {
        static_cast<int16_t*>(p.out)[row * p.out_ld + col] = (int16_t)o;
    } else if (MODE == kOut32) {
        static_cast<int32_t*>(p.out)[row * p.out_ld + col] = add_res(p.res[row * p.res_ld + col], o, p.shift);
    } else {
        static_cast<int16_t*>(p.out)[row * p.out_ld + col] = (int16_t)gate16(o, out16(acc1, a, c1), p);
    }
}

// 64 rows by two pairs of column blocks a workgroup, a wavefront 32 rows and a pair, operands straight from memory.
template <uint32_t MODE>
__global__ __launch_bounds__(256) void linear8_tile_kernel(Prod p) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, lh = lane >> 5;
    const uint32_t rb = blockIdx.y * 2 + (wave >> 1), pair = blockIdx.x * 2 + (wave & 1);
    if (rb >= p.rblocks || 2 * pair >= p.cblocks) return;
    const uint32_t cb[2] = {2 * pair, min(2 * pair + 1, p.cblocks - 1)};
    const int8_t* a = p.a + (uint64_t)rb * p.steps * kPiece + lane * 16;
    const int8_t* w0 = p.w + (uint64_t)cb[0] * p.steps * kPiece + lane * 16;
    const int8_t* w1 = p.w + (uint64_t)cb[1] * p.steps * kPiece + lane * 16;
    v16i s0{}, s1{};
    for (uint32_t i = 0; i < 2 * p.steps; i++) {
        const uint64_t at = (uint64_t)i * 1024;
        const v4i av = *reinterpret_cast<const v4i*>(a + at);
        s0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, *reinterpret_cast<const v4i*>(w0 + at), s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, *reinterpret_cast<const v4i*>(w1 + at), s1, 0, 0, 0);
    }
    const double2 c0 = p.cols[cb[0] * kLine + l32], c1 = p.cols[cb[1] * kLine + l32];
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const uint32_t row = rb * kLine + 8 * (r >> 2) + 4 * lh + (r & 3);
        const double am = (double)p.amax[min(row, p.n - 1)];
        if (MODE == kGated) {
            store<MODE>(p, row, pair * kLine + l32, s0[r], s1[r], am, c0, c1);
        } else {
            store<MODE>(p, row, cb[0] * kLine + l32, s0[r], 0, am, c0, c0);
            if (cb[1] != cb[0]) store<MODE>(p, row, cb[1] * kLine + l32, s1[r], 0, am, c1, c1);
        }
    }
}

// ---------------------------------------------------------------- few rows
// At most 16 RF rows: the weight is read once and the time is the latency of a launch, of x and of a
// weight's bytes.  A workgroup of W wavefronts takes NF fragments of 16 columns (kGated: half gate, half up) at
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

template <uint32_t MODE, uint32_t RF, uint32_t NF, uint32_t S, bool DIRECT>
__global__ __launch_bounds__(64 * kFewWaves) void linear8_few_kernel(Prod p, const int16_t* __restrict__ x, uint64_t ld, uint32_t k) {
    constexpr uint32_t R = 16 * RF, COLS = 16 * NF, OUT = MODE == kGated ? COLS / 2 : COLS;
    constexpr uint32_t LD = COLS + 4;                // the four k groups' rows in different banks
    __shared__ int32_t red[R * LD];                  // the unit's sums, zeros between units
    __shared__ int32_t part[R * kFewWaves], top[R];  // the rows' maxima: of a wavefront's pieces, and all
    const uint32_t W = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint32_t units = (p.m + OUT - 1) / OUT;
    const int8_t* w[NF];
    // fragment f of unit u: its column block and half (kGated: gate and up blocks alternate)
    auto weights_of = [&](uint32_t u) {
#pragma unroll
        for (uint32_t f = 0; f < NF; f++) {
            constexpr uint32_t per = MODE == kGated ? NF / 2 : NF;
            const uint32_t q = u * per + f % per;
            const uint32_t blk = MODE == kGated ? 2 * (q >> 1) + f / per : q >> 1;
            // columns past the last block: any, never stored
            w[f] = p.w + (uint64_t)min(blk, p.cblocks - 1) * p.steps * kPiece + g * 512 + (q & 1) * 256 + c * 16;
        }
    };
    uint32_t u = blockIdx.x;
    weights_of(u);
    v4i a[S][RF], b[S][NF];
    for (uint32_t e = threadIdx.x; e < R * LD; e += blockDim.x) red[e] = 0;
    if constexpr (DIRECT) {
        int4 xv[S][RF][2];
        const int16_t* xr[RF];
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) xr[f] = x + (uint64_t)min(16 * f + c, p.n - 1) * ld;
#pragma unroll
        for (uint32_t i = 0; i < S; i++) {
            const uint32_t k0 = (wave + i * W) * kStep + 16 * g;
#pragma unroll
            for (uint32_t f = 0; f < RF; f++) {
                if (k0 + 16 <= k) {
                    xv[i][f][0] = load8(xr[f] + k0);
                    xv[i][f][1] = load8(xr[f] + k0 + 8);
                } else {
                    int16_t e[16];
#pragma unroll
                    for (uint32_t q = 0; q < 16; q++) e[q] = k0 + q < k ? xr[f][k0 + q] : (int16_t)0;
                    __builtin_memcpy(&xv[i][f][0], e, 32);
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < S; i++)
            if (wave + i * W < p.steps) load_weights<NF>(b[i], w, wave + i * W);
        // the rows' maxima: this wavefront's pieces, its four k groups, then the wavefronts
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) {
            int32_t t = 0;
#pragma unroll
            for (uint32_t i = 0; i < S; i++) {
                const int16_t* e = reinterpret_cast<const int16_t*>(&xv[i][f][0]);
#pragma unroll
                for (int q = 0; q < 16; q++) t = max(t, abs((int32_t)e[q]));
            }
            t = max(t, __shfl_xor(t, 16, 64));
            t = max(t, __shfl_xor(t, 32, 64));
            if (g == 0) part[(16 * f + c) * kFewWaves + wave] = t;
        }
        lds_barrier();
#pragma unroll
        for (uint32_t f = 0; f < RF; f++) {
            int32_t am = 0;
            for (uint32_t i = 0; i < W; i++) am = max(am, part[(16 * f + c) * kFewWaves + i]);
            if (wave == 0 && g == 0) top[16 * f + c] = am;
            const int32_t rc = (int32_t)recip((uint32_t)am);
#pragma unroll
            for (uint32_t i = 0; i < S; i++) {
                const int16_t* e = reinterpret_cast<const int16_t*>(&xv[i][f][0]);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t word = 0;               // four codes: the top bytes of four sums
#pragma unroll
                    for (int h = 0; h < 4; h++) word |= ((uint32_t)(e[4 * q + h] * rc + (1 << 23)) >> 24) << (8 * h);
                    a[i][f][q] = (int)word;
                }
            }
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
        for (uint32_t e = threadIdx.x; e < R * OUT; e += blockDim.x) {
            const uint32_t row = e / OUT, cl = e % OUT, col = u * OUT + cl;
            const int32_t s0 = red[row * LD + cl], s1 = MODE == kGated ? red[row * LD + OUT + cl] : 0;
            red[row * LD + cl] = 0;
            if (MODE == kGated) red[row * LD + OUT + cl] = 0;
            if (row >= p.n || col >= p.m) continue;
            const double am = (double)(DIRECT ? top[row] : p.amax[row]);
            const uint32_t at = MODE == kGated ? (col >> 5) * 64 + (col & 31) : col;
            store<MODE>(p, row, col, s0, s1, am, p.cols[at], MODE == kGated ? p.cols[at + 32] : double2{});
        }
        if (next >= units) return;
        u = next;
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

int quantise(const int16_t* x, uint64_t x_ld, void* rows, uint32_t n, uint32_t k, hipStream_t s) {
    int8_t* codes = static_cast<int8_t*>(rows);
    int32_t* amax = reinterpret_cast<int32_t*>(codes + codes_bytes(blocks_of(n), k));
    CM_LAUNCH("linear8_rows_kernel", linear8_rows_kernel, dim3(ceil_div(n, 4)), dim3(256), 0, s, x, x_ld, n, k, codes, amax,
              steps_of(k));
    return CM_OK;
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

// Few rows: fragments of columns a workgroup, and the grid.
template <uint32_t MODE, uint32_t RF, uint32_t NF>
int few_rows_at(const Prod& p, const int16_t* x, uint64_t ld, uint32_t k, uint32_t grid, hipStream_t s) {
    const uint32_t W = std::min(kFewWaves, p.steps), per = (p.steps + W - 1) / W;
#define CM_FEW(S, D) \
    CM_LAUNCH("linear8_few_kernel", (linear8_few_kernel<MODE, RF, NF, S, D>), dim3(grid), dim3(64 * W), 0, s, p, x, ld, k)
    if (x == nullptr) { CM_FEW(kFewSteps, false); }
    else if (per == 1) { CM_FEW(1, true); }
    else if (per == 2) { CM_FEW(2, true); }
    else { CM_FEW(kFewSteps, true); }
#undef CM_FEW
    return CM_OK;
}

template <uint32_t MODE>
int few_rows(const DeviceState* st, const Prod& p, const int16_t* x, uint64_t ld, uint32_t k, hipStream_t s) {
    constexpr uint32_t P = MODE == kGated ? 2 : 1;
    const uint32_t cap = 2 * (uint32_t)st->cus;
    if (p.n > 16) return few_rows_at<MODE, 2, P>(p, x, ld, k, std::min(ceil_div(p.m, 16), cap), s);
    if (p.m <= 16 * cap) return few_rows_at<MODE, 1, P>(p, x, ld, k, ceil_div(p.m, 16), s);
    return few_rows_at<MODE, 1, 2 * P>(p, x, ld, k, std::min(ceil_div(p.m, 32), cap), s);
}

// The product behind its checks: the rows' codes (the caller's, or made in the workspace), then the kernel.
template <uint32_t MODE>
int product(const cm_linear8_weight* w, const int16_t* x, uint64_t x_ld, const void* rows, Prod p, hipStream_t s) {
    DeviceState* st;
    int rc = state(&st);
    if (rc) return rc;
    const bool few = p.n <= 32, direct = few && rows == nullptr && steps_of(w->k) <= kFewSteps * kFewWaves;
    if (rows == nullptr && !direct) {
        void* ws;
        if ((rc = workspace(st, rows_bytes(p.n, w->k), &ws, s))) return rc;
        if ((rc = quantise(x, x_ld, ws, p.n, w->k, s))) return rc;
        rows = ws;
    }
    p.m = w->m;
    p.steps = steps_of(w->k);
    p.rblocks = blocks_of(p.n);
    p.cblocks = blocks_of(w->m) * (MODE == kGated ? 2 : 1);
    if (!direct) {
        p.a = static_cast<const int8_t*>(rows);
        p.amax = reinterpret_cast<const int32_t*>(p.a + codes_bytes(p.rblocks, w->k));
    }
    p.w = static_cast<const int8_t*>(w->image);
    p.cols = reinterpret_cast<const double2*>(p.w + codes_bytes(p.cblocks, w->k));
    if (MODE == kGated) {
        p.act = w->act;
        p.sa = w->gate_shift;
        p.scale = __builtin_ldexp(1.0, -(int)w->out_shift);
        p.tab = w->act == kSilu ? st->ro_tables : st->act_tab + w->act * kActTabBytes;
        p.len = w->act == kSilu ? 0 : st->act_len[w->act];
    }
    if (few) {
        const int16_t* src = direct ? x : nullptr;
        return few_rows<MODE>(st, p, src, x_ld, w->k, s);
    }
    const dim3 grid(ceil_div(p.cblocks, 4), ceil_div(p.rblocks, 2));
    if (grid.y > 65535u) return fail(CM_EINVAL, "linear8: %u rows", p.n);
    CM_LAUNCH("linear8_tile_kernel", linear8_tile_kernel<MODE>, grid, dim3(256), 0, s, p);
    return CM_OK;
}

int check_out(const char* what, const void* out, uint64_t ld, uint32_t n, uint32_t m, uint32_t bytes) {
    if (out == nullptr) return fail(CM_EINVAL, "%s: a null output", what);
    if (reinterpret_cast<uintptr_t>(out) & (bytes - 1)) return fail(CM_EALIGN, "%s: an operand is not aligned to its elements", what);
    if (n > 1 && ld < m) return fail(CM_EINVAL, "%s: rows of %u columns overlap at a stride of %llu", what, m, (unsigned long long)ld);
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
    return quantise(x, x_ld, rows, n, k, as_stream(stream));
}

extern "C" int cm_linear8(const cm_linear8_weight* weight, const int16_t* x, uint64_t x_ld, const void* rows, uint32_t n,
                          void* out, uint64_t out_ld, const int32_t* residual, uint64_t residual_ld, uint32_t shift,
                          void* stream) {
    using namespace cm;
    int rc = check_weight("linear8", weight, false);
    if (rc || (rc = check_rows("linear8", x, x_ld, rows, n, weight->k)) || n == 0) return rc;
    if ((rc = check_out("linear8", out, out_ld, n, weight->m, residual ? 4 : 2))) return rc;
    if (shift > 16) return fail(CM_EINVAL, "linear8: a residual shift of %u (up to 16)", shift);
    Prod p{};
    p.n = n;
    p.out = out;
    p.out_ld = out_ld;
    if (residual == nullptr) return product<kOut16>(weight, x, x_ld, rows, p, as_stream(stream));
    if ((rc = check_out("linear8", residual, residual_ld, n, weight->m, 4))) return rc;
    if (residual == out && residual_ld != out_ld && n > 1) return fail(CM_EINVAL, "linear8: the output is the residual at another stride");
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
    Prod p{};
    p.n = n;
    p.out = out;
    p.out_ld = out_ld;
    return product<kGated>(weight, x, x_ld, rows, p, as_stream(stream));
}
