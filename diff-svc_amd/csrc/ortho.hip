// Orthogonalising an update by Newton-Schulz products, and the optimisation step built on it (include/dsvc.h: dsvc_orthogonalize,
// dsvc_muon_step).
//
//   X = G / (||G||_F + eps)      (G transposed if it has more rows than columns, so X is [m x n] with m <= n)
//   steps times:  A = X X^T,  M = a I + b A + c A A,  X <- M X            (the singular values go through s (a + b s^2 + c s^4))
//   O = scale * X                (transposed back)
//
// Arithmetic: every product is an fp16 MFMA (v_mfma_f32_32x32x16_f16) with fp32 accumulation, on hi + lo planes and three MFMAs per product (hi hi + hi lo +
// lo hi: 22 bits per operand, fp32-class, the trainer's own scheme), whatever the tensor's type: a rounding of an early iterate grows by up to a^steps
// (485 for the usual five) in the directions in which the update has next to nothing.  [512, 768] of rank 1: 1.1e-4 of the result's norm from exact (fp32
// products 6e-5), of full rank 2.5e-6.  ONE plane is the caller's own choice (cfg.planes = 1): a third of the MFMAs, 11 bits, and so 1.9e-3 at full
// rank but 4e-2 at rank 16 and 1e-1 at rank 1, where a bf16 result's own rounding is 1.7e-3.
// The planes hold X * 2^12 and A, M * 2^10: |X| and |M| are bounded by the polynomial on [0, 1] (checked on the host for the caller's
// coefficients), so fp16's top is out of reach and small elements keep their bits; an update whose norm eps swamps is carried with an
// extra power of two that shrinks as the iterate grows (Scalars::e0).  Norms are summed in fp64: no square of a tiny gradient underflows.
//
// Layout: every matrix between the products lies in MFMA FRAGMENT ORDER -- [32-row block][16-wide k step][plane][lane][8]: lane l of a
// 1 KiB piece holds row l & 31, k = 8 (l >> 5) .. + 7.  A stage of a tile is then a few contiguous KiB that global_load_lds copies into LDS as
// they lie and ds_read_b128 reads without bank conflicts; the accumulator layout (lane = column, registers = 4 consecutive rows) writes
// the TRANSPOSED result as whole 512-byte runs, and the untransposed one after the tile went through the matrix core once more against an
// identity fragment (exact: one fp16 value times one).  Rows and columns are padded with zeros to 128, which every product keeps zero.
//
// A and M are symmetric: only the tiles on and above the diagonal are computed, the mirrored tile is written by the same workgroup.
#include <math.h>

#include <utility>

#include "../../include/dsvc.h"
#include "common.h"

using namespace dsvc;

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef const half8 __attribute__((address_space(3))) * lds_half8;

constexpr float X_SCALE = 4096.f, A_SCALE = 1024.f;
constexpr int PAD = 128;                     // rows and columns of every intermediate are padded to this
// Padded elements up to which one workgroup takes a matrix of up to 64 rows.  fp32, one workgroup against 17 launches (GPU time; the host takes 60 us to
// launch them): [1, 1] 24 / 71 us, [64, 64] x 8 27 / 76, [64, 256] 52 / 80, [32, 500] 72 / 88, [64, 1024] 163 / 103; [48, 64] x 2000 197 / 1162
constexpr long long ONE_WORK = 16384;
constexpr int ONE_LDS = 156 * 1024;          // its LDS (the rest: static)
constexpr int SUM_BLOCKS = 256;              // partial sums of squares per matrix

enum { F32 = DSVC_DTYPE_F32, F16 = DSVC_DTYPE_F16, BF16 = DSVC_DTYPE_BF16 };

template <int T> struct Elem;
template <> struct Elem<F32> { typedef float type; };
template <> struct Elem<F16> { typedef _Float16 type; };
template <> struct Elem<BF16> { typedef __bf16 type; };

struct View { long long ld, bs; };           // elements between rows / between matrices

// per matrix, written by the normalising kernel's block 0 and read by the products
struct Scalars { int e0; };

struct MuonArgs {                            // momentum: null for the plain operator
    float* mom; View mv;
    float mu, lr, wd;
    int nesterov;
    const float* gscale_dev;
    float gscale;
};

// u = the tensor that is orthogonalised, from the gradient and the UPDATED momentum
__device__ __forceinline__ float muon_mom(const MuonArgs& u, float g, float m) { return fmaf(u.mu, m, (1.f - u.mu) * g); }
__device__ __forceinline__ float muon_u(const MuonArgs& u, float g, float m) { return u.nesterov ? fmaf(u.mu, m, (1.f - u.mu) * g) : m; }

// ---- sums of squares (fp64), and the momentum update on the way: grid (blocks, matrices).  Partials are combined in a fixed order. ----
// Bound by memory: [20, 768, 1152] fp32 15 - 17 us (71 MB, 4.2 - 4.8 TB/s), [2048, 8192] bf16 with the fp32 momentum read and written 27 us (168 MB, 6.2 TB/s:
// part of it from the last-level cache).
// flat: rows follow one another without gaps in every tensor (one row of rows * cols elements); vec: every row start and the row length allow
// 16-byte accesses of VEC elements
template <int T, bool MUON, int VEC>
__global__ __launch_bounds__(256) void k_ns_sums(const void* __restrict__ in, View iv, int rows, long long cols, MuonArgs mu, double* __restrict__ part,
                                                 int* __restrict__ count, int n_count) {
    typedef typename Elem<T>::type E;
    typedef E EV __attribute__((ext_vector_type(VEC)));
    typedef float FV __attribute__((ext_vector_type(VEC)));
    const int b = blockIdx.y;
    const E* src = (const E*)in + b * iv.bs;
    float* mom = MUON ? mu.mom + b * mu.mv.bs : nullptr;
    const float gs = MUON ? (mu.gscale_dev ? *mu.gscale_dev : mu.gscale) : 1.f;
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < n_count; i += gridDim.x * gridDim.y * 256) count[i] = 0;
    const long long per_row = cols / VEC, n = rows * per_row, step = (long long)gridDim.x * 256;
    double s = 0.0;
    for (long long i0 = (long long)blockIdx.x * 256 + threadIdx.x; i0 < n; i0 += 4 * step) {
        EV v[4];
        FV m[4];
        long long at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long i = i0 + k * step;
            if (i >= n) continue;
            const long long r = rows == 1 ? 0 : (unsigned long long)i < (1ull << 32) && per_row < (1ll << 32) ? (unsigned)i / (unsigned)per_row : i / per_row;
            const long long c = (i - r * per_row) * VEC;
            v[k] = *(const EV*)(src + r * iv.ld + c);
            if (MUON) {
                at[k] = r * mu.mv.ld + c;
                m[k] = *(const FV*)(mom + at[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i0 + k * step >= n) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float x = (float)v[k][e];
                if (MUON) {
                    x *= gs;
                    m[k][e] = muon_mom(mu, x, m[k][e]);
                    x = muon_u(mu, x, m[k][e]);
                }
                s = fma((double)x, (double)x, s);
            }
            if (MUON) *(FV*)(mom + at[k]) = m[k];
        }
    }
    __shared__ double red[256];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[(long long)b * gridDim.x + blockIdx.x] = red[0];
}

// ---- normalise and lay out: one workgroup = a 64 x 64 tile of X, written in fragment order as X (k = columns) and X^T (k = rows) ----
// Bound by memory: an fp32 element is read once and written as four fp16 (hi + lo of both orders), 12 bytes: [20, 768, 1152] 42 us (212 MB, 5.1 TB/s).
template <int T, bool MUON, int P>
__global__ __launch_bounds__(256) void k_ns_prep(const void* __restrict__ in, View iv, int rows, int cols, int tall, MuonArgs mu, const double* __restrict__ part,
                                                 int n_part, double eps, _Float16* __restrict__ x, _Float16* __restrict__ xt, int mp, int np, Scalars* __restrict__ sc) {
    typedef typename Elem<T>::type E;
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64, tid = threadIdx.x;
    __shared__ double red[SUM_BLOCKS];
    __shared__ float tile[64][65];
    red[tid] = tid < n_part ? part[(long long)b * n_part + tid] : 0.0;
    __syncthreads();
    for (int k = SUM_BLOCKS / 2; k > 0; k >>= 1) {
        if (tid < k) red[tid] += red[tid + k];
        __syncthreads();
    }
    const double norm = sqrt(red[0]), t = norm / (norm + eps);
    // t < 1/2 only where eps matters: planes carry 2^e0 more
    int e0 = 0;
    if (t < 0.5) e0 = t > 1e-18 ? -ilogb(t) - 1 : 59;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) sc[b].e0 = e0;
    const double f = ldexp((double)X_SCALE, e0) / (norm + eps);
    const E* src = (const E*)in + b * iv.bs;
    const float* mom = MUON ? mu.mom + b * mu.mv.bs : nullptr;
    const float gs = MUON ? (mu.gscale_dev ? *mu.gscale_dev : mu.gscale) : 1.f;
    const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
    for (int k = tid; k < 4096; k += 256) {
        const int r = k >> 6, c = k & 63;
        float v = 0.f;
        if (r0 + r < rows && c0 + c < cols) {
            v = (float)src[(long long)(r0 + r) * iv.ld + c0 + c];
            if (MUON) v = muon_u(mu, v * gs, mom[(long long)(r0 + r) * mu.mv.ld + c0 + c]);
            v = (float)((double)v * f);
        }
        if (tall) tile[c][r] = v; else tile[r][c] = v;          // tile[i][j]
    }
    __syncthreads();
    const int wave = tid >> 6, lane = tid & 63;
    const int nk_x = np >> 4, nk_t = mp >> 4;
    _Float16* xb = x + (long long)b * mp * np * P;
    _Float16* tb = xt + (long long)b * mp * np * P;
    for (int q = wave; q < 16; q += 4) {                        // 8 pieces of X, 8 of X^T
        const int blk = (q >> 2) & 1, k16 = q & 3, row = 32 * blk + (lane & 31), k = 16 * k16 + 8 * (lane >> 5);
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = one_value(q < 8 ? tile[row][k + e] : tile[k + e][row]);
            hi[e] = (_Float16)v;
            lo[e] = (_Float16)(v - (float)hi[e]);
        }
        _Float16* d = q < 8 ? xb + (((long long)((i0 >> 5) + blk) * nk_x + (j0 >> 4) + k16) * P) * 512
                            : tb + (((long long)((j0 >> 5) + blk) * nk_t + (i0 >> 4) + k16) * P) * 512;
        *(half8*)(d + lane * 8) = hi;
        if (P == 2) *(half8*)(d + 512 + lane * 8) = lo;
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------------------------
enum { GRAM, POLY, FULL, FINAL };

// the caller's tensor: the result, or (mu.mom) the parameter, out <- (1 - lr wd) out - lr result.  wide: neighbouring elements of a row may be accessed
// as one (4 of a transposed result's, 2 of 16 bits of the other's)
struct Output {
    void* out; View ov;
    int dtype, m, n, tall, wide;
    MuonArgs mu;
};
// 32 x 32 block (bi, bj) of matrix b, scaled by c: register r of a lane = row 8 (r >> 2) + 4 (lane >> 5) + (r & 3), column lane & 31.  Transposed, a lane has
// four neighbours in memory; else neighbours are in neighbouring lanes, and pairs of 16-bit elements are put together by one exchange (element by
// element a [768, 384] x 20 step's last product took 53 us, where the others take 25)
template <class E>
__device__ __forceinline__ void store_block(const Output& o, int b, int bi, int bj, int lane, const f32x16& acc, float c) {
    typedef E E2 __attribute__((ext_vector_type(2)));
    typedef E E4 __attribute__((ext_vector_type(4)));
    E* out = (E*)o.out + b * o.ov.bs;
    const int col = 32 * bj + (lane & 31), row0 = 32 * bi + 4 * (lane >> 5);
    const bool step = o.mu.mom != nullptr;
    const float keep = 1.f - o.mu.lr * o.mu.wd, lr = -o.mu.lr;
    auto put = [&](E* p, float v) { *p = (E)(step ? fmaf(lr, v, keep * (float)*p) : v); };
    if (o.tall) {
        if (col >= o.n) return;
        E* line = out + col * o.ov.ld;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = row0 + 8 * q;
            if (o.wide && row + 3 < o.m) {
                E4 v;
                if (step) v = *(const E4*)(line + row);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (E)(step ? fmaf(lr, acc[4 * q + e] * c, keep * (float)v[e]) : acc[4 * q + e] * c);
                *(E4*)(line + row) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row + e < o.m) put(line + row + e, acc[4 * q + e] * c);
            }
        }
        return;
    }
    if (sizeof(E) == 2 && o.wide) {
        const bool odd = lane & 1;
        const int c0 = col & ~1;             // the pair's columns: even lanes take a row's, odd lanes the next row's
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float mine = (odd ? acc[r + 1] : acc[r]) * c, other = __shfl_xor((odd ? acc[r] : acc[r + 1]) * c, 1);
            const int row = row0 + 8 * (r >> 2) + (r & 3) + odd;
            if (row >= o.m || c0 >= o.n) continue;
            E* p = out + row * o.ov.ld + c0;
            const float a = odd ? other : mine, z = odd ? mine : other;
            if (c0 + 1 < o.n) {
                E2 v;
                if (step) v = *(const E2*)p;
                v[0] = (E)(step ? fmaf(lr, a, keep * (float)v[0]) : a);
                v[1] = (E)(step ? fmaf(lr, z, keep * (float)v[1]) : z);
                *(E2*)p = v;
            } else put(p, a);
        }
        return;
    }
    if (col >= o.n) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = row0 + 8 * (r >> 2) + (r & 3);
        if (row < o.m) put(out + row * o.ov.ld + col, acc[r] * c);
    }
}
__device__ __forceinline__ void store_result(const Output& o, int b, int bi, int bj, int lane, const f32x16& acc, float c) {
    if (o.dtype == F32) store_block<float>(o, b, bi, bj, lane, acc, c);
    else if (o.dtype == F16) store_block<_Float16>(o, b, bi, bj, lane, acc, c);
    else store_block<__bf16>(o, b, bi, bj, lane, acc, c);
}

struct NsGemm {
    const _Float16 *a, *b;                   // fragment-order operands, rows x K each: result[i][j] = sum_k a[i][k] b[j][k]
    long long a_bs, b_bs;                    // halfs per matrix
    int nk16;                                // K / 16
    int tiles_i, n_tiles;                    // tiles along i, tiles of a matrix
    int full, rest, slices;                  // of all matrices' tiles: the first `full` in one piece, the `rest` in `slices` pieces of K each
    float* part; int* count;                 // split K: partial tiles and arrival counters
    _Float16 *o, *ot;                        // FULL: result (k = j), transposed result (k = i); GRAM / POLY: ot only (symmetric)
    long long o_bs, ot_bs;
    int o_nk16, ot_nk16;
    const _Float16* am;                      // POLY: A
    float c0, c1, c2;                        // POLY: c0 on the diagonal, c1 A, c2 acc; others: c2 acc
    const Scalars* sc;
    int step, dec;                           // e_k = max(0, e0 - k dec)
    Output fin;                              // FINAL
};

template <int N> __device__ __forceinline__ void wait_vm_lgkm() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// 32 x 32 accumulator tile whose lane is the ROW of the stored matrix: rows 32 rowblk .. + 31, k = 16 k16 .. + 31
template <int P>
__device__ __forceinline__ void store_frag(_Float16* __restrict__ base, int nk16, int rowblk, int k16, int lane, const half4 (&hi)[4], const half4 (&lo)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        _Float16* d = base + ((long long)rowblk * nk16 + k16 + (q >> 1)) * P * 512 + ((lane & 31) + 32 * (q & 1)) * 8 + 4 * (lane >> 5);
        *(half4*)d = hi[q];
        if (P == 2) *(half4*)(d + 512) = lo[q];
    }
}

// lane / register roles of a tile exchanged: t[c][r] of v[r][c], exact
__device__ __forceinline__ void transpose_tile(const half4 (&v)[4], const half8 (&ident)[2], half4 (&t)[4]) {
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
    for (int pi = 0; pi < 2; ++pi) {
        const half8 a = __builtin_shufflevector(v[2 * pi], v[2 * pi + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ident[pi], acc, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) t[r >> 2][r & 3] = (_Float16)acc[r];
}

// One workgroup = a tile of (32 TM WR) x (32 TN WC) of one matrix (or one K slice of it): WR x WC waves, a wave = TM x TN accumulator tiles; NST stages
// of KS k steps in LDS.  Bound by the matrix cores where the tiles are large: X <- M X of [4096, 4096] 350 us (137 GFLOP in three MFMAs each: 1178 TFLOP/s
// of fp16; the library's bf16 product runs at 1214), on one plane 124 us (1108), of [20, 768, 1152] 106 us (768).  A tile of 64 reads two fragments per MFMA from
// LDS (X X^T of [2048, 8192] 136 us, 780 TFLOP/s, on one plane 64 us, 541), and one [384, 384] product is 6.9 us of latency.
template <int P_, int TM_, int TN_, int WR_, int WC_, int KS_, int NST_, int PER_CU_>
struct Tile {
    static constexpr int P = P_, TM = TM_, TN = TN_, WR = WR_, WC = WC_, KS = KS_, NST = NST_, PER_CU = PER_CU_;
    static constexpr int NW = WR * WC, RA = TM * WR, RB = TN * WC, U = KS * P, PIECES = (RA + RB) * U, PER = PIECES / NW;
    static constexpr int LDS = PIECES * NST * 1024;
    static_assert(PIECES % NW == 0 && PER * (NST - 2) < 64 && LDS * PER_CU <= 160 * 1024, "");
};

template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }

template <class C, int MODE>
__global__ __launch_bounds__(C::NW * 64) void k_ns_gemm(const NsGemm g) {
    constexpr int P = C::P, TM = C::TM, TN = C::TN, WC = C::WC, KS = C::KS, NST = C::NST, NW = C::NW, RA = C::RA, RB = C::RB, U = C::U, PIECES = C::PIECES, PER = C::PER;
    constexpr int TILE4 = TM * TN * 4 * NW * 64;                                   // f32x4 of a tile
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr int CHAINS = TM * TN == 1 && P == 2 ? 3 : 1;                         // one accumulator tile: the three products run as chains of their own
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // workgroups of one XCD (id % 8) take neighbouring tiles: they share operand rows in its L2, and the slices of a tile meet there
    int at, slice = 0, slices = 1;
    {
        const int first = (g.full + 7) & ~7, id = blockIdx.x;
        if (id < first) {
            at = (id & 7) * (first >> 3) + (id >> 3);
            if (at >= g.full) return;
        } else {
            const int units = g.rest * g.slices, per = (units + 7) >> 3, u = ((id - first) & 7) * per + ((id - first) >> 3);
            if (u >= units) return;
            slices = g.slices;
            at = u / slices;
            slice = u - at * slices;
            at += g.full;
        }
    }
    const int b = at / g.n_tiles, tile = at - b * g.n_tiles;
    int ti, tj;
    if (SYM) {
        tj = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
        while ((tj + 1) * (tj + 2) / 2 <= tile) ++tj;
        while (tj * (tj + 1) / 2 > tile) --tj;
        ti = tile - tj * (tj + 1) / 2;
    } else {
        tj = tile / g.tiles_i;
        ti = tile - tj * g.tiles_i;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wr = wave / WC, wc = wave % WC;
    const int all = g.nk16 / KS, s_begin = slice * all / slices, n_stages = (slice + 1) * all / slices - s_begin;
    const _Float16* abase = g.a + b * g.a_bs + (long long)ti * RA * g.nk16 * P * 512;
    const _Float16* bbase = g.b + b * g.b_bs + (long long)tj * RB * g.nk16 * P * 512;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

    auto dma = [&](int s) {
        char* dst = smem + (s % NST) * (PIECES * 1024);
        const long long k = (long long)(s_begin + s) * U;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int pc = wave + NW * i, rb = pc / U, u = pc % U;
            const _Float16* src = (rb < RA ? abase + (long long)rb * g.nk16 * (P * 512) : bbase + (long long)(rb - RA) * g.nk16 * (P * 512)) + (k + u) * 512 + lane * 8;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)(dst + pc * 1024), 16, 0, 0);
        }
    };

    f32x16 acc[TM][TN], more[CHAINS];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j][r] = 0.f;
#pragma unroll
        for (int c = 0; c < CHAINS; ++c) more[c][r] = 0.f;
    }

#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < n_stages) dma(s);
    for (int s = 0; s < n_stages; ++s) {
        // this wave's copies of stage s have landed (vmcnt retires in order) and its own LDS reads of stage s - 1 are done; behind the barrier
        // that holds for every wave, so buffer (s + NST - 1) % NST = (s - 1) % NST may be overwritten
        if (s + NST - 2 < n_stages) wait_vm_lgkm<PER * (NST - 2)>();
        else wait_vm_lgkm<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const unsigned buf = lds0 + (unsigned)(s % NST) * (PIECES * 1024) + (unsigned)lane * 16u;
        half8 fa[2][TM][P], fb[2][TN][P];
        auto load = [&](int k) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[k & 1][i][p] = *(lds_half8)(size_t)(buf + (unsigned)(((wr * TM + i) * U + k * P + p) * 1024));
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[k & 1][j][p] = *(lds_half8)(size_t)(buf + (unsigned)(((RA + wc * TN + j) * U + k * P + p) * 1024));
            }
        };
        load(0);
        if (s + NST - 1 < n_stages) dma(s + NST - 1);     // (issued under the latency of the first fragments' reads)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (k + 1 < KS) load(k + 1);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[k & 1][i][0], fb[k & 1][j][0], acc[i][j], 0, 0, 0);
                    if constexpr (P == 2) {
                        f32x16& x1 = CHAINS > 1 ? more[1 % CHAINS] : acc[i][j];
                        f32x16& x2 = CHAINS > 1 ? more[2 % CHAINS] : acc[i][j];
                        x1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[k & 1][i][1], fb[k & 1][j][0], x1, 0, 0, 0);
                        x2 = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[k & 1][i][0], fb[k & 1][j][1], x2, 0, 0, 0);
                    }
                }
        }
    }
    if constexpr (CHAINS > 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][0][r] += more[1 % CHAINS][r] + more[2 % CHAINS][r];
    }

    if (slices > 1) {
        // every slice leaves its partial tile; the workgroup that arrives last adds them up in slice order (whoever it is: the same sum).  The partials
        // go through agent-scope accesses, which pass the XCDs' own L2s: a fence would write a whole L2 back (__threadfence() here made a
        // [2048, 2048] fp32 call 1.40 instead of 0.89 ms)
        typedef unsigned long long u64;
        const int slot = at - g.full;
        auto part = [&](int z, int x) { return (u64*)g.part + (((long long)slot * slices + z) * TILE4 + x * (NW * 64) + threadIdx.x) * 2; };
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 v = make_float2(acc[i][j][4 * q + 2 * h], acc[i][j][4 * q + 2 * h + 1]);
                        __hip_atomic_store(part(slice, (i * TN + j) * 4 + q) + h, __builtin_bit_cast(u64, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // this wave's partials are where every XCD sees them ...
        __syncthreads();                                         // ... and so are the workgroup's
        int* last = (int*)smem;
        if (threadIdx.x == 0) {
            const int n = __hip_atomic_fetch_add(g.count + slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *last = n == slices - 1;
            if (n == slices - 1) __hip_atomic_store(g.count + slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // for the next launch
        }
        __syncthreads();
        if (!*last) return;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        for (int z = 0; z < slices; ++z)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 v = __builtin_bit_cast(float2, __hip_atomic_load(part(z, (i * TN + j) * 4 + q) + h, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                            acc[i][j][4 * q + 2 * h] += v.x;
                            acc[i][j][4 * q + 2 * h + 1] += v.y;
                        }
    }

    // ---- epilogue: registers and lanes as in store_result ----
    const int e0 = g.sc[b].e0, ek = max(0, e0 - g.step * g.dec), ek1 = max(0, e0 - (g.step + 1) * g.dec);
    float c2 = g.c2;
    if (MODE == GRAM) c2 = ldexpf(c2, -2 * ek);
    if (MODE == FULL) c2 = ldexpf(c2, ek1 - ek);
    if (MODE == FINAL) c2 = ldexpf(c2, -ek);
    if constexpr (MODE == FINAL) {           // (not a loop: with this body hipcc keeps one, and the accumulators in scratch)
        auto put = [&](auto ij) {
            constexpr int i = decltype(ij)::value / TN, j = decltype(ij)::value % TN;
            store_result(g.fin, b, ti * RA + wr * TM + i, tj * RB + wc * TN + j, lane, acc[i][j], c2);
        };
        each(put, std::make_integer_sequence<int, TM * TN>{});
        return;
    }
    half8 ident[2];
#pragma unroll
    for (int pi = 0; pi < 2; ++pi)
#pragma unroll
        for (int e = 0; e < 8; ++e) ident[pi][e] = (lane & 31) == 16 * pi + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int bi = ti * RA + wr * TM + i, bj = tj * RB + wc * TN + j;      // 32-blocks of the result
            {
                half4 am_hi[4], am_lo[4];
                if constexpr (MODE == POLY) {
                    const _Float16* am = g.am + b * g.ot_bs;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const _Float16* s = am + ((long long)bj * g.ot_nk16 + 2 * bi + (q >> 1)) * P * 512 + ((lane & 31) + 32 * (q & 1)) * 8 + 4 * (lane >> 5);
                        am_hi[q] = *(const half4*)s;
                        if (P == 2) am_lo[q] = *(const half4*)(s + 512);
                    }
                }
                half4 hi[4], lo[4];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = acc[i][j][r] * c2;
                    if constexpr (MODE == POLY) {
                        float am = (float)am_hi[r >> 2][r & 3];
                        if (P == 2) am += (float)am_lo[r >> 2][r & 3];
                        v = fmaf(g.c1, am, v);
                        if (bi == bj && 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) == (lane & 31)) v += g.c0;
                    }
                    v = one_value(v);
                    hi[r >> 2][r & 3] = (_Float16)v;
                    if (P == 2) lo[r >> 2][r & 3] = (_Float16)(v - (float)hi[r >> 2][r & 3]);
                }
                store_frag<P>(g.ot + b * g.ot_bs, g.ot_nk16, bj, 2 * bi, lane, hi, lo);
                if (MODE == FULL || ti != tj) {
                    half4 th[4], tl[4];
                    transpose_tile(hi, ident, th);
                    if (P == 2) transpose_tile(lo, ident, tl);
                    if (MODE == FULL) store_frag<P>(g.o + b * g.o_bs, g.o_nk16, bi, 2 * bj, lane, th, tl);
                    else store_frag<P>(g.ot + b * g.ot_bs, g.ot_nk16, bi, 2 * bj, lane, th, tl);
                }
            }
        }
}

// ---- a whole matrix in one workgroup and one launch ----------------------------------------------------------------------------------------
// Small matrices are bound by launches: 17 of them take 70 us of GPU or 60 us of host time whatever the size.  Here one workgroup of 16 waves
// normalises, iterates and stores: A and M lie in LDS, X and X^T too where they fit (LOCAL; else in the workspace: the CU's own writes and reads).
// MB = 32-row blocks of X; Gram's K is shared out to G = 16 / MB^2 groups of waves and added up in LDS.  A wave takes 32 columns of X from X^T, and
// writes them back in place: nobody else reads them before the barrier.
struct OneArgs {
    const void* in; View iv;
    int rows, cols;
    _Float16 *x, *xt;                        // per matrix 32 MB x np x P halfs each
    int np;                                  // columns, padded to 32
    double eps;
    int steps, dec;
    float c0, c1, c2, scale;
    MuonArgs mu;
    Output fin;
};
constexpr int one_groups(int mb) { return 16 / (mb * mb); }
// LDS: A, M, partial Gram tiles; X and X^T for LOCAL
constexpr int one_lds(int mb, int p, int np) { return 2 * mb * 2 * mb * p * 1024 + (one_groups(mb) - 1) * mb * mb * 4096 + 2 * 32 * mb * np * p * 2; }

template <int P>
__device__ __forceinline__ void split(const f32x16& v, half4 (&hi)[4], half4 (&lo)[4]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float x = one_value(v[r]);
        hi[r >> 2][r & 3] = (_Float16)x;
        if (P == 2) lo[r >> 2][r & 3] = (_Float16)(x - (float)hi[r >> 2][r & 3]);
    }
}
template <int P>
__device__ __forceinline__ void mfma_split(const half8 (&a)[P], const half8 (&b)[P], f32x16& acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc, 0, 0, 0);
    if constexpr (P == 2) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], acc, 0, 0, 0);
    }
}

template <int T, bool MUON, int P, int MB, bool LOCAL>
__global__ __launch_bounds__(1024) void k_ns_one(const OneArgs g) {
    typedef typename Elem<T>::type E;
    constexpr int WAVES = 16, KM = 2 * MB, G = one_groups(MB), AH = MB * KM * P * 512;       // k steps of A; groups; halfs of A
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    _Float16 *la = (_Float16*)smem, *lm = la + AH;               // A, M in fragment order
    f32x4* red = (f32x4*)(lm + AH);                              // partial Gram tiles of groups 1 .. G - 1
    __shared__ double sums[WAVES];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const E* src = (const E*)g.in + b * g.iv.bs;
    float* mom = MUON ? g.mu.mom + b * g.mu.mv.bs : nullptr;
    const float gs = MUON ? (g.mu.gscale_dev ? *g.mu.gscale_dev : g.mu.gscale) : 1.f;
    // ---- norm, and the momentum update ----
    double s = 0.0;
    {
        const unsigned cols = g.cols, n = (unsigned)g.rows * cols;
        for (unsigned i0 = tid; i0 < n; i0 += 4 * WAVES * 64) {
            float v[4], m[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned i = i0 + WAVES * 64 * k, r = i / cols, c = i - r * cols;
                v[k] = i < n ? (float)src[r * g.iv.ld + c] : 0.f;
                if (MUON) m[k] = i < n ? mom[r * g.mu.mv.ld + c] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned i = i0 + WAVES * 64 * k, r = i / cols, c = i - r * cols;
                if (MUON && i < n) {
                    v[k] *= gs;
                    m[k] = muon_mom(g.mu, v[k], m[k]);
                    mom[r * g.mu.mv.ld + c] = m[k];
                    v[k] = muon_u(g.mu, v[k], m[k]);
                }
                s = fma((double)v[k], (double)v[k], s);
            }
        }
    }
    for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += sums[w];
    const double norm = sqrt(s), t = norm / (norm + g.eps);
    int e0 = 0;
    if (t < 0.5) e0 = t > 1e-18 ? -ilogb(t) - 1 : 59;            // (as k_ns_prep)
    const double f = ldexp((double)X_SCALE, e0) / (norm + g.eps);
    // ---- normalised fragments of X and X^T ----
    const int nk = g.np >> 4, jb = g.np >> 5;                    // k steps and 32-column blocks of X
    const long long xs = (long long)32 * MB * g.np * P;
    _Float16 *x, *xt;
    if constexpr (LOCAL) { x = (_Float16*)(red + (G - 1) * MB * MB * 256); xt = x + 32 * MB * g.np * P; }
    else { x = g.x + b * xs; xt = g.xt + b * xs; }
    for (int q = wave; q < 2 * MB * nk; q += WAVES) {
        const bool tr = q >= MB * nk;
        const int z = tr ? q - MB * nk : q, blk = tr ? z / KM : z / nk, k16 = tr ? z - blk * KM : z - blk * nk;
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int p0 = 32 * blk + (lane & 31), p1 = 16 * k16 + 8 * (lane >> 5) + e;       // (row, column) of X, or (column, row)
            const int r = tr == (g.fin.tall != 0) ? p0 : p1, c = tr == (g.fin.tall != 0) ? p1 : p0;
            float v = 0.f;
            if (r < g.rows && c < g.cols) {
                v = (float)src[r * g.iv.ld + c];
                if (MUON) v = muon_u(g.mu, v * gs, mom[r * g.mu.mv.ld + c]);
                v = (float)((double)v * f);
            }
            v = one_value(v);
            hi[e] = (_Float16)v;
            lo[e] = (_Float16)(v - (float)hi[e]);
        }
        _Float16* d = (tr ? xt + ((long long)blk * KM + k16) * P * 512 : x + ((long long)blk * nk + k16) * P * 512) + lane * 8;
        *(half8*)d = hi;
        if (P == 2) *(half8*)(d + 512) = lo;
    }
    __syncthreads();
    half8 ident[2];
#pragma unroll
    for (int pi = 0; pi < 2; ++pi)
#pragma unroll
        for (int e = 0; e < 8; ++e) ident[pi][e] = (lane & 31) == 16 * pi + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) ? (_Float16)1.f : (_Float16)0.f;
    const int grp = wave / (MB * MB), tile = wave % (MB * MB), bi = tile / MB, bj = tile % MB, used = nk < G ? nk : G;      // groups with a k step
    for (int step = 0; step < g.steps; ++step) {
        const int ek = max(0, e0 - step * g.dec), ek1 = max(0, e0 - (step + 1) * g.dec);
        half4 hi[4], lo[4];
        f32x16 acc;
        // ---- A = X X^T ----
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
        {
            const _Float16 *pa = x + (long long)bi * nk * P * 512 + lane * 8, *pb = x + (long long)bj * nk * P * 512 + lane * 8;
            constexpr int R = 4;                                 // k steps in flight
            for (int k0 = grp; k0 < nk; k0 += R * G) {
                half8 fa[R][P], fb[R][P];
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const int k = k0 + u * G < nk ? k0 + u * G : k0;
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        fa[u][p] = *(const half8*)(pa + ((long long)k * P + p) * 512);
                        fb[u][p] = *(const half8*)(pb + ((long long)k * P + p) * 512);
                    }
                }
#pragma unroll
                for (int u = 0; u < R; ++u)
                    if (k0 + u * G < nk) mfma_split<P>(fa[u], fb[u], acc);
            }
        }
        if (grp > 0 && grp < used) {
#pragma unroll
            for (int q = 0; q < 4; ++q) red[((grp - 1) * MB * MB + tile) * 256 + q * 64 + lane] = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
        }
        __syncthreads();
        if (grp == 0) {
#pragma unroll 3
            for (int z = 0; z < used - 1; ++z)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = red[(z * MB * MB + tile) * 256 + q * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[4 * q + e] += v[e];
                }
            const float c = ldexpf(A_SCALE / (X_SCALE * X_SCALE), -2 * ek);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] *= c;
            split<P>(acc, hi, lo);
            store_frag<P>(la, KM, bj, 2 * bi, lane, hi, lo);
        }
        __syncthreads();
        // ---- M = c0 I + c1 A + c2 A A ----
        if (grp == 0) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
            for (int k = 0; k < KM; ++k) {
                half8 fa[P], fb[P];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    fa[p] = *(const half8*)(la + ((bi * KM + k) * P + p) * 512 + lane * 8);
                    fb[p] = *(const half8*)(la + ((bj * KM + k) * P + p) * 512 + lane * 8);
                }
                mfma_split<P>(fa, fb, acc);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int q = r >> 2, d = ((bj * KM + 2 * bi + (q >> 1)) * P) * 512 + ((lane & 31) + 32 * (q & 1)) * 8 + 4 * (lane >> 5) + (r & 3);
                float am = (float)la[d];
                if (P == 2) am += (float)la[d + 512];
                acc[r] = fmaf(g.c1, am, acc[r] * g.c2);
                if (bi == bj && 8 * q + 4 * (lane >> 5) + (r & 3) == (lane & 31)) acc[r] += g.c0;
            }
            split<P>(acc, hi, lo);
            store_frag<P>(lm, KM, bj, 2 * bi, lane, hi, lo);
        }
        __syncthreads();
        // ---- X <- M X: a wave takes 32 columns at a time ----
        const bool last = step + 1 == g.steps;
        const float c = last ? ldexpf(g.scale / (A_SCALE * X_SCALE), -ek) : ldexpf(1.f / A_SCALE, ek1 - ek);
        for (int j = wave; j < jb; j += WAVES) {
            half8 fb[KM][P];
#pragma unroll
            for (int k = 0; k < KM; ++k)
#pragma unroll
                for (int p = 0; p < P; ++p) fb[k][p] = *(const half8*)(xt + (((long long)j * KM + k) * P + p) * 512 + lane * 8);
#pragma unroll 1
            for (int i = 0; i < MB; ++i) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
                for (int k = 0; k < KM; ++k) {
                    half8 fa[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) fa[p] = *(const half8*)(lm + ((i * KM + k) * P + p) * 512 + lane * 8);
                    mfma_split<P>(fa, fb[k], acc);
                }
                if (last) {
                    store_result(g.fin, b, i, j, lane, acc, c);
                    continue;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] *= c;
                split<P>(acc, hi, lo);
                store_frag<P>(xt, KM, j, 2 * i, lane, hi, lo);
                half4 th[4], tl[4];
                transpose_tile(hi, ident, th);
                if (P == 2) transpose_tile(lo, ident, tl);
                store_frag<P>(x, nk, i, 2 * j, lane, th, tl);
            }
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
// Tiles.  128: 64 x 64 per wave (4 or 8 fragment reads feed 4 or 12 MFMAs), two workgroups a CU hide each other's barriers; four stages of 16 k at two
// planes (against two of 32: [768, 384] x 20 fp32 272 -> 253 us, [768, 1152] x 20 1055 -> 1031, [4096, 4096] 4.01 -> 4.10 ms), two of 64 at one.  ALONE: the
// same tile by eight waves, where there is about one to a CU ([2048, 2048] fp32: 757 -> 690 us, [1000, 3000] 362 -> 334).  256: 128 x 64 per wave, fewer LDS
// reads per MFMA.  64: a wave has one accumulator tile, four stages ahead; for grids that 128 leaves mostly empty.
constexpr int ALONE = 129;                   // a tile of 128 with a CU to itself
template <int P, int SIZE> struct Tiles;
template <> struct Tiles<1, 64> { typedef Tile<1, 1, 1, 2, 2, 4, 4, 2> type; };
template <> struct Tiles<2, 64> { typedef Tile<2, 1, 1, 2, 2, 2, 4, 2> type; };
template <> struct Tiles<1, 128> { typedef Tile<1, 2, 2, 2, 2, 4, 2, 2> type; };
template <> struct Tiles<2, 128> { typedef Tile<2, 2, 2, 2, 2, 1, 4, 2> type; };
template <> struct Tiles<1, ALONE> { typedef Tile<1, 1, 2, 4, 2, 8, 2, 1> type; };
template <> struct Tiles<2, ALONE> { typedef Tile<2, 1, 2, 4, 2, 4, 2, 1> type; };
template <> struct Tiles<1, 256> { typedef Tile<1, 4, 2, 2, 4, 4, 2, 1> type; };

constexpr int CUS = 256;

// How one product is cut: the tile's edge, and which tiles are split along K.
struct Cut {
    int kind, size, tiles_i, n_tiles, full, rest, slices;
    long long part_bytes() const { return slices > 1 ? (long long)rest * slices * size * size * 4 : 0; }
};
// A slice keeps at least 16 stages: a partial tile's way through memory costs about as much as 8 ([4, 1024, 1024] on one plane: 253 us whole, 344 us in
// slices of 8 or more; [100, 4000] fp32: 250 us whole, 124 us in slices of 16; the last 16 of [4096, 4096]'s 528 tiles on one plane: 1783 -> 1638 us).
constexpr int MIN_STAGES = 16;
template <class C>
Cut cut_for(int kind, bool sym, int batch, int mi, int nj, int k16) {
    const int size = 32 * C::TM * C::WR;
    Cut c{};
    c.kind = kind; c.size = size;
    c.tiles_i = mi / size;
    c.n_tiles = sym ? c.tiles_i * (c.tiles_i + 1) / 2 : c.tiles_i * (nj / size);
    const long long total = (long long)batch * c.n_tiles, slots = C::PER_CU * CUS;
    c.rest = (int)(total % slots);
    c.full = (int)(total - c.rest);
    c.slices = 1;
    if (c.rest) {
        const long long by_slots = slots / c.rest, by_work = k16 / C::KS / MIN_STAGES;
        c.slices = (int)(by_slots < by_work ? by_slots : by_work);
        if (c.slices > 16) c.slices = 16;
    }
    if (c.slices <= 1) { c.slices = 1; c.full = (int)total; c.rest = 0; }
    return c;
}
template <int P>
Cut cut(bool sym, int batch, int mi, int nj, int k16) {
    // 128 where that gives about every CU a tile ([1000, 3000] fp32 on 36 ... 192 tiles of 128 by four waves: 665 us, on tiles of 64: 376 us; [2048, 2048]'s
    // symmetric products on 136 tiles in K slices: 869 us, on tiles of 64: 781 us).  256 where it still gives one to each and nothing is padded for it
    // ([4096, 4096] on one plane, the full product: 158 -> 140 us)
    const int t = mi / 128;
    const long long tiles = (long long)batch * (sym ? t * (t + 1) / 2 : (long long)t * (nj / 128));
    if (P == 1 && !sym && mi % 256 == 0 && nj % 256 == 0 && tiles >= 4 * CUS) return cut_for<typename Tiles<1, 256>::type>(256, sym, batch, mi, nj, k16);
    if (tiles > CUS) return cut_for<typename Tiles<P, 128>::type>(128, sym, batch, mi, nj, k16);
    if (tiles >= CUS * 3 / 4) return cut_for<typename Tiles<P, ALONE>::type>(ALONE, sym, batch, mi, nj, k16);
    return cut_for<typename Tiles<P, 64>::type>(64, sym, batch, mi, nj, k16);
}

template <class C, int MODE>
int launch_gemm(const NsGemm& g, hipStream_t st) {
    auto kernel = k_ns_gemm<C, MODE>;
    if (C::LDS > 64 * 1024) DSVC_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS));
    const int grid = (g.full + 7) / 8 * 8 + (g.rest * g.slices + 7) / 8 * 8;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(C::NW * 64), C::LDS, st, g);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}
template <int P, int MODE>
int gemm(NsGemm& g, const Cut& c, hipStream_t st) {
    g.tiles_i = c.tiles_i; g.n_tiles = c.n_tiles; g.full = c.full; g.rest = c.rest; g.slices = c.slices;
    if constexpr (P == 1 && (MODE == FULL || MODE == FINAL)) {
        if (c.kind == 256) return launch_gemm<typename Tiles<1, 256>::type, MODE>(g, st);
    }
    if (c.kind == 128) return launch_gemm<typename Tiles<P, 128>::type, MODE>(g, st);
    if (c.kind == ALONE) return launch_gemm<typename Tiles<P, ALONE>::type, MODE>(g, st);
    return launch_gemm<typename Tiles<P, 64>::type, MODE>(g, st);
}

struct Plan {
    int P, m, n, mp, np, tall, n_part, dec;
    int one, local;                          // 32-row blocks of X where one workgroup takes a matrix (k_ns_one), else 0; with X in LDS
    Cut gram, poly, full;
    long long off_part, off_sc, off_count, n_count, off_split, off_x, off_xt[2], off_a, off_m, bytes;
};

// The largest singular value that the polynomial can reach from [0, 1] and the largest |a + b s^2 + c s^4| on the way: both stay far from where the
// fp16 planes end (65504 / X_SCALE, 65504 / A_SCALE).
int check_coefficients(const float* c, int steps, double* growth) {
    double s_max = 1.0, most = 0.0;
    for (int k = 0; k < 3; ++k)
        if (!isfinite(c[k])) return fail(DSVC_EINVAL, "orthogonalize: coefficient %d is not finite", k);
    for (int k = 0; k < steps; ++k) {
        // extrema on [0, s_max], with l = s^2: of f = a + b l + c l^2 at the ends and where b + 2 c l = 0, of s f at the end and where a + 3 b l + 5 c l^2 = 0
        const double A = c[0], B = c[1], C = c[2], top = s_max * s_max, disc = 9.0 * B * B - 20.0 * A * C;
        double next = 0.0, at[5] = {0.0, top, C != 0.0 ? -B / (2.0 * C) : -1.0, -1.0, -1.0};
        if (C != 0.0 && disc >= 0.0) { at[3] = (-3.0 * B + sqrt(disc)) / (10.0 * C); at[4] = (-3.0 * B - sqrt(disc)) / (10.0 * C); }
        else if (C == 0.0 && B != 0.0) at[3] = -A / (3.0 * B);
        for (double l : at) {
            if (!(l >= 0.0 && l <= top)) continue;
            const double f = fabs(A + l * (B + l * C));
            if (f > most) most = f;
            if (f * sqrt(l) > next) next = f * sqrt(l);
        }
        s_max = 1.01 * next;
        if (s_max * s_max > 48.0 || most > 48.0 || s_max > 12.0)
            return fail(DSVC_EINVAL, "orthogonalize: the coefficients (%g, %g, %g) take singular values from [0, 1] to %g", c[0], c[1], c[2], s_max);
        if (s_max < 1.0) s_max = 1.0;
    }
    *growth = most;
    return DSVC_OK;
}

int make_plan(const dsvc_ortho_cfg* c, Plan* p) {
    if (!c) return fail(DSVC_EINVAL, "null argument");
    if (c->dtype < F32 || c->dtype > BF16) return fail(DSVC_EINVAL, "orthogonalize: unknown type %d", c->dtype);
    if (c->planes != 0 && c->planes != 1 && c->planes != 2) return fail(DSVC_EINVAL, "orthogonalize: %d planes (1, 2 or 0: 2)", c->planes);
    if (c->batch < 0 || c->rows < 0 || c->cols < 0) return fail(DSVC_EINVAL, "orthogonalize: bad shape [%d, %d, %d]", c->batch, c->rows, c->cols);
    if (c->rows > (1 << 20) || c->cols > (1 << 20) || c->batch > 65535) return fail(DSVC_EINVAL, "orthogonalize: shape [%d, %d, %d] is too large", c->batch, c->rows, c->cols);
    if (c->steps < 1 || c->steps > 64) return fail(DSVC_EINVAL, "orthogonalize: %d steps", c->steps);
    if (!(c->eps >= 0.f) || !isfinite(c->eps)) return fail(DSVC_EINVAL, "orthogonalize: eps %g", c->eps);
    if (!isfinite(c->scale)) return fail(DSVC_EINVAL, "orthogonalize: scale %g", c->scale);
    double growth = 0.0;
    DSVC_TRY(check_coefficients(c->coef, c->steps, &growth));
    *p = Plan{};
    p->dec = growth > 1.0 ? (int)ceil(log2(growth) + 1e-6) : 0;
    p->tall = c->rows > c->cols;
    p->m = p->tall ? c->cols : c->rows;
    p->n = p->tall ? c->rows : c->cols;
    p->P = c->planes ? c->planes : 2;
    if (!c->batch || !p->m) return DSVC_OK;
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 1023) / 1024 * 1024; return o; };
    const int mb = p->m <= 32 ? 1 : 2;
    if (p->m <= 64 && (long long)32 * mb * p->n <= ONE_WORK) {
        p->one = mb;
        p->mp = 32 * mb;
        p->np = round_up(p->n, 32);
        p->local = one_lds(mb, p->P, p->np) <= ONE_LDS;
        const long long xs = p->local ? 0 : (long long)c->batch * p->mp * p->np * p->P * 2;
        p->off_x = take(xs);
        p->off_xt[0] = take(xs);
        p->bytes = at ? at : 256;
        return DSVC_OK;
    }
    p->mp = round_up(p->m, PAD);
    p->np = round_up(p->n, PAD);
    if ((long long)c->batch * (p->mp / 64) * (p->np / 64) >= (1LL << 22)) return fail(DSVC_EINVAL, "orthogonalize: shape [%d, %d, %d] is too large", c->batch, c->rows, c->cols);
    if (p->P == 1) {
        p->gram = cut<1>(true, c->batch, p->mp, p->mp, p->np / 16);
        p->poly = cut<1>(true, c->batch, p->mp, p->mp, p->mp / 16);
        p->full = cut<1>(false, c->batch, p->mp, p->np, p->mp / 16);
    } else {
        p->gram = cut<2>(true, c->batch, p->mp, p->mp, p->np / 16);
        p->poly = cut<2>(true, c->batch, p->mp, p->mp, p->mp / 16);
        p->full = cut<2>(false, c->batch, p->mp, p->np, p->mp / 16);
    }
    const long long want = ((long long)p->m * p->n + 8191) / 8192;
    p->n_part = (int)(want < SUM_BLOCKS ? want : SUM_BLOCKS);
    const long long B = c->batch, xs = B * p->mp * p->np * p->P * 2, as = B * p->mp * p->mp * p->P * 2;
    p->off_part = take(B * p->n_part * 8);
    p->off_sc = take(B * (long long)sizeof(Scalars));
    long long split = 0;
    for (const Cut* k : {&p->gram, &p->poly, &p->full}) {
        if (k->rest > p->n_count) p->n_count = k->rest;
        if (k->part_bytes() > split) split = k->part_bytes();
    }
    p->off_count = take(p->n_count * 4);
    p->off_split = take(split);
    p->off_x = take(xs);
    p->off_xt[0] = take(xs);
    p->off_xt[1] = take(xs);
    p->off_a = take(as);
    p->off_m = take(as);
    p->bytes = at;
    return DSVC_OK;
}

Output output(const dsvc_ortho_cfg* c, const Plan& p, void* out, View ov, const MuonArgs& mu) {
    const int size = c->dtype == F32 ? 4 : 2, together = p.tall ? 4 : 2;
    const bool wide = (uintptr_t)out % (size * together) == 0 && ov.ld % together == 0 && (c->batch == 1 || ov.bs % together == 0);
    return Output{out, ov, c->dtype, p.m, p.n, p.tall, wide, mu};
}

template <int T, bool MUON, int P, int MB, bool LOCAL>
int one_mb(const OneArgs& g, int batch, hipStream_t st) {
    const int lds = one_lds(MB, P, LOCAL ? g.np : 0);
    if (lds > 64 * 1024) DSVC_HIP(hipFuncSetAttribute((const void*)k_ns_one<T, MUON, P, MB, LOCAL>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL((k_ns_one<T, MUON, P, MB, LOCAL>), dim3(batch), dim3(1024), lds, st, g);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}
template <int T, bool MUON, int P>
int one(const dsvc_ortho_cfg* c, const Plan& p, const void* in, View iv, void* out, View ov, const MuonArgs& mu, char* ws, hipStream_t st) {
    const OneArgs g{in, iv, c->rows, c->cols, (_Float16*)(ws + p.off_x), (_Float16*)(ws + p.off_xt[0]), p.np, (double)c->eps, c->steps, p.dec,
                    c->coef[0] * A_SCALE, c->coef[1], c->coef[2] / A_SCALE, c->scale, mu, output(c, p, out, ov, mu)};
    if (p.one == 1) return p.local ? one_mb<T, MUON, P, 1, true>(g, c->batch, st) : one_mb<T, MUON, P, 1, false>(g, c->batch, st);
    return p.local ? one_mb<T, MUON, P, 2, true>(g, c->batch, st) : one_mb<T, MUON, P, 2, false>(g, c->batch, st);
}

template <int T, bool MUON, int P>
int prep(const dsvc_ortho_cfg* c, const Plan& p, const void* in, View iv, const MuonArgs& mu, char* ws, hipStream_t st) {
    constexpr int VEC = T == F32 ? 4 : 8;
    const bool flat = (c->rows == 1 || iv.ld == c->cols) && (!MUON || c->rows == 1 || mu.mv.ld == c->cols);
    const int rows = flat ? 1 : c->rows;
    const long long cols = flat ? (long long)c->rows * c->cols : c->cols;
    auto fits = [&](const void* q, const View& v, int esize) {
        return (uintptr_t)q % 16 == 0 && (rows == 1 || v.ld * esize % 16 == 0) && (c->batch == 1 || v.bs * esize % 16 == 0);
    };
    const bool vec = cols % VEC == 0 && fits(in, iv, T == F32 ? 4 : 2) && (!MUON || fits(mu.mom, mu.mv, 4));
    double* part = (double*)(ws + p.off_part);
    int* count = (int*)(ws + p.off_count);
    if (vec) hipLaunchKernelGGL((k_ns_sums<T, MUON, VEC>), dim3(p.n_part, c->batch), dim3(256), 0, st, in, iv, rows, cols, mu, part, count, (int)p.n_count);
    else hipLaunchKernelGGL((k_ns_sums<T, MUON, 1>), dim3(p.n_part, c->batch), dim3(256), 0, st, in, iv, rows, cols, mu, part, count, (int)p.n_count);
    hipLaunchKernelGGL((k_ns_prep<T, MUON, P>), dim3(p.np / 64, p.mp / 64, c->batch), dim3(256), 0, st, in, iv, c->rows, c->cols, p.tall, mu,
                       (const double*)(ws + p.off_part), p.n_part, (double)c->eps, (_Float16*)(ws + p.off_x), (_Float16*)(ws + p.off_xt[0]), p.mp, p.np,
                       (Scalars*)(ws + p.off_sc));
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}

template <int P>
int iterate(const dsvc_ortho_cfg* c, const Plan& p, void* out, View ov, const MuonArgs& mu, char* ws, hipStream_t st) {
    const long long xs = (long long)p.mp * p.np * P, as = (long long)p.mp * p.mp * P;
    _Float16 *x = (_Float16*)(ws + p.off_x), *a = (_Float16*)(ws + p.off_a), *m = (_Float16*)(ws + p.off_m);
    for (int k = 0; k < c->steps; ++k) {
        _Float16 *xt = (_Float16*)(ws + p.off_xt[k & 1]), *xt1 = (_Float16*)(ws + p.off_xt[(k + 1) & 1]);
        NsGemm g{};
        g.part = (float*)(ws + p.off_split); g.count = (int*)(ws + p.off_count); g.sc = (const Scalars*)(ws + p.off_sc); g.step = k; g.dec = p.dec;
        g.a = g.b = x; g.a_bs = g.b_bs = xs; g.nk16 = p.np / 16;
        g.ot = a; g.ot_bs = as; g.ot_nk16 = p.mp / 16;
        g.c2 = A_SCALE / (X_SCALE * X_SCALE);
        DSVC_TRY((gemm<P, GRAM>(g, p.gram, st)));
        g.a = g.b = a; g.a_bs = g.b_bs = as; g.nk16 = p.mp / 16;
        g.ot = m; g.am = a;
        g.c0 = c->coef[0] * A_SCALE; g.c1 = c->coef[1]; g.c2 = c->coef[2] / A_SCALE;
        DSVC_TRY((gemm<P, POLY>(g, p.poly, st)));
        g.a = m; g.b = xt; g.b_bs = xs;
        g.o = x; g.o_bs = xs; g.o_nk16 = p.np / 16;
        g.ot = xt1; g.ot_bs = xs;
        g.c2 = 1.f / A_SCALE;
        if (k + 1 < c->steps) { DSVC_TRY((gemm<P, FULL>(g, p.full, st))); continue; }
        g.c2 = c->scale / (A_SCALE * X_SCALE);
        g.fin = output(c, p, out, ov, mu);
        DSVC_TRY((gemm<P, FINAL>(g, p.full, st)));
    }
    return DSVC_OK;
}

// the whole operator on the workspace's plan
template <int T, bool MUON, int P>
int run_t(const dsvc_ortho_cfg* c, const Plan& p, const void* in, View iv, void* out, View ov, const MuonArgs& mu, char* ws, hipStream_t st) {
    if (p.one) return one<T, MUON, P>(c, p, in, iv, out, ov, mu, ws, st);
    DSVC_TRY((prep<T, MUON, P>(c, p, in, iv, mu, ws, st)));
    return iterate<P>(c, p, out, ov, mu, ws, st);
}
template <bool MUON>
int run(const dsvc_ortho_cfg* c, const Plan& p, const void* in, View iv, void* out, View ov, const MuonArgs& mu, char* ws, hipStream_t st) {
    if (c->dtype == F32) return p.P == 2 ? run_t<F32, MUON, 2>(c, p, in, iv, out, ov, mu, ws, st) : run_t<F32, MUON, 1>(c, p, in, iv, out, ov, mu, ws, st);
    if (c->dtype == F16) return p.P == 2 ? run_t<F16, MUON, 2>(c, p, in, iv, out, ov, mu, ws, st) : run_t<F16, MUON, 1>(c, p, in, iv, out, ov, mu, ws, st);
    return p.P == 2 ? run_t<BF16, MUON, 2>(c, p, in, iv, out, ov, mu, ws, st) : run_t<BF16, MUON, 1>(c, p, in, iv, out, ov, mu, ws, st);
}

int check_view(const char* what, int64_t ld, int64_t bs, int rows, int cols, int batch, bool written) {
    if (ld < cols && rows > 1) return fail(DSVC_EINVAL, "orthogonalize: %s: row stride %lld < %d columns", what, (long long)ld, cols);
    if (ld < 0 || bs < 0) return fail(DSVC_EINVAL, "orthogonalize: %s: negative stride", what);
    if (written && batch > 1 && bs < (int64_t)(rows - 1) * ld + cols) return fail(DSVC_EINVAL, "orthogonalize: %s: matrices overlap (stride %lld)", what, (long long)bs);
    return DSVC_OK;
}

}  // namespace

extern "C" {

int dsvc_ortho_workspace(const dsvc_ortho_cfg* c, int64_t* bytes) {
    if (!bytes) return fail(DSVC_EINVAL, "null argument");
    Plan p;
    DSVC_TRY(make_plan(c, &p));
    *bytes = p.bytes;
    return DSVC_OK;
}

int dsvc_orthogonalize(const dsvc_ortho_cfg* c, const void* in, int64_t in_ld, int64_t in_bs, void* out, int64_t out_ld, int64_t out_bs, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    Plan p;
    DSVC_TRY(make_plan(c, &p));
    if (!c->batch || !p.m) return DSVC_OK;
    if (!in || !out || !workspace) return fail(DSVC_EINVAL, "null argument");
    if (workspace_bytes < p.bytes || (uintptr_t)workspace % 256) return fail(DSVC_EINVAL, "orthogonalize: workspace of %lld bytes at %p, need %lld on 256", (long long)workspace_bytes, workspace, p.bytes);
    DSVC_TRY(check_view("input", in_ld, in_bs, c->rows, c->cols, c->batch, false));
    DSVC_TRY(check_view("output", out_ld, out_bs, c->rows, c->cols, c->batch, true));
    return run<false>(c, p, in, View{in_ld, in_bs}, out, View{out_ld, out_bs}, MuonArgs{}, (char*)workspace, (hipStream_t)stream);
}

int dsvc_muon_step(const dsvc_ortho_cfg* c, void* param, int64_t param_ld, int64_t param_bs, const void* grad, int64_t grad_ld, int64_t grad_bs, float* momentum,
                   int64_t mom_ld, int64_t mom_bs, float lr, float mu, int32_t nesterov, float weight_decay, const float* grad_scale_dev, float grad_scale,
                   void* workspace, int64_t workspace_bytes, void* stream) {
    Plan p;
    DSVC_TRY(make_plan(c, &p));
    if (!isfinite(lr) || !isfinite(weight_decay) || !(mu >= 0.f && mu < 1.f)) return fail(DSVC_EINVAL, "muon_step: lr %g, weight decay %g, momentum %g", lr, weight_decay, mu);
    if (!c->batch || !p.m) return DSVC_OK;
    if (!param || !grad || !momentum || !workspace) return fail(DSVC_EINVAL, "null argument");
    if (workspace_bytes < p.bytes || (uintptr_t)workspace % 256) return fail(DSVC_EINVAL, "muon_step: workspace of %lld bytes at %p, need %lld on 256", (long long)workspace_bytes, workspace, p.bytes);
    DSVC_TRY(check_view("parameter", param_ld, param_bs, c->rows, c->cols, c->batch, true));
    DSVC_TRY(check_view("gradient", grad_ld, grad_bs, c->rows, c->cols, c->batch, false));
    DSVC_TRY(check_view("momentum", mom_ld, mom_bs, c->rows, c->cols, c->batch, true));
    const MuonArgs u{momentum, View{mom_ld, mom_bs}, mu, lr, weight_decay, nesterov, grad_scale_dev, grad_scale};
    return run<true>(c, p, grad, View{grad_ld, grad_bs}, param, View{param_ld, param_bs}, u, (char*)workspace, (hipStream_t)stream);
}

}  // extern "C"
