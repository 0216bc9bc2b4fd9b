// Token embedding with scaling and its gradient by sorted tokens (include/dsvc.h: dsvc_embed_tokens, dsvc_embed_tokens_grad).
//
//   y[i, :]  = scale * W[t_i, :]
//   dW[v, :] (+)= scale * sum over the places i with t_i = v of dy[i, :]          (nothing for v = padding_idx)
//
// Both are bound by memory: the lookup reads a row and writes a row per token, the gradient reads N rows and writes V.  Adding dy rows to
// dW with atomics would read and write a table row per token and give another sum in every run; sorted, every row of dW is written once and
// the sums have a fixed order:
//   1. stable radix sort of (token, place); tokens outside [0, V) and padding_idx get the key V and end up behind all others
//   2. the sorted places are cut into chunks of equal length, whatever the tokens are; a wave adds one chunk's rows (a slice of 64 lanes' columns) in
//      fp32 and writes the rows of dW whose places all lie in its chunk.  What a chunk boundary cuts goes to a partial row.  Waves of the same
//      launch zero the rows of dW that have no place
//   3. a run that spans chunks is closed by the chunk in which it starts: partial rows in chunk order, a fixed tree over four waves
// A token that fills the batch costs what a batch of different tokens costs.
#include <math.h>

#include "../../include/dsvc.h"
#include "common.h"

using namespace dsvc;

namespace {

enum { F32 = DSVC_DTYPE_F32, F16 = DSVC_DTYPE_F16, BF16 = DSVC_DTYPE_BF16 };
template <int T> struct Elem;
template <> struct Elem<F32> { typedef float type; };
template <> struct Elem<F16> { typedef _Float16 type; };
template <> struct Elem<BF16> { typedef __bf16 type; };

template <class E, int N> struct Vec { typedef E type __attribute__((ext_vector_type(N))); };

__device__ __forceinline__ long long token_at(const void* __restrict__ t, int i64, long long i) {
    return i64 ? ((const long long*)t)[i] : (long long)((const int*)t)[i];
}

// ---- lookup: tx threads along a row, 256 / tx rows per pass of a block -----------------------------------------------------------------------
template <int T, int VEC>
__global__ __launch_bounds__(256) void k_embed(const void* __restrict__ tokens, int i64, long long n, const void* __restrict__ table, long long table_ld, long long V, int H,
                                               float scale, void* __restrict__ out, long long out_ld, int tx_log2, int* __restrict__ flag) {
    typedef typename Elem<T>::type E;
    typedef typename Vec<E, VEC>::type EV;
    const int tx = 1 << tx_log2, x = threadIdx.x & (tx - 1), ty = 256 >> tx_log2, y = threadIdx.x >> tx_log2;
    const E* w = (const E*)table;
    E* o = (E*)out;
    constexpr int R = 4;                     // rows in flight per thread
    for (long long i0 = (long long)blockIdx.x * ty * R; i0 < n; i0 += (long long)gridDim.x * ty * R) {
        long long t[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long long i = i0 + r * ty + y;
            t[r] = i < n ? token_at(tokens, i64, i) : -1;
            if (i < n && (t[r] < 0 || t[r] >= V)) {
                if (flag && x == 0) *flag = 1;
                t[r] = -1;
            }
        }
        for (int c = x * VEC; c < H; c += tx * VEC) {
            EV v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (t[r] >= 0) v[r] = *(const EV*)(w + t[r] * table_ld + c);
                else
                    for (int e = 0; e < VEC; ++e) v[r][e] = (E)0.f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const long long i = i0 + r * ty + y;
                if (i >= n) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[r][e] = (E)((float)v[r][e] * scale);
                *(EV*)(o + i * out_ld + c) = v[r];
            }
        }
    }
}

// ---- 1. stable radix sort, 8 bits a pass ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned key_of(long long t, long long V, long long pad) { return t < 0 || t >= V || t == pad ? (unsigned)V : (unsigned)t; }

// rank of every lane's digit among the equal digits of the wave's earlier items; cnt = this wave's 256 running counts
__device__ __forceinline__ int wave_rank(int d, int lane, volatile int* cnt) {
    unsigned long long same = ~0ull;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const unsigned long long set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
    }
    const int before = cnt[d], below = __popcll(same & ((1ull << lane) - 1));
    __builtin_amdgcn_wave_barrier();
    if (below == 0) cnt[d] = before + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    return before + below;
}

// NW waves' counts -> first slot of every (wave, digit): exclusive over digits, then over waves.  256 or more threads; tot: 256 ints
template <int NW>
__device__ __forceinline__ void scan_counts(int (*cnt)[256], int* tot) {
    const int t = threadIdx.x;
    int run = 0;
    if (t < 256) {
#pragma unroll
        for (int w = 0; w < NW; ++w) { const int c = cnt[w][t]; cnt[w][t] = run; run += c; }
        tot[t] = run;
    }
    __syncthreads();
    for (int k = 1; k < 256; k <<= 1) {
        const int v = t < 256 && t >= k ? tot[t - k] : 0;
        __syncthreads();
        if (t < 256) tot[t] += v;
        __syncthreads();
    }
    if (t < 256) {
        const int first = tot[t] - run;
#pragma unroll
        for (int w = 0; w < NW; ++w) cnt[w][t] += first;
    }
    __syncthreads();
}

// up to 1024 IPT tokens in one workgroup: items stay in registers, each pass exchanges them through LDS
template <int IPT>
__global__ __launch_bounds__(1024) void k_sort_one(const void* __restrict__ tokens, int i64, int n, long long V, long long pad, int passes, unsigned* __restrict__ keys,
                                                   int* __restrict__ order) {
    extern __shared__ int sm[];
    int(*cnt)[256] = (int(*)[256])sm;
    int* tot = sm + 16 * 256;
    unsigned* skey = (unsigned*)(tot + 256);
    int* sidx = (int*)(skey + 1024 * IPT);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, first = wave * 64 * IPT + lane;
    unsigned key[IPT];
    int idx[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
        idx[i] = first + i * 64;
        key[i] = idx[i] < n ? key_of(token_at(tokens, i64, idx[i]), V, pad) : (unsigned)V;       // (items behind the end stay behind all others: stable)
    }
    for (int p = 0; p < passes; ++p) {
        for (int i = threadIdx.x; i < 16 * 256; i += 1024) sm[i] = 0;
        __syncthreads();
        int rank[IPT];
#pragma unroll
        for (int i = 0; i < IPT; ++i) rank[i] = wave_rank((key[i] >> (8 * p)) & 255, lane, cnt[wave]);
        __syncthreads();
        scan_counts<16>(cnt, tot);
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
            const int at = cnt[wave][(key[i] >> (8 * p)) & 255] + rank[i];
            skey[at] = key[i];
            sidx[at] = idx[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
            key[i] = skey[first + i * 64];
            idx[i] = sidx[first + i * 64];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < IPT; ++i)
        if (first + i * 64 < n) {
            keys[first + i * 64] = key[i];
            order[first + i * 64] = idx[i];
        }
}

// more tokens: blocks of 4096.  hist[digit][block]; src_keys == nullptr: the first pass, from the tokens themselves
constexpr int SORT_BLOCK = 4096;
struct SortSrc { const void* tokens; int i64; long long V, pad; const unsigned* keys; const int* order; };
__device__ __forceinline__ void sort_load(const SortSrc& s, long long i, long long n, unsigned& key, int& idx) {
    if (i >= n) { key = ~0u; idx = 0; return; }
    key = s.keys ? s.keys[i] : key_of(token_at(s.tokens, s.i64, i), s.V, s.pad);
    idx = s.keys ? s.order[i] : (int)i;
}
__global__ __launch_bounds__(256) void k_sort_hist(SortSrc s, long long n, int shift, int* __restrict__ hist) {
    __shared__ int cnt[256];
    cnt[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < SORT_BLOCK / 256; ++i) {
        const long long at = (long long)blockIdx.x * SORT_BLOCK + i * 256 + threadIdx.x;
        unsigned key; int idx;
        sort_load(s, at, n, key, idx);
        if (at < n) atomicAdd(&cnt[(key >> shift) & 255], 1);
    }
    __syncthreads();
    hist[(long long)threadIdx.x * gridDim.x + blockIdx.x] = cnt[threadIdx.x];
}
__global__ __launch_bounds__(1024) void k_sort_scan(int* __restrict__ hist, int n) {      // exclusive scan in place
    __shared__ int wsum[16];
    __shared__ int carry;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (t == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < n; base += 8192) {
        int v[8], sum = 0;
        const int at = base + t * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = at + i < n ? hist[at + i] : 0; sum += v[i]; }
        int inc = sum;
        for (int k = 1; k < 64; k <<= 1) { const int o = __shfl_up(inc, k); if (lane >= k) inc += o; }
        if (lane == 63) wsum[wave] = inc;
        __syncthreads();
        int run = carry + inc - sum;
        for (int w = 0; w < wave; ++w) run += wsum[w];
        __syncthreads();
        if (t == 1023) carry = run + sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) { if (at + i < n) hist[at + i] = run; run += v[i]; }
        __syncthreads();
    }
}
__global__ __launch_bounds__(256) void k_sort_scatter(SortSrc s, long long n, int shift, const int* __restrict__ hist, unsigned* __restrict__ keys, int* __restrict__ order) {
    __shared__ int cnt[4][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int w = 0; w < 4; ++w) cnt[w][threadIdx.x] = 0;
    __syncthreads();
    constexpr int IPT = SORT_BLOCK / 256;
    const long long first = (long long)blockIdx.x * SORT_BLOCK + wave * 64 * IPT + lane;
    unsigned key[IPT];
    int idx[IPT], rank[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) sort_load(s, first + i * 64, n, key[i], idx[i]);
#pragma unroll
    for (int i = 0; i < IPT; ++i) rank[i] = wave_rank((key[i] >> shift) & 255, lane, cnt[wave]);
    __syncthreads();
    // this block's slots of a digit start at hist[digit][block]; the waves' shares follow one another.  Items behind the end have the highest
    // digit and come last in the last block: they take no slot of another's
    int run = hist[(long long)threadIdx.x * gridDim.x + blockIdx.x];
    for (int w = 0; w < 4; ++w) { const int c = cnt[w][threadIdx.x]; cnt[w][threadIdx.x] = run; run += c; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPT; ++i)
        if (first + i * 64 < n) {
            const int at = cnt[wave][(key[i] >> shift) & 255] + rank[i];
            keys[at] = key[i];
            order[at] = idx[i];
        }
}

// ---- 2. chunks of sorted places --------------------------------------------------------------------------------------------------------------
constexpr int ZERO_ROWS = 16;                // rows of dW that one wave looks up and zeroes

struct SegArgs {
    const unsigned* keys; const int* order;
    long long n;
    unsigned V;
    int H, chunk, slices;                    // chunk <= 64 places; a slice = 64 lanes' columns
    long long n_chunks;
    const void* dy; long long dy_ld;
    void* dw; long long dw_ld;
    float* part;                             // [chunk][2][H]: 0 = the run that came from the chunk before, 1 = the run that goes on into the next
    float scale;
    int accumulate;
};

// VECTOR: lane = VEC neighbouring columns in one load (rows aligned for it); else VEC columns 64 apart
template <class E, int VEC, bool VECTOR>
__device__ __forceinline__ void load_row(const E* __restrict__ p, int c0, int H, float (&v)[VEC]) {
    if constexpr (VECTOR) {
        typedef typename Vec<E, VEC>::type EV;
        if (c0 < H) {
            const EV x = *(const EV*)(p + c0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = (float)x[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = 0.f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = c0 + 64 * e < H ? (float)p[c0 + 64 * e] : 0.f;
    }
}
template <class E, int VEC, bool VECTOR>
__device__ __forceinline__ void store_row(E* __restrict__ p, int c0, int H, const float (&v)[VEC]) {
    if constexpr (VECTOR) {
        typedef typename Vec<E, VEC>::type EV;
        if (c0 < H) {
            EV x;
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = (E)v[e];
            *(EV*)(p + c0) = x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c0 + 64 * e < H) p[c0 + 64 * e] = (E)v[e];
    }
}
template <class E, int VEC, bool VECTOR>
__device__ __forceinline__ void write_dw(const SegArgs& a, unsigned key, int c0, float (&v)[VEC]) {
    E* p = (E*)a.dw + (long long)key * a.dw_ld;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] *= a.scale;
    if (a.accumulate) {
        float w[VEC];
        load_row<E, VEC, VECTOR>(p, c0, a.H, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += w[e];
    }
    store_row<E, VEC, VECTOR>(p, c0, a.H, v);
}

template <int TD, int TO, int VEC, bool VECTOR>
__global__ __launch_bounds__(256) void k_seg_sum(const SegArgs a) {
    typedef typename Elem<TD>::type D;
    typedef typename Elem<TO>::type O;
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_seg = a.n_chunks * a.slices;
    if (unit >= n_seg) {                     // zero the rows that no place belongs to
        const long long v0 = (unit - n_seg) * ZERO_ROWS;
        if (a.accumulate || v0 >= a.V) return;
        bool absent = false;
        if (lane < ZERO_ROWS && v0 + lane < a.V) {
            const unsigned v = (unsigned)(v0 + lane);
            long long lo = 0, hi = a.n;      // first place whose key is not below v
            while (lo < hi) {
                const long long mid = (lo + hi) >> 1;
                if (a.keys[mid] < v) lo = mid + 1; else hi = mid;
            }
            absent = lo >= a.n || a.keys[lo] != v;
        }
        unsigned long long todo = __ballot(absent);
        float zero[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
        while (todo) {
            const int r = __ffsll((long long)todo) - 1;
            todo &= todo - 1;
            O* p = (O*)a.dw + (v0 + r) * a.dw_ld;
            for (int s = 0; s < a.slices; ++s) store_row<O, VEC, VECTOR>(p, s * 64 * VEC + (VECTOR ? lane * VEC : lane), a.H, zero);
        }
        return;
    }
    const long long c = unit / a.slices, r0 = c * a.chunk;
    const int slice = (int)(unit - c * a.slices), c0 = slice * 64 * VEC + (VECTOR ? lane * VEC : lane);
    const int rows = (int)(a.n - r0 < a.chunk ? a.n - r0 : a.chunk);
    const unsigned kk = lane < rows ? a.keys[r0 + lane] : a.V;
    const int oo = lane < rows ? a.order[r0 + lane] : 0;
    const unsigned none = ~0u;
    const unsigned prev = r0 > 0 ? a.keys[r0 - 1] : none, next = r0 + rows < a.n ? a.keys[r0 + rows] : none;
    const D* dy = (const D*)a.dy;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    unsigned cur = (unsigned)__builtin_amdgcn_readfirstlane((int)kk);
    if (cur == a.V) return;                  // everything from here on is ignored
    bool from_prev = prev == cur;
    constexpr int R = 8;                     // rows in flight
    for (int i0 = 0; i0 < rows; i0 += R) {
        float v[R][VEC];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = i0 + r < rows ? i0 + r : rows - 1;
            load_row<D, VEC, VECTOR>(dy + (long long)__builtin_amdgcn_readlane(oo, i) * a.dy_ld, c0, a.H, v[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (i0 + r >= rows) break;
            const unsigned k = (unsigned)__builtin_amdgcn_readlane((int)kk, i0 + r);
            if (k != cur) {                  // the run of `cur` ends here
                if (from_prev) {
                    if (c0 < a.H) store_row<float, VEC, VECTOR>(a.part + (c * 2) * a.H, c0, a.H, acc);
                } else write_dw<O, VEC, VECTOR>(a, cur, c0, acc);
                from_prev = false;
                cur = k;
                if (cur == a.V) return;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[r][e];
        }
    }
    if (from_prev || next == cur) store_row<float, VEC, VECTOR>(a.part + (c * 2 + (from_prev ? 0 : 1)) * a.H, c0, a.H, acc);
    else write_dw<O, VEC, VECTOR>(a, cur, c0, acc);
}

// ---- 3. runs that span chunks: grid (chunks, slices), four waves -----------------------------------------------------------------------------
template <int TO, int VEC, bool VECTOR>
__global__ __launch_bounds__(256) void k_seg_join(const SegArgs a) {
    typedef typename Elem<TO>::type O;
    const long long c = blockIdx.x, r0 = c * a.chunk, r1 = r0 + a.chunk;
    if (r1 >= a.n) return;                   // the last chunk hands nothing on
    const unsigned key = a.keys[r1 - 1];
    if (key == a.V || a.keys[r1] != key || (r0 > 0 && a.keys[r0 - 1] == key)) return;      // no run starts here and goes on
    long long lo = r1, hi = a.n;             // first place behind the run
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (a.keys[mid] <= key) lo = mid + 1; else hi = mid;
    }
    const long long last = (lo - 1) / a.chunk, terms = last - c + 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.y * 64 * VEC + (VECTOR ? lane * VEC : lane);
    const long long per = (terms + 3) / 4, t0 = wave * per, t1 = t0 + per < terms ? t0 + per : terms;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (long long t = t0; t < t1; ++t) {
        float v[VEC];
        load_row<float, VEC, VECTOR>(a.part + ((c + t) * 2 + (t == 0 ? 1 : 0)) * a.H, c0, a.H, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[e];
    }
    __shared__ float red[4][VEC][64];
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = (red[0][e][lane] + red[1][e][lane]) + (red[2][e][lane] + red[3][e][lane]);
    write_dw<O, VEC, VECTOR>(a, key, c0, acc);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------
inline int size_of(int dtype) { return dtype == F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == F32 || dtype == F16 || dtype == BF16; }

struct GradPlan {
    int passes, one, ipt, chunk;
    long long n_chunks, blocks, off_k[2], off_o[2], off_hist, off_part, bytes;
};

int grad_plan(int64_t n, int64_t V, int32_t H, GradPlan* p) {
    if (n < 0 || n > (1LL << 28)) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld tokens", (long long)n);
    if (V < 1 || V > (1LL << 30)) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld rows", (long long)V);
    if (H < 1 || H > (1 << 20)) return fail(DSVC_EINVAL, "embed_tokens_grad: %d columns", H);
    *p = GradPlan{};
    int bits = 1;
    while ((V >> bits) != 0) ++bits;         // keys 0 ... V
    p->passes = (bits + 7) / 8;
    p->one = n <= 16384;
    p->ipt = n <= 1024 ? 1 : n <= 2048 ? 2 : n <= 4096 ? 4 : n <= 8192 ? 8 : 16;
    p->chunk = 32;
    p->n_chunks = (n + p->chunk - 1) / p->chunk;
    p->blocks = (n + SORT_BLOCK - 1) / SORT_BLOCK;
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 255) / 256 * 256; return o; };
    for (int i = 0; i < (p->one ? 1 : 2); ++i) { p->off_k[i] = take(n * 4); p->off_o[i] = take(n * 4); }
    if (!p->one) p->off_hist = take(256 * p->blocks * 4);
    p->off_part = take(p->n_chunks * 2 * H * 4);
    p->bytes = at < 256 ? 256 : at;
    return DSVC_OK;
}

template <int IPT>
int sort_one(const void* tokens, int i64, int n, long long V, long long pad, int passes, unsigned* keys, int* order, hipStream_t st) {
    constexpr int LDS = (16 * 256 + 256 + 2 * 1024 * IPT) * 4;
    if (LDS > 64 * 1024) DSVC_HIP(hipFuncSetAttribute((const void*)k_sort_one<IPT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    hipLaunchKernelGGL(k_sort_one<IPT>, dim3(1), dim3(1024), LDS, st, tokens, i64, n, V, pad, passes, keys, order);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}

template <int TD, int TO, int VEC, bool VECTOR>
int segments(SegArgs a, hipStream_t st) {
    a.slices = ceil_div(a.H, 64 * VEC);
    const long long zero = a.accumulate ? 0 : ((long long)a.V + ZERO_ROWS - 1) / ZERO_ROWS, units = a.n_chunks * a.slices + zero;
    if (units >= (1LL << 26)) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld work items", units);
    if (units) hipLaunchKernelGGL((k_seg_sum<TD, TO, VEC, VECTOR>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a);
    if (a.n_chunks > 1) hipLaunchKernelGGL((k_seg_join<TO, VEC, VECTOR>), dim3((unsigned)(a.n_chunks - 1), a.slices), dim3(256), 0, st, a);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}

template <int T, int VEC>
int lookup(const void* tokens, int i64, long long n, const void* table, long long ld, long long V, int H, float scale, void* out, long long out_ld, int* flag, hipStream_t st) {
    int lg = 0;
    while (lg < 8 && (1 << lg) * VEC < H) ++lg;
    const long long rows = (256 >> lg) * 4, want = (n + rows - 1) / rows;
    hipLaunchKernelGGL((k_embed<T, VEC>), dim3((unsigned)(want < 16384 ? want : 16384)), dim3(256), 0, st, tokens, i64, n, table, ld, V, H, scale, out, out_ld, lg, flag);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}

bool aligned16(const void* p, long long ld, int esize) { return (uintptr_t)p % 16 == 0 && ld * esize % 16 == 0; }

}  // namespace

extern "C" {

int dsvc_embed_tokens(const void* tokens, int32_t tokens_i64, int64_t n, const void* table, int64_t table_ld, int64_t vocab, int32_t H, int32_t dtype, float scale,
                      void* out, int64_t out_ld, int32_t* out_of_range, void* stream) {
    if (!known(dtype)) return fail(DSVC_EINVAL, "embed_tokens: unknown type %d", dtype);
    if (n < 0 || vocab < 1 || H < 1 || H > (1 << 20)) return fail(DSVC_EINVAL, "embed_tokens: %lld tokens, table [%lld, %d]", (long long)n, (long long)vocab, H);
    if ((table_ld < H && vocab > 1) || (out_ld < H && n > 1)) return fail(DSVC_EINVAL, "embed_tokens: row strides %lld, %lld of %d columns", (long long)table_ld, (long long)out_ld, H);
    if (!isfinite(scale)) return fail(DSVC_EINVAL, "embed_tokens: scale %g", scale);
    if (n == 0) return DSVC_OK;
    if (!tokens || !table || !out) return fail(DSVC_EINVAL, "null argument");
    hipStream_t st = (hipStream_t)stream;
    const int i64 = tokens_i64 != 0, es = size_of(dtype);
    const bool vec = H * es % 16 == 0 && aligned16(table, table_ld, es) && aligned16(out, out_ld, es);
    if (dtype == F32) return vec ? lookup<F32, 4>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st)
                                 : lookup<F32, 1>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st);
    if (dtype == F16) return vec ? lookup<F16, 8>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st)
                                 : lookup<F16, 1>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st);
    return vec ? lookup<BF16, 8>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st)
               : lookup<BF16, 1>(tokens, i64, n, table, table_ld, vocab, H, scale, out, out_ld, out_of_range, st);
}

int dsvc_embed_tokens_grad_workspace(int64_t n, int64_t vocab, int32_t H, int64_t* bytes) {
    if (!bytes) return fail(DSVC_EINVAL, "null argument");
    GradPlan p;
    DSVC_TRY(grad_plan(n, vocab, H, &p));
    *bytes = p.bytes;
    return DSVC_OK;
}

int dsvc_embed_tokens_grad(const void* tokens, int32_t tokens_i64, int64_t n, const void* dy, int64_t dy_ld, int32_t dy_dtype, int64_t vocab, int32_t H, float scale,
                           int64_t padding_idx, void* dw, int64_t dw_ld, int32_t dw_dtype, int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
    GradPlan p;
    DSVC_TRY(grad_plan(n, vocab, H, &p));
    if (!known(dy_dtype) || (dw_dtype != dy_dtype && dw_dtype != F32)) return fail(DSVC_EINVAL, "embed_tokens_grad: types %d -> %d", dy_dtype, dw_dtype);
    if ((dy_ld < H && n > 1) || (dw_ld < H && vocab > 1)) return fail(DSVC_EINVAL, "embed_tokens_grad: row strides %lld, %lld of %d columns", (long long)dy_ld, (long long)dw_ld, H);
    if (!isfinite(scale)) return fail(DSVC_EINVAL, "embed_tokens_grad: scale %g", scale);
    if (!dw || !workspace || (n > 0 && (!tokens || !dy))) return fail(DSVC_EINVAL, "null argument");
    if (workspace_bytes < p.bytes || (uintptr_t)workspace % 256) return fail(DSVC_EINVAL, "embed_tokens_grad: workspace of %lld bytes at %p, need %lld on 256", (long long)workspace_bytes, workspace, p.bytes);
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    const int i64 = tokens_i64 != 0;
    unsigned* keys[2] = {(unsigned*)(ws + p.off_k[0]), (unsigned*)(ws + p.off_k[1])};
    int* order[2] = {(int*)(ws + p.off_o[0]), (int*)(ws + p.off_o[1])};
    int at = 0;
    if (n > 0 && p.one) {
        const int m = (int)n;
        if (p.ipt == 1) DSVC_TRY(sort_one<1>(tokens, i64, m, vocab, padding_idx, p.passes, keys[0], order[0], st));
        else if (p.ipt == 2) DSVC_TRY(sort_one<2>(tokens, i64, m, vocab, padding_idx, p.passes, keys[0], order[0], st));
        else if (p.ipt == 4) DSVC_TRY(sort_one<4>(tokens, i64, m, vocab, padding_idx, p.passes, keys[0], order[0], st));
        else if (p.ipt == 8) DSVC_TRY(sort_one<8>(tokens, i64, m, vocab, padding_idx, p.passes, keys[0], order[0], st));
        else DSVC_TRY(sort_one<16>(tokens, i64, m, vocab, padding_idx, p.passes, keys[0], order[0], st));
    } else if (n > 0) {
        int* hist = (int*)(ws + p.off_hist);
        for (int k = 0; k < p.passes; ++k) {
            const SortSrc s{tokens, i64, vocab, padding_idx, k ? keys[(k + 1) & 1] : nullptr, k ? order[(k + 1) & 1] : nullptr};
            at = k & 1;
            hipLaunchKernelGGL(k_sort_hist, dim3((unsigned)p.blocks), dim3(256), 0, st, s, n, 8 * k, hist);
            hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, hist, (int)(256 * p.blocks));
            hipLaunchKernelGGL(k_sort_scatter, dim3((unsigned)p.blocks), dim3(256), 0, st, s, n, 8 * k, hist, keys[at], order[at]);
        }
        DSVC_HIP(hipGetLastError());
    }
    const SegArgs a{keys[at], order[at], n, (unsigned)vocab, H, p.chunk, 0, p.n_chunks, dy, dy_ld, dw, dw_ld, (float*)(ws + p.off_part), scale, accumulate != 0};
    const int ds = size_of(dy_dtype), os = size_of(dw_dtype);
    const bool vec = H % (16 / ds) == 0 && aligned16(dy, dy_ld, ds) && aligned16(dw, dw_ld, os);
    if (dy_dtype == F32) return vec ? segments<F32, F32, 4, true>(a, st) : segments<F32, F32, 4, false>(a, st);
    if (dy_dtype == F16) {
        if (dw_dtype == F16) return vec ? segments<F16, F16, 8, true>(a, st) : segments<F16, F16, 4, false>(a, st);
        return vec ? segments<F16, F32, 8, true>(a, st) : segments<F16, F32, 4, false>(a, st);
    }
    if (dw_dtype == BF16) return vec ? segments<BF16, BF16, 8, true>(a, st) : segments<BF16, BF16, 4, false>(a, st);
    return vec ? segments<BF16, F32, 8, true>(a, st) : segments<BF16, F32, 4, false>(a, st);
}

}  // extern "C"
