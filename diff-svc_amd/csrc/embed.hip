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
//   3. a run that spans chunks is closed by the chunk in which it starts: partial rows in chunk order, shared out to eight waves in fixed pieces
// A token that fills the batch costs what a batch of different tokens costs.
#include <math.h>

#include <type_traits>

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
// Bound by memory, small calls by the launch: 65536 tokens of 2048 bf16 columns 88 us (rows read once each and written: 473 MB, 5.4 TB/s; a large copy
// reaches 4.8), 861 fp32 rows of 256 columns 3.6 us, one token 1.9 us.
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
                for (int e = 0; e < VEC; ++e) v[r][e] = (E)one_value((float)v[r][e] * scale);      // (left alone, fp16 element by element rounds the exact product)
                *(EV*)(o + i * out_ld + c) = v[r];
            }
        }
    }
}

// ---- 1. stable radix sort ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned key_of(long long t, long long V, long long pad) { return t < 0 || t >= V || t == pad ? (unsigned)V : (unsigned)t; }

// rank of every lane's digit among the equal digits of the wave's earlier items; cnt = this wave's running counts
template <class Count>
__device__ __forceinline__ int wave_rank(int d, int bits, int lane, volatile Count* cnt) {
    unsigned long long same = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
    }
    const int before = cnt[d], below = __popcll(same & ((1ull << lane) - 1));
    __builtin_amdgcn_wave_barrier();
    if (below == 0) cnt[d] = (Count)(before + __popcll(same));
    __builtin_amdgcn_wave_barrier();
    return before + below;
}

// exclusive sum over the workgroup's threads (NW waves); tot: NW ints of LDS
template <int NW>
__device__ __forceinline__ int block_scan(int v, int* tot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int o = __shfl_up(inc, k);
        if (lane >= k) inc += o;
    }
    if (lane == 63) tot[wave] = inc;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < NW; ++w) before += w < wave ? tot[w] : 0;
    __syncthreads();
    return before + inc - v;
}

// Up to 8192 tokens in one workgroup and one launch: items stay in registers, each pass exchanges them through LDS.  Digits of up to 10 bits: a table of
// 256 rows and its ignored places (257 keys) is one pass.  Bound by one CU's latencies (8192 places of 257 keys: 17 us in two passes of 8 bits with the
// digits scanned in 16 barriers, 11 us in one pass with shuffles).
constexpr int ONE_MAX = 8192, ONE_BITS = 10;
template <int IPT>
__global__ __launch_bounds__(1024) void k_sort_one(const void* __restrict__ tokens, int i64, int n, long long V, long long pad, int passes, int bits, unsigned* __restrict__ keys,
                                                   int* __restrict__ order) {
    extern __shared__ int sm[];
    unsigned* skey = (unsigned*)sm;
    unsigned short* sidx = (unsigned short*)(skey + 1024 * IPT);
    int* tot = (int*)(sidx + 1024 * IPT);
    unsigned short* cnt = (unsigned short*)(tot + 16);           // [16][1 << bits]
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, first = wave * 64 * IPT + lane, bins = 1 << bits;
    unsigned key[IPT];
    int idx[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
        idx[i] = first + i * 64;
        key[i] = idx[i] < n ? key_of(token_at(tokens, i64, idx[i]), V, pad) : (unsigned)V;       // (items behind the end stay behind all others: stable)
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = bits * p;
        for (int i = threadIdx.x; i < 16 * bins / 2; i += 1024) ((int*)cnt)[i] = 0;
        __syncthreads();
        int rank[IPT];
#pragma unroll
        for (int i = 0; i < IPT; ++i) rank[i] = wave_rank((key[i] >> shift) & (bins - 1), bits, lane, (volatile unsigned short*)(cnt + wave * bins));
        __syncthreads();
        // counts -> first slot of every (wave, digit): over the waves, then over the digits.  (At most 8192 items: slots fit 16 bits.)
        int run = 0, c[16];
        if ((int)threadIdx.x < bins) {
#pragma unroll
            for (int w = 0; w < 16; ++w) { c[w] = cnt[w * bins + threadIdx.x]; run += c[w]; }
        }
        int at = block_scan<16>(run, tot);
        if ((int)threadIdx.x < bins) {
#pragma unroll
            for (int w = 0; w < 16; ++w) { cnt[w * bins + threadIdx.x] = (unsigned short)at; at += c[w]; }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
            const int to = cnt[wave * bins + ((key[i] >> shift) & (bins - 1))] + rank[i];
            skey[to] = key[i];
            sidx[to] = (unsigned short)idx[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
            key[i] = skey[first + i * 64];
            idx[i] = sidx[first + i * 64];
        }
    }
#pragma unroll
    for (int i = 0; i < IPT; ++i)
        if (first + i * 64 < n) {
            keys[first + i * 64] = key[i];
            order[first + i * 64] = idx[i];
        }
}

// More tokens: blocks of 256 IPT, up to 8 bits a pass or 9 (D = 1 or 2 digits to a thread), counts as hist[digit][block].  The first pass reads the tokens
// themselves (keys == nullptr).  Up to 64 blocks a block finds its first slots from the whole table of counts itself (64 D KiB in L2): two launches a pass.  Beyond, the table is
// scanned by a launch of its own.  (Counting a pass's digits while the pass before it scatters saves a launch, but its atomics meet at a skewed
// text's few digits: 32768 places 31 us instead of 7.5 + 4.7.)
constexpr int FEW_BLOCKS = 64;
struct SortSrc { const void* tokens; int i64; long long V, pad; const unsigned* keys; const int* order; };
__device__ __forceinline__ void sort_load(const SortSrc& s, long long i, long long n, unsigned& key, int& idx) {
    if (i >= n) { key = ~0u; idx = 0; return; }
    key = s.keys ? s.keys[i] : key_of(token_at(s.tokens, s.i64, i), s.V, s.pad);
    idx = s.keys ? s.order[i] : (int)i;
}
template <int IPT, int D>
__global__ __launch_bounds__(256) void k_sort_hist(SortSrc s, long long n, int shift, int mask, int* __restrict__ hist, int ld) {
    __shared__ int cnt[256 * D];
#pragma unroll
    for (int d = 0; d < D; ++d) cnt[256 * d + threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
        const long long at = (long long)blockIdx.x * (256 * IPT) + i * 256 + threadIdx.x;
        unsigned key; int idx;
        sort_load(s, at, n, key, idx);
        if (at < n) atomicAdd(&cnt[(key >> shift) & mask], 1);
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < D; ++d) hist[(long long)(256 * d + threadIdx.x) * ld + blockIdx.x] = cnt[256 * d + threadIdx.x];
}
__global__ __launch_bounds__(1024) void k_sort_scan(int* __restrict__ hist, int n) {      // exclusive scan in place
    __shared__ int tot[16];
    __shared__ int carry;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < n; base += 8192) {
        int v[8], sum = 0;
        const int at = base + threadIdx.x * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = at + i < n ? hist[at + i] : 0; sum += v[i]; }
        int run = block_scan<16>(sum, tot) + carry;
        __syncthreads();
        if (threadIdx.x == 1023) carry = run + sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) { if (at + i < n) hist[at + i] = run; run += v[i]; }
        __syncthreads();
    }
}
// FEW: hist holds counts (ld = FEW_BLOCKS); else first slots
template <int IPT, int D, bool FEW>
__global__ __launch_bounds__(256) void k_sort_scatter(SortSrc s, long long n, int shift, int bits, const int* __restrict__ hist, int ld, unsigned* __restrict__ keys,
                                                      int* __restrict__ order) {
    __shared__ int cnt[4][256 * D];
    __shared__ int tot[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, mask = (1 << bits) - 1;
    for (int i = threadIdx.x; i < 4 * 256 * D; i += 256) cnt[0][i] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * (256 * IPT) + wave * 64 * IPT + lane;
    unsigned key[IPT];
    int idx[IPT], rank[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) sort_load(s, first + i * 64, n, key[i], idx[i]);
    int run[D];                              // digits D threadIdx.x + d
    if (FEW) {
        int all[D], sum = 0;
#pragma unroll
        for (int d = 0; d < D; ++d) {
            all[d] = run[d] = 0;
            const int4* h = (const int4*)(hist + (D * threadIdx.x + d) * FEW_BLOCKS);
#pragma unroll
            for (int q = 0; q < FEW_BLOCKS / 4; ++q) {
                const int4 v = h[q];
                const int e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int c = 4 * q + k < (int)gridDim.x ? e[k] : 0;
                    all[d] += c;
                    run[d] += 4 * q + k < (int)blockIdx.x ? c : 0;
                }
            }
            sum += all[d];
        }
        int base = block_scan<4>(sum, tot);
#pragma unroll
        for (int d = 0; d < D; ++d) { run[d] += base; base += all[d]; }
    } else {
#pragma unroll
        for (int d = 0; d < D; ++d) run[d] = hist[(long long)(D * threadIdx.x + d) * ld + blockIdx.x];
    }
#pragma unroll
    for (int i = 0; i < IPT; ++i) rank[i] = wave_rank((key[i] >> shift) & mask, bits, lane, (volatile int*)cnt[wave]);
    __syncthreads();
    // this block's slots of a digit start at `run`; the waves' shares follow one another.  Items behind the end have the highest digit and come
    // last in the last block: they take no slot of another's
#pragma unroll
    for (int d = 0; d < D; ++d)
        for (int w = 0; w < 4; ++w) { const int c = cnt[w][D * threadIdx.x + d]; cnt[w][D * threadIdx.x + d] = run[d]; run[d] += c; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPT; ++i)
        if (first + i * 64 < n) {
            const int at = cnt[wave][(key[i] >> shift) & mask] + rank[i];
            keys[at] = key[i];
            order[at] = idx[i];
        }
}

// ---- 2. chunks of sorted places --------------------------------------------------------------------------------------------------------------
// Bound by memory: 32768 places of 2048 bf16 columns and a table of 50000 rows take 73 us (339 MB, 4.7 TB/s: a large copy's rate).  Eight rows are in
// flight per wave, since a gathered row's latency is all there is to hide.  8192 fp32 rows of 256 columns onto 256 rows: 6 us.
constexpr long long MAX_WAVES = 1 << 25;     // a launch's share of each kind of work: 2^26 waves of 64 are more than a grid may hold
constexpr int ZERO_ROWS = 16, ZERO_SLICES = 4;   // rows of dW that one wave looks up and zeroes, and slices of them (a wave for whole rows: 45 rows of 4245
                                             // columns take 25 us, when two places are all there is to add)

struct SegArgs {
    const unsigned* keys; const int* order;
    long long n;
    unsigned V;
    int H, chunk, slices;                    // places of a chunk; a slice = 64 lanes' columns
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
        if (a.accumulate) return;
        const int groups = (a.slices + ZERO_SLICES - 1) / ZERO_SLICES;
        const long long units = (a.V + ZERO_ROWS - 1ll) / ZERO_ROWS * groups, waves = gridDim.x * 4ll - n_seg;
        for (long long u = unit - n_seg; u < units; u += waves) {        // (once, up to MAX_WAVES of them)
            const long long z = u / groups, v0 = z * ZERO_ROWS;
            const int s0 = (int)(u - z * groups) * ZERO_SLICES, s1 = s0 + ZERO_SLICES < a.slices ? s0 + ZERO_SLICES : a.slices;
            bool absent = false;
            if (lane < ZERO_ROWS && v0 + lane < a.V) {
                const unsigned v = (unsigned)(v0 + lane);
                long long lo = 0, hi = a.n;  // first place whose key is not below v
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
                for (int s = s0; s < s1; ++s) store_row<O, VEC, VECTOR>(p, s * 64 * VEC + (VECTOR ? lane * VEC : lane), a.H, zero);
            }
        }
        return;
    }
    const long long c = unit / a.slices, r0 = c * a.chunk;
    const int slice = (int)(unit - c * a.slices), c0 = slice * 64 * VEC + (VECTOR ? lane * VEC : lane);
    const long long r1 = a.n - r0 < a.chunk ? a.n : r0 + a.chunk;
    const unsigned none = ~0u;
    const unsigned prev = r0 > 0 ? a.keys[r0 - 1] : none, next = r1 < a.n ? a.keys[r1] : none;
    const D* dy = (const D*)a.dy;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    unsigned cur = none;                     // the run that is being added up, and whether it came from the chunk before
    bool from_prev = false;
    constexpr int R = 8;                     // rows in flight
    for (long long base = r0; base < r1; base += 64) {
        const int rows = r1 - base < 64 ? (int)(r1 - base) : 64;
        const unsigned kk = lane < rows ? a.keys[base + lane] : a.V;
        const int oo = lane < rows ? a.order[base + lane] : 0;
        if (base == r0) {
            cur = (unsigned)__builtin_amdgcn_readfirstlane((int)kk);
            if (cur == a.V) return;          // everything from here on is ignored
            from_prev = prev == cur;
        }
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
                if (k != cur) {              // the run of `cur` ends here
                    if (from_prev) store_row<float, VEC, VECTOR>(a.part + (c * 2) * a.H, c0, a.H, acc);
                    else write_dw<O, VEC, VECTOR>(a, cur, c0, acc);
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
    }
    if (from_prev || next == cur) store_row<float, VEC, VECTOR>(a.part + (c * 2 + (from_prev ? 0 : 1)) * a.H, c0, a.H, acc);
    else write_dw<O, VEC, VECTOR>(a, cur, c0, acc);
}

// ---- 3. runs that span chunks: grid (chunks, slices), eight waves.  Most blocks find nothing to close, most runs a few chunks: latency counts, so the
// lanes of a wave look at the first places of 64 chunks at once and only longer runs are searched (8192 places 3.6 us, 32768 of 2048 columns 11 us; 16 waves
// spill) ----
constexpr int JOIN_WAVES = 8;
template <int TO, int VEC, bool VECTOR>
__global__ __launch_bounds__(JOIN_WAVES * 64) void k_seg_join(const SegArgs a) {
    typedef typename Elem<TO>::type O;
    const long long c = blockIdx.x, r0 = c * a.chunk, r1 = r0 + a.chunk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.y * 64 * VEC + (VECTOR ? lane * VEC : lane);
    if (r1 >= a.n) return;                   // the last chunk hands nothing on
    const long long probe = r1 + (long long)lane * a.chunk;
    const unsigned key = a.keys[r1 - 1], before = r0 > 0 ? a.keys[r0 - 1] : ~0u, there = probe < a.n ? a.keys[probe] : ~0u;
    const unsigned long long on = __ballot(there == key);
    if (key == a.V || !(on & 1) || before == key) return;        // no run starts here and goes on
    long long terms;                         // chunks that the run touches
    if (~on) terms = 1 + __ffsll((long long)~on) - 1;
    else {
        long long lo = r1 + 63 * (long long)a.chunk, hi = a.n;   // first place behind the run
        while (lo < hi) {
            const long long mid = (lo + hi) >> 1;
            if (a.keys[mid] <= key) lo = mid + 1; else hi = mid;
        }
        terms = (lo - 1) / a.chunk - c + 1;
    }
    const long long per = (terms + JOIN_WAVES - 1) / JOIN_WAVES, t0 = wave * per, t1 = t0 + per < terms ? t0 + per : terms;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
#pragma unroll (64 / VEC)
    for (long long t = t0; t < t1; ++t) {
        float v[VEC];
        load_row<float, VEC, VECTOR>(a.part + ((c + t) * 2 + (t == 0 ? 1 : 0)) * a.H, c0, a.H, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[e];
    }
    __shared__ float red[JOIN_WAVES][VEC][64];
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < JOIN_WAVES; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += red[w][e][lane];
    write_dw<O, VEC, VECTOR>(a, key, c0, acc);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------
inline int size_of(int dtype) { return dtype == F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == F32 || dtype == F16 || dtype == BF16; }

struct GradPlan {
    int passes, bits, one, ipt, digits, chunk;    // digits: 256 of them, or 512
    long long n_chunks, blocks, off_k[2], off_o[2], off_hist, off_part, bytes;
};

int grad_plan(int64_t n, int64_t V, int32_t H, int esize, GradPlan* p) {
    if (n < 0 || n > (1LL << 28)) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld tokens", (long long)n);
    if (V < 1 || V > (1LL << 30)) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld rows", (long long)V);
    if (H < 1 || H > (1 << 20)) return fail(DSVC_EINVAL, "embed_tokens_grad: %d columns", H);
    *p = GradPlan{};
    int bits = 1;
    while ((V >> bits) != 0) ++bits;         // keys 0 ... V
    // one workgroup or two launches a pass, the whole operator on 64 columns: 8192 places of 1000 rows 22 / 29 us, 16384 38 / 31; two passes: 4096 of 5000
    // rows 19 / 28
    p->one = bits <= ONE_BITS ? n <= ONE_MAX : n <= ONE_MAX / 2;
    // digits of 9 bits where they save a pass (114310 places of 83939 rows, 30 columns: 73 -> 67 us, 9000 of 300 rows 28 -> 22)
    const int most = p->one ? ONE_BITS : (bits + 8) / 9 < (bits + 7) / 8 ? 9 : 8;
    p->passes = (bits + most - 1) / most;
    p->bits = (bits + p->passes - 1) / p->passes;
    p->digits = p->bits > 8 ? 512 : 256;
    p->ipt = p->one ? (n <= 1024 ? 1 : n <= 2048 ? 2 : n <= 4096 ? 4 : 8) : (n <= FEW_BLOCKS * 1024 ? 4 : n <= FEW_BLOCKS * 2048 ? 8 : 16);
    // chunks: 16 waves a CU (32768 places of 50000 rows, 2048 bf16 columns 108 us, 8 a CU: 113; a single token's partial rows would have fewer: 100000 of 256
    // fp32 columns 103 us, 80); at least 8 places, 16 from 8192 slices on (8192 places of one token, 256 columns: 30 -> 25 us; 500 places of 64: 10 -> 12)
    const long long slices = (H + 64 * (16 / esize) - 1) / (64 * (16 / esize));
    const long long want = n * slices / 4096;
    p->chunk = (int)(want < 2 ? 8 : want < 16 ? 16 : want > 2048 ? 2048 : (want + 7) / 8 * 8);
    p->n_chunks = (n + p->chunk - 1) / p->chunk;
    if (p->n_chunks * ((H + 255) / 256) > MAX_WAVES) return fail(DSVC_EINVAL, "embed_tokens_grad: %lld tokens of %d columns are too many", (long long)n, H);
    p->blocks = (n + 256 * p->ipt - 1) / (256 * p->ipt);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += (bytes + 255) / 256 * 256; return o; };
    for (int i = 0; i < (p->one ? 1 : 2); ++i) { p->off_k[i] = take(n * 4); p->off_o[i] = take(n * 4); }
    if (!p->one) p->off_hist = take(p->digits * (p->blocks <= FEW_BLOCKS ? FEW_BLOCKS : p->blocks) * 4);
    p->off_part = take(p->n_chunks * 2 * H * 4);
    p->bytes = at < 256 ? 256 : at;
    return DSVC_OK;
}

template <int IPT>
int sort_one(const void* tokens, int i64, int n, long long V, long long pad, const GradPlan& p, unsigned* keys, int* order, hipStream_t st) {
    const int lds = 1024 * IPT * 6 + 64 + 32 * (1 << p.bits);
    if (lds > 64 * 1024) DSVC_HIP(hipFuncSetAttribute((const void*)k_sort_one<IPT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL(k_sort_one<IPT>, dim3(1), dim3(1024), lds, st, tokens, i64, n, V, pad, p.passes, p.bits, keys, order);
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}
// returns through `at` which of the two buffers holds the result
template <int IPT, int D>
int sort_many(const void* tokens, int i64, long long n, long long V, long long pad, const GradPlan& p, int* hist, unsigned* const (&keys)[2], int* const (&order)[2], int* at,
              hipStream_t st) {
    const dim3 grid((unsigned)p.blocks), block(256);
    const bool few = p.blocks <= FEW_BLOCKS;
    const int mask = (1 << p.bits) - 1, ld = few ? FEW_BLOCKS : (int)p.blocks;
    for (int k = 0; k < p.passes; ++k) {
        const SortSrc s{tokens, i64, V, pad, k ? keys[(k + 1) & 1] : nullptr, k ? order[(k + 1) & 1] : nullptr};
        *at = k & 1;
        hipLaunchKernelGGL((k_sort_hist<IPT, D>), grid, block, 0, st, s, n, p.bits * k, mask, hist, ld);
        if (few) hipLaunchKernelGGL((k_sort_scatter<IPT, D, true>), grid, block, 0, st, s, n, p.bits * k, p.bits, hist, ld, keys[*at], order[*at]);
        else {
            hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, hist, (int)(256 * D * p.blocks));
            hipLaunchKernelGGL((k_sort_scatter<IPT, D, false>), grid, block, 0, st, s, n, p.bits * k, p.bits, hist, ld, keys[*at], order[*at]);
        }
    }
    DSVC_HIP(hipGetLastError());
    return DSVC_OK;
}

template <int TD, int TO, int VEC, bool VECTOR>
int segments(SegArgs a, hipStream_t st) {
    a.slices = ceil_div(a.H, 64 * VEC);
    const long long all = a.accumulate ? 0 : (((long long)a.V + ZERO_ROWS - 1) / ZERO_ROWS) * ceil_div(a.slices, ZERO_SLICES), zero = all < MAX_WAVES - 4 ? all : MAX_WAVES - 4;
    const long long units = a.n_chunks * a.slices + zero;        // (at most MAX_WAVES of the first: grad_plan)
    if (units) hipLaunchKernelGGL((k_seg_sum<TD, TO, VEC, VECTOR>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a);
    if (a.n_chunks > 1) hipLaunchKernelGGL((k_seg_join<TO, VEC, VECTOR>), dim3((unsigned)(a.n_chunks - 1), a.slices), dim3(JOIN_WAVES * 64), 0, st, a);
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
    DSVC_TRY(grad_plan(n, vocab, H, 2, &p));                    // (16-bit gradients have the shortest chunks, and so the most partial rows)
    *bytes = p.bytes;
    return DSVC_OK;
}

int dsvc_embed_tokens_grad(const void* tokens, int32_t tokens_i64, int64_t n, const void* dy, int64_t dy_ld, int32_t dy_dtype, int64_t vocab, int32_t H, float scale,
                           int64_t padding_idx, void* dw, int64_t dw_ld, int32_t dw_dtype, int32_t accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
    GradPlan p;
    DSVC_TRY(grad_plan(n, vocab, H, dy_dtype == F32 ? 4 : 2, &p));
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
        if (p.ipt == 1) DSVC_TRY(sort_one<1>(tokens, i64, m, vocab, padding_idx, p, keys[0], order[0], st));
        else if (p.ipt == 2) DSVC_TRY(sort_one<2>(tokens, i64, m, vocab, padding_idx, p, keys[0], order[0], st));
        else if (p.ipt == 4) DSVC_TRY(sort_one<4>(tokens, i64, m, vocab, padding_idx, p, keys[0], order[0], st));
        else DSVC_TRY(sort_one<8>(tokens, i64, m, vocab, padding_idx, p, keys[0], order[0], st));
    } else if (n > 0) {
        int* hist = (int*)(ws + p.off_hist);
        auto sort = [&](auto digits) {
            constexpr int D = decltype(digits)::value;
            if (p.ipt == 4) return sort_many<4, D>(tokens, i64, n, vocab, padding_idx, p, hist, keys, order, &at, st);
            if (p.ipt == 8) return sort_many<8, D>(tokens, i64, n, vocab, padding_idx, p, hist, keys, order, &at, st);
            return sort_many<16, D>(tokens, i64, n, vocab, padding_idx, p, hist, keys, order, &at, st);
        };
        DSVC_TRY(p.digits == 512 ? sort(std::integral_constant<int, 2>{}) : sort(std::integral_constant<int, 1>{}));
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
