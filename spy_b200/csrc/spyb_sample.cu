// The next token of every row of logits: temperature, top-k, top-p and min-p, drawn by a given uniform number.

#include <algorithm>
#include <cmath>

#include <math_constants.h>

#include "spyb_common.cuh"
#include "spyb_internal.h"

namespace spyb {
namespace {

// A cluster of CTAs has a row, each a slice of it in shared memory: the logits are read once, by bulk copies. Which token a number falls on must not depend on how
// sums are rounded, so weights are integers: w = 2^S exp((x - largest) / T), S = 45 for up to 2^17 tokens (62 less the bits of their number for more). Their sums are exact in any
// order, a histogram's too. A weight is off by some 2^-34 of itself, as often up as down, and is cut to whole units, half a unit down on average: a border of N weights' sums
// moves by some 2^-34 / sqrt(N) of the whole and N / 2 units (2^-30 of the largest weight for 2^16 tokens). An exponential to so many bits costs some 35
// instructions, so it is taken where it is needed only:
//   greedy            none
//   top-k             every CTA takes its share of k among its threads' own maxima (a histogram of their distances from its largest); the lowest such
//                     threshold has at least k logits above it. Threads whose maximum reaches it give theirs to the first CTA, which ranks them and does the rest
//   top-p alone       a histogram of all distances (counts) brackets the bin in which top_p is reached (a bin is 0.031 wide, its weights are known to 1.6 %);
//                     one pass of weights gives the sums around the bracket and a second histogram inside it, and the elements of its one bin are sorted
//   draw              one pass of the weights that stayed; the warp on whose stretch the number falls walks it again. Numbers below 2^-20: see SA_FINE
// Candidates that do not fit a list (ties by the thousand, a top_k of thousands) take a binary search over (logit, index): slow, and as right.
// Measured: 192 rows of 128 000 f32 logits (98 MB: 15 us of memory) greedy 36 us, top-k with the other settings 74, temperature alone 97, settings that differ by row
// 133; one row of 32 000 in a row of calls: top-k 9.8, temperature alone 7.5. Two CTAs an SM are all that their slices leave room for, so 192 rows go in five to six waves, and a wave takes as long as a
// row's chain: 5 us until the largest is known to all, 9 more for top-k (thresholds, list, ranks), 28 for top-p alone (two histograms, two passes of
// weights, the list's sort), each of them a few barriers of the cluster of 0.7 us and more.
constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 1024, SA_SUB = SA_THREADS, SA_LIST = 1024, SA_RANKED = 256, SA_MAX_CLUSTER = 8, SA_PIECES = 4;
constexpr int SA_INDEX_BITS = 20;
constexpr size_t SA_MAX_SLICE = 40960;    // logits that a CTA keeps in shared memory; longer slices are read again in every pass

struct SampleParams {
    const void    *logits;
    int64_t        row_stride;
    int            n_vocab, per, frac_bits;     // per: logits of a slice (a multiple of 128); frac_bits: S
    const float   *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t       *ids;
    float         *probs;
    const uint64_t *powers;                     // 2^46 2^-(j / 1024), j = 0 .. 1023, to the nearest
    int           *error_flag;
    uint64_t       wait_limit;
};

__device__ __forceinline__ uint32_t ordered(float x) { const uint32_t b = __float_as_uint(x + 0.f); return b & 0x80000000u ? ~b : b | 0x80000000u; }   // (-0 and 0 are equals)
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t key_of(float x, int i) { return ((uint64_t)ordered(x) << SA_INDEX_BITS) | (uint32_t)((1 << SA_INDEX_BITS) - 1 - i); }   // descending: largest first, ties by index
__device__ __forceinline__ int   index_of(uint64_t key) { return (1 << SA_INDEX_BITS) - 1 - (int)(key & ((1 << SA_INDEX_BITS) - 1)); }
__device__ __forceinline__ float value_of(uint64_t key) { return unordered((uint32_t)(key >> SA_INDEX_BITS)); }
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

__device__ __forceinline__ uint32_t rank_in_cluster() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_ctas() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint64_t cluster_load64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_load32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_add(uint32_t addr, uint32_t n) {
    uint32_t v;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(v) : "r"(addr), "r"(n) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { v += __shfl_xor_sync(0xffffffffu, v, o); }
    return v;
}
__device__ __forceinline__ uint64_t warp_upto64(uint64_t v) {   // inclusive sums over the lanes
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint64_t u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) { v += u; } }
    return v;
}

struct SampleShared {
    uint32_t count[SA_BINS];
    uint32_t limb[3][SA_SUB];                // sums of weights in pieces of 15, 15 and the rest of their bits (up to 2^17 weights a CTA)
    uint64_t compact[SA_LIST], weights[SA_LIST];
    uint64_t list[SA_LIST];                  // the first CTA's: candidates
    uint64_t scan[SA_WARPS];
    uint64_t share[2][SA_MAX_CLUSTER];       // what every CTA of the cluster tells all others
    uint64_t share2[SA_MAX_CLUSTER], told[SA_MAX_CLUSTER];
    uint64_t arrived[SA_PIECES];             // barriers of the slice's pieces
    uint64_t cut, total;
    double   c, edge;                        // of this row: Weight's, found by one thread while the slice comes (64 bits are slow: see Weight)
    uint64_t least;                          // the smallest weight that min_p leaves
    float    bin_scale, unused;
    uint64_t table[1024];                    // Weight's
    uint32_t n_list, n_own;
    int      found, found2;
};

// The weight of a logit as an integer, 2^S 2^-z with z = (largest - x) c, c = log2(e) / T, to 2^-31.8 of itself at most and a unit (see below). (An operation in 64 bits takes eight clocks of a
// quarter of an SM, one in f32 one: 192 rows of 128 000 at a temperature alone took 108 us with them, 100 like this.) z is taken apart as r / 1024 + f + e without an error that counts:
//   p + p' = x c, by FMA; A = largest c in 64 bits, A = a + a' with a a multiple of 2^-14; r = round(1024 (a - p));
//   f = (a - r / 1024) - p: the first difference is exact (multiples of 2^-14 below 2^10), the second too (|f| <= 2^-11); e = a' - p'.
// 2^-(r / 1024) is a table's 2^46-fold and a shift, 2^-(f + e) = 1 + y with |y| < 2^-11.5. Of the weight: y's roundings 2^-34.2 (two steps and a constant, each half a step of
// f32), the table's entry cut to 23 bits in its product with y 2^-33.5, that product rounded to 2^-33 of the largest entry, which is 2^-32 of the smallest, half of it 2^-33; p', a' and the
// series' third term 2^-36 together.
// Where |A| is too large for that (1000 and more: tiny temperatures, huge logits), or c itself for f32, the same in 64 bits.
struct Weight {
    const uint64_t *table;      // 2^46 2^-(j / 1024)
    float  c_hi, c_lo, a_hi, a_lo;
    float  least;               // no logit below it has weight: it stands for them, and for -inf
    bool   wide;                // in 64 bits
    double c, largest;
    int    shift;               // 46 - S
    static __device__ __forceinline__ double factor(float temp) { return 1.4426950408889634073599 / (double)temp; }   // c (4e-39 to 1e45, or 0)
    __device__ __forceinline__ void set(const uint64_t *powers, float top, double scale, double edge, int bits) {   // edge: 56 / c (2^-56 is no unit: rounds to nothing)
        table = powers; c = scale; largest = top; shift = 46 - bits;
        const double a = largest * c, lowest = largest - edge;
        wide = !(fabs(a) < 960.0 && lowest > -3.4e38 && c > 1e-30 && c < 1e30);
        least = wide ? 0.f : (float)lowest;
        c_hi = (float)c; c_lo = (float)(c - c_hi);
        a_hi = (float)(rint(a * 16384.0) * (1.0 / 16384)); a_lo = (float)(a - a_hi);
    }
    static __device__ __noinline__ uint64_t in_64_bits(const uint64_t *table, double z, int shift) {
        z = fmin(z, 56.0);                                                               // (NaN reads as no weight)
        const double r = rint(z * 1024.0), f = (r * (1.0 / 1024) - z) * 0.69314718055994530942;
        const int    k = (int)r;
        const double t = (double)table[k & 1023] * (1.0 + f * (1.0 + f * (0.5 + f * (1.0 / 6))));
        return (uint64_t)(t + 0.5) >> ((k >> 10) + shift);
    }
    template <int N> __device__ __forceinline__ void of(const float (&x)[N], uint64_t (&w)[N]) const {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; ++i) { w[i] = in_64_bits(table, (largest - (double)x[i]) * c, shift); }
            return;
        }
        float p[N], e[N], t[N], f[N], y[N];
        uint64_t full[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float v = fmaxf(x[i], least);                                          // (NaN reads as no weight)
            p[i] = __fmul_rn(v, c_hi);
            e[i] = fmaf(v, c_lo, fmaf(v, c_hi, -p[i]));
            t[i] = __fadd_rn(fmaf(v, -1024.f * c_hi, 1024.f * a_hi), 12582912.f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) { full[i] = table[__float_as_uint(t[i]) & 1023]; }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float r = __fsub_rn(t[i], 12582912.f);
            f[i] = __fadd_rn(__fsub_rn(fmaf(r, -1.f / 1024, a_hi), p[i]), __fsub_rn(a_lo, e[i]));
            y[i] = f[i] * fmaf(f[i], 0.2402265f, -0.69314718f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float whole = __fsub_rn(__uint_as_float((uint32_t)(full[i] >> 23) | 0x4b000000u), 8388608.f);   // 2^23 2^-(j / 1024), cut
            const int   more = (int)(__float_as_uint(__fadd_rn(whole * y[i], 1.5f * 8192)) - 0x46400000u);        // their product in units of 2^-10 (2^-33 of the largest weight)
            w[i] = (full[i] + (int64_t)more * 8192) >> (((__float_as_uint(t[i]) >> 10) & 63) + shift);
        }
    }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const float one[1] = {x};
        uint64_t w[1];
        of(one, w);
        return w[0];
    }
};

// A slice of the row: in shared memory (NaN is -inf there, and where the largest is +inf it is 0 and all else -inf), or read from where it lies
template <class T, bool KEPT> struct Slice {
    const T     *row;       // of the slice's first logit
    const float *kept;
    int          n, base;
    bool         inf;
    __device__ __forceinline__ float operator()(int i) const {
        if (KEPT) { return kept[i]; }
        float x = as_float(row[i]);
        x = x == x ? x : -CUDART_INF_F;
        return inf ? (x == CUDART_INF_F ? 0.f : -CUDART_INF_F) : x;
    }
    // f(four logits, place of the first) for this thread's share; -inf behind the slice's end
    template <class F> __device__ __forceinline__ void fours(const F &f) const { stretch(0, n, threadIdx.x, SA_THREADS, f); }
    template <class F> __device__ __forceinline__ void stretch(int from, int to, int first, int step, const F &f) const {   // from: a multiple of 4
        for (int i = from + 4 * first; i < to; i += 4 * step) {
            float v[4];
            if (KEPT) {
                const float4 u = *reinterpret_cast<const float4 *>(kept + i);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = i + e < n ? (*this)(i + e) : -CUDART_INF_F; }
            }
            f(v, i);
        }
    }
    template <class F> __device__ __forceinline__ void each(const F &f) const {   // f(logit, place)
        fours([&](const float (&v)[4], int i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) { f(v[e], i + e); }
        });
    }
};

// inclusive sums over all threads in their order; *all: of all
__device__ __forceinline__ uint64_t block_upto(uint64_t v, uint64_t *scan, uint64_t *all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t upto = warp_upto64(v);
    __syncthreads();
    if (lane == 31) { scan[warp] = upto; }
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) { const uint64_t u = scan[w]; upto += w < warp ? u : 0; sum += u; }
    *all = sum;
    return upto;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t *scan) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) { scan[threadIdx.x >> 5] = v; }
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) { sum += scan[w]; }
    return sum;
}
// v of every CTA to all of the cluster (thread 0's counts), summed after the barrier
__device__ __forceinline__ uint64_t cluster_total(uint64_t v, uint64_t *slots, uint32_t ctas, uint32_t rank) {
    if (threadIdx.x < ctas) { cluster_store64(cluster_map(smem_u32(slots + rank), threadIdx.x), v); }
    cluster_sync();
    uint64_t sum = 0;
    for (uint32_t i = 0; i < ctas; ++i) { sum += slots[i]; }
    return sum;
}
// a list of up to SA_LIST keys, the largest first
__device__ __noinline__ void sort_list(uint64_t *a, int n) {
    int size = 32;
    while (size < n) { size <<= 1; }
    for (int i = n + threadIdx.x; i < size; i += SA_THREADS) { a[i] = 0; }
    for (int k = 2; k <= size; k <<= 1) {
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += SA_THREADS) {
                const int i = 2 * t - (t & (j - 1)), l = i + j;
                const uint64_t x = a[i], y = a[l];
                if ((x < y) == ((i & k) == 0)) { a[i] = y; a[l] = x; }
            }
        }
    }
    __syncthreads();
}
__device__ __forceinline__ uint64_t of_total(float share, uint64_t total) {   // the sum on which the number falls, below the total
    return min((uint64_t)((double)(share > 0.f ? share : 0.f) * (double)total), total - 1);
}

// Uniform numbers below SA_FINE fall among weights that are no unit, down to what 64 bits hold: at 0 on the first index whose weight is not 0 there. Such rows - one in a
// million of evenly spread numbers - are drawn by weights in floating point of 64 bits. What stays is found as ever, but for min_p, which is asked of these weights. (192 rows of
// 128 000 that are all drawn so, no numbers given: 136 us at a temperature alone, 82 with top-k, against 97 and 74.)
// (A function of its own, and its exponential too: the registers of what runs for all other rows stay theirs.)
constexpr float SA_FINE = 1.f / (1 << 20);
__device__ __noinline__ double fine_weight(float x, float largest, float temp) {
    if (x == -CUDART_INF_F) { return 0.0; }
    const double z = ((double)x - (double)largest) / (double)temp;
    if (z > -700) { return exp(z); }
    const double half = exp(0.5 * z);
    return half * half;                                   // (exp may be off by a step, and 0 in place of the smallest numbers; a product is rounded)
}
__device__ __forceinline__ double fine_upto(double v) {   // inclusive sums over the lanes
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const double u = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) { v += u; } }
    return v;
}
// The list's: weights in the order `by_index`'s entries name them, by one thread
__device__ __noinline__ void fine_draw_list(const SampleParams &p, int row, const uint64_t *by_index, const uint64_t *weights, int n, float uni) {
    double total = 0, upto = 0;
    for (int i = 0; i < n; ++i) { total += __longlong_as_double((long long)weights[(by_index[i] - 1) & 2047]); }
    const double t = (uni > 0.f ? (double)uni : 0.0) * total;
    for (int i = 0; i < n; ++i) {
        const double w = __longlong_as_double((long long)weights[(by_index[i] - 1) & 2047]);
        upto += w;
        if (upto > t || i == n - 1) {
            p.ids[row] = (1 << SA_INDEX_BITS) - 1 - (int)((by_index[i] - 1) >> 11);
            if (p.probs) { p.probs[row] = (float)(w / total); }
            return;
        }
    }
}
// All of the row. Sums of CTAs, of a CTA's warps and of a warp's lanes are not rounded alike: each step takes the first part whose sum passes the number, or the last that has
// any weight.
template <class T, bool KEPT>
__device__ __noinline__ void fine_draw(const SampleParams &p, SampleShared &sh, const Slice<T, KEPT> x, int row, float largest, float temp, float min_p, float uni, float cut_value, int cut_index, uint32_t rank, uint32_t ctas) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int stretch = ((x.n + SA_WARPS - 1) / SA_WARPS + 127) & ~127, from = min(warp * stretch, x.n), to = min(from + stretch, x.n);
    const double least = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0;
    auto weight = [&](int i) {
        const float v = i < to ? x(i) : -CUDART_INF_F;
        if (!(v >= cut_value) || (v == cut_value && x.base + i > cut_index)) { return 0.0; }
        const double w = fine_weight(v, largest, temp);
        return w >= least ? w : 0.0;
    };
    double s = 0;
    for (int i = from + lane; i < to; i += 32) { s += weight(i); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); }
    __syncthreads();
    if (lane == 0) { sh.scan[warp] = (uint64_t)__double_as_longlong(s); }
    __syncthreads();
    double mine = 0;
    for (int w = 0; w < SA_WARPS; ++w) { mine += __longlong_as_double((long long)sh.scan[w]); }
    cluster_sync();                                       // (shares of earlier exchanges are read)
    if (threadIdx.x < ctas) { cluster_store64(cluster_map(smem_u32(sh.share[0] + rank), threadIdx.x), (uint64_t)__double_as_longlong(mine)); }
    cluster_sync();
    double total = 0, before = 0;
    for (uint32_t r = 0; r < ctas; ++r) { total += __longlong_as_double((long long)sh.share[0][r]); }
    const double t = (uni > 0.f ? (double)uni : 0.0) * total;                 // (below the total, which is 1 at least)
    uint32_t at = 0;
    for (;; ++at) {
        const double next = before + __longlong_as_double((long long)sh.share[0][at]);
        if (next > t || at == ctas - 1) { break; }
        before = next;
    }
    if (at != rank) { return; }
    int    who = -1;
    double start = before;
    for (int w = 0; w < SA_WARPS; ++w) {
        const double v = __longlong_as_double((long long)sh.scan[w]);
        if (v > 0) {
            who = w; start = before;
            if (before + v > t) { break; }
        }
        before += v;
    }
    if (who != warp) { return; }
    before = start;
    int    last = -1;
    double last_w = 0;
    for (int i0 = from; i0 < to; i0 += 32) {
        const double   w = weight(i0 + lane), upto = before + fine_upto(w);
        const unsigned any = __ballot_sync(0xffffffffu, w > 0), hit = __ballot_sync(0xffffffffu, w > 0 && upto > t);
        if (any) {
            const int l = hit ? __ffs(hit) - 1 : 31 - __clz(any);
            last = i0 + l;
            last_w = __shfl_sync(0xffffffffu, w, l);
            if (hit) { break; }
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0 && last >= 0) {
        p.ids[row] = x.base + last;
        if (p.probs) { p.probs[row] = (float)(last_w / total); }
    }
}

template <class T, bool KEPT>
__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(const __grid_constant__ SampleParams p) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(dynamic);
    float *slice = reinterpret_cast<float *>(dynamic + sizeof(SampleShared));
    static_assert(sizeof(SampleShared) % 16 == 0, "the slice is read in pieces of 16 bytes");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = rank_in_cluster(), ctas = cluster_ctas();
    const int row = blockIdx.x / ctas;
    pdl_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < SA_PIECES; ++i) { mbar_init(smem_u32(sh.arrived + i), 1); }
        mbar_init_fence();
        sh.n_list = sh.n_own = 0; sh.cut = 0; sh.found = sh.found2 = 0;
    }
    *reinterpret_cast<uint2 *>(sh.count + 2 * tid) = make_uint2(0, 0);
    static_assert(2 * SA_THREADS == 1024, "a thread brings two of the table's powers");
    const uint4 powers = __ldg(reinterpret_cast<const uint4 *>(p.powers) + tid);
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");   // (waited for in front of the first access to another CTA's memory)
    pdl_wait();

    Slice<T, KEPT> x;
    x.base = (int)rank * p.per;
    x.n = max(0, min(p.per, p.n_vocab - x.base));
    x.row = static_cast<const T *>(p.logits) + row * p.row_stride + x.base;
    x.kept = slice;
    x.inf = false;
    // pieces of the slice by bulk copies, from whole 16 bytes on
    const bool bulk = KEPT && sizeof(T) == 4 && (reinterpret_cast<uintptr_t>(x.row) & 15) == 0;
    const int  whole = bulk ? x.n & ~3 : 0, piece = (whole / SA_PIECES + 3) & ~3;
    if (bulk && tid == 0) {
        for (int i = 0; i < SA_PIECES; ++i) {
            const int from = min(i * piece, whole), n = min(piece, whole - from);
            if (n > 0) {
                const uint32_t bar = smem_u32(sh.arrived + i);
                mbar_expect_tx(bar, n * 4);
                bulk_copy_g2s(smem_u32(slice + from), x.row + from, n * 4, bar);
            }
        }
    }
    const float temp = p.temperature ? p.temperature[row] : 1.f, top_p = p.top_p ? p.top_p[row] : 1.f;
    const float min_p = p.min_p ? p.min_p[row] : 0.f, uni = p.uniform ? p.uniform[row] : 0.f;
    const int   top_k = p.top_k ? p.top_k[row] : 0;

    *reinterpret_cast<uint4 *>(sh.table + 2 * tid) = powers;
    if (tid == SA_THREADS - 1) {
        const double c = Weight::factor(temp);
        sh.c = c; sh.edge = 56 / c;
        sh.least = min_p > 0.f ? (uint64_t)max(1.0, ceil((double)fminf(min_p, 1.f) * __hiloint2double((1023 + p.frac_bits) << 20, 0))) : 1;
        sh.bin_scale = (float)fmin(c * (2 * SA_BINS / (double)(p.frac_bits + 1)), 3e38);   // of halves (cut: bins hold more than they should, and the slow search decides)
    }
    // this thread's largest (of the elements that Slice::each gives it), the row's, and where that is
    float own = -CUDART_INF_F, from_here = CUDART_INF_F;      // (top-k: nothing below from_here is among the k largest)
    uint64_t best = 0;
    const bool greedy = !(temp > 0.f), by_k = !greedy && top_k > 0 && top_k < p.n_vocab, by_p = top_p < 1.f;
    const bool quick = by_k && top_k <= 32 * (int)ctas;        // by the threads' maxima first
    const uint64_t need = ctas > 1 ? (top_k + ctas - 2) / (ctas - 1) : top_k;
    {
        int at = -1;                                       // the first of the four that own is in
        auto take4 = [&](float4 v, int i) {
            const float m = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
            if (m > own) { own = m; at = i; }
        };
        if (bulk) {
            __syncthreads();                               // (the barriers are there)
            bool ok = true;
            for (int q = 0; q < SA_PIECES; ++q) {
                const int from = min(q * piece, whole), to = min(from + piece, whole);
                if (from < to) { ok &= mbar_wait_prompt(smem_u32(sh.arrived + q), 0, p.wait_limit); }
                // every thread meets the fours that it meets in the passes to come
                const int first = (from / 4 - tid + SA_THREADS - 1) / SA_THREADS * SA_THREADS + tid;
                for (int i = 4 * max(first, tid); i < to; i += 4 * SA_THREADS) {
                    float4 v = *reinterpret_cast<const float4 *>(slice + i);
                    const float all = (v.x + v.y) + (v.z + v.w);     // (NaN if one of them is)
                    if (!(all == all)) {
                        v = make_float4(v.x == v.x ? v.x : -CUDART_INF_F, v.y == v.y ? v.y : -CUDART_INF_F, v.z == v.z ? v.z : -CUDART_INF_F, v.w == v.w ? v.w : -CUDART_INF_F);
                        *reinterpret_cast<float4 *>(slice + i) = v;
                    }
                    take4(v, i);
                }
            }
            if (!ok) {   // reported; what is on its way lands first, or is given a last chance to
                for (int q = 0; q < SA_PIECES; ++q) { if (min(q * piece, whole) < whole) { mbar_wait_bounded(smem_u32(sh.arrived + q), 0, 1000000000); } }
                if (lane == 0 && p.error_flag != nullptr) { atomicExch(p.error_flag, 1); }
            }
            if (whole < x.n && tid == (whole / 4) % SA_THREADS) {
                float v[4];
                for (int e = 0; e < 4; ++e) { v[e] = whole + e < x.n ? as_float(x.row[whole + e]) : -CUDART_INF_F; v[e] = v[e] == v[e] ? v[e] : -CUDART_INF_F; }
                *reinterpret_cast<float4 *>(slice + whole) = make_float4(v[0], v[1], v[2], v[3]);
                take4(make_float4(v[0], v[1], v[2], v[3]), whole);
            }
        } else if (KEPT) {
#pragma unroll 2
            for (int i = 4 * tid; i < x.n; i += 4 * SA_THREADS) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = i + e < x.n ? as_float(x.row[i + e]) : -CUDART_INF_F; v[e] = v[e] == v[e] ? v[e] : -CUDART_INF_F; }
                *reinterpret_cast<float4 *>(slice + i) = make_float4(v[0], v[1], v[2], v[3]);
                take4(make_float4(v[0], v[1], v[2], v[3]), i);
            }
        } else {
            x.fours([&](const float (&v)[4], int i) { take4(make_float4(v[0], v[1], v[2], v[3]), i); });
        }
        if (at >= 0) {
            at = x(at) == own ? at : x(at + 1) == own ? at + 1 : x(at + 2) == own ? at + 2 : at + 3;
            best = key_of(own, x.base + at);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { best = max(best, __shfl_xor_sync(0xffffffffu, best, o)); }
        if (lane == 0) { sh.scan[warp] = best; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SA_WARPS; ++w) { best = max(best, sh.scan[w]); }
        // this CTA's threshold: its largest minus so many 32nds that `need` of its threads' maxima lie above
        float threshold = -CUDART_INF_F;
        if (quick) {
            const float top = best == 0 ? -CUDART_INF_F : value_of(best), b = (top - own) * 32.f;
            if (b < (float)SA_BINS) { atomicAdd(&sh.count[(int)b], 1u); }
            __syncthreads();
            const uint2 n2 = *reinterpret_cast<const uint2 *>(sh.count + 2 * tid);
            uint64_t all;
            const uint64_t upto = block_upto((uint64_t)n2.x + n2.y, sh.scan, &all), before = upto - n2.x - n2.y;
            if (before < need && need <= upto) { sh.found = 2 * tid + 1; }
            __syncthreads();
            // (a slice's end may lack them: it is left out, and the others' shares suffice)
            threshold = all >= need ? top - (float)(sh.found + 2) * (1.f / 32) : ctas > 1 && rank == ctas - 1 ? CUDART_INF_F : -CUDART_INF_F;
        }
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (tid < (int)ctas) {
            cluster_store64(cluster_map(smem_u32(sh.share[0] + rank), tid), best);
            cluster_store64(cluster_map(smem_u32(sh.share2 + rank), tid), __float_as_uint(threshold));
        }
        cluster_sync();
        for (uint32_t i = 0; i < ctas; ++i) { best = max(best, sh.share[0][i]); from_here = fminf(from_here, __uint_as_float((uint32_t)sh.share2[i])); }
    }
    if (best == 0 || greedy) {
        if (rank == 0 && tid == 0) {
            p.ids[row] = best == 0 ? -1 : index_of(best);
            if (p.probs) { p.probs[row] = best == 0 ? 0.f : 1.f; }
        }
        return;
    }
    float largest = value_of(best);
    if (largest == CUDART_INF_F) {
        x.inf = true; largest = 0.f;
        own = own == CUDART_INF_F ? 0.f : -CUDART_INF_F;
        from_here = 0.f;
        if (KEPT) {
            for (int i = tid; i < ((x.n + 3) & ~3); i += SA_THREADS) { slice[i] = slice[i] == CUDART_INF_F ? 0.f : -CUDART_INF_F; }
            __syncthreads();
        }
    }
    Weight weight;
    weight.set(sh.table, largest, sh.c, sh.edge, p.frac_bits);
    const bool     fine = !(uni >= SA_FINE);
    const uint64_t least = sh.least;
    const float    bin_scale = sh.bin_scale;
    const float half_largest = 0.5f * largest;
    auto bin_of = [&](float v) { return fmaf(v, -0.5f, half_largest) * bin_scale; };   // not below SA_BINS (or NaN): no weight (halves: a difference may leave f32)
    auto reach = [&](uint64_t total) { return max((uint64_t)1, (uint64_t)ceil((double)max(top_p, 0.f) * (double)total)); };   // a token stays while less than this is in front of it
    uint64_t cut = 0;                        // keys from here on stay
    bool     search = false;                 // ... by the slow way

    // the whole row's counts, two bins a thread (all CTAs' in flight together)
    auto counts = [&]() {
        cluster_sync();
        uint64_t v[SA_MAX_CLUSTER];
        uint2 n2 = make_uint2(0, 0);
#pragma unroll
        for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) { v[r] = r < ctas ? cluster_load64(cluster_map(smem_u32(sh.count) + tid * 8, r)) : 0; }
#pragma unroll
        for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) { n2.x += (uint32_t)v[r]; n2.y += (uint32_t)(v[r] >> 32); }
        return n2;
    };
    auto count_all = [&]() {
        x.each([&](float v, int) {
            const float b = bin_of(v);
            if (b < (float)SA_BINS) { atomicAdd(&sh.count[(int)b], 1u); }
        });
    };
    // Elements that `wanted` names, of the threads whose largest is wanted, to the first CTA: how many there are (more than SA_LIST: they do not fit), and where. Every
    // CTA has its part of the list, so that nobody waits for a place in it; the first one closes the gaps
    uint64_t *const compact = sh.compact, *const weights = sh.weights;
    uint64_t *candidates = sh.list;
    auto gather = [&](bool mine, auto wanted) {
        const uint32_t part = SA_LIST / ctas, list = cluster_map(smem_u32(sh.list), 0) + rank * part * 8;
        if (mine) {
            x.each([&](float v, int i) {
                if (!wanted(v)) { return; }
                const uint32_t at = atomicAdd(&sh.n_own, 1u);
                if (at < part) { cluster_store64(list + at * 8, key_of(v, x.base + i)); }
            });
        }
        __syncthreads();
        if (tid < (int)ctas) { cluster_store64(cluster_map(smem_u32(sh.told + rank), tid), sh.n_own); }
        cluster_sync();
        uint32_t n = 0;
        bool fits = true;
        for (uint32_t r = 0; r < ctas; ++r) { const uint32_t c = (uint32_t)sh.told[r]; fits &= c <= part; n += c; }
        if (!fits) { return (uint32_t)SA_LIST + 1; }
        if (rank == 0 && ctas > 1) {
            for (uint32_t e = tid; e < SA_LIST; e += SA_THREADS) {
                const uint32_t r = e / part, o = e - r * part;
                if (o < (uint32_t)sh.told[r]) {
                    uint32_t before = 0;
                    for (uint32_t k = 0; k < r; ++k) { before += (uint32_t)sh.told[k]; }
                    compact[before + o] = sh.list[e];
                }
            }
            candidates = compact;
            __syncthreads();
        }
        return n;
    };
    // the same where places are given out one by one: candidates may all lie in one slice
    auto gather_one_by_one = [&](auto wanted) {
        const uint32_t counter = cluster_map(smem_u32(&sh.n_list), 0), list = cluster_map(smem_u32(sh.list), 0);
        x.each([&](float v, int i) {
            if (!wanted(v)) { return; }
            const uint32_t at = cluster_add(counter, 1);
            if (at < SA_LIST) { cluster_store64(list + at * 8, key_of(v, x.base + i)); }
        });
        cluster_sync();
        const uint32_t n = cluster_load32(counter);
        candidates = sh.list;
        cluster_sync();                                   // (all have read how many there are)
        return n;
    };
    // the sum over all keys from `from` on
    auto sum_from = [&](uint64_t from, bool counting, int turn) {
        uint64_t s = 0;
        x.each([&](float v, int i) {
            if (v != -CUDART_INF_F && key_of(v, x.base + i) >= from) { s += counting ? 1 : weight(v); }
        });
        return cluster_total(block_sum(s, sh.scan), sh.share[turn & 1], ctas, rank);
    };

    if (by_k) {
        uint32_t n = SA_LIST + 1;
        if (quick) { n = gather(own >= from_here, [&](float v) { return v >= from_here; }); }
        if (n > SA_LIST) {                                // from a histogram of all the row
            if (quick) { *reinterpret_cast<uint2 *>(sh.count + 2 * tid) = make_uint2(0, 0); }
            __syncthreads();
            count_all();
            const uint2 n2 = counts();
            uint64_t all;
            const uint64_t upto = block_upto((uint64_t)n2.x + n2.y, sh.scan, &all);
            const uint64_t before = upto - n2.x - n2.y, want = min((uint64_t)top_k, all);
            if (before < want && want <= upto) {
                uint64_t c = before + n2.x; int b = tid * 2;
                if (c < want) { c += n2.y; ++b; }
                sh.found = b; sh.found2 = (int)min(c, (uint64_t)SA_LIST + 1);
            }
            __syncthreads();
            const float behind = (float)(sh.found + 1);
            // (a drawing to the bottom asks for what has no unit, too, and so is in no bin)
            if (sh.found2 <= SA_LIST && !(fine && all < (uint64_t)top_k)) { n = gather_one_by_one([&](float v) { return bin_of(v) < behind; }); }
        }
        if (n <= SA_LIST) {
            if (rank != 0) { return; }
            // everything else is the first CTA's
            const int n_list = (int)n;
            if (n_list <= SA_RANKED && !fine) {
                // few candidates: a group of threads ranks each, by counting and weighing what is in front of it - first in the order of weights, then of indices
                int per = 512 / SA_RANKED;
                while (per < 32 && n_list * per * 2 <= SA_THREADS) { per *= 2; }
                const int i = tid / per, part = tid & (per - 1);
                const bool is = i < n_list;
                const uint64_t key = is ? candidates[i] : 0;
                uint64_t w = 0;
                if (is) { w = weight(value_of(key)); if (part == 0) { weights[i] = w; } }
                __syncthreads();
                auto group_sum = [&](uint64_t v) {
                    for (int o = 1; o < per; o <<= 1) { v += __shfl_xor_sync(0xffffffffu, v, o); }
                    return v;
                };
                uint64_t in_front = 0, before_w = 0;
                if (is) {
                    for (int j = part; j < n_list; j += per) { if (candidates[j] > key) { ++in_front; before_w += weights[j]; } }
                }
                in_front = group_sum(in_front); before_w = group_sum(before_w);
                bool stays = is && in_front < (uint64_t)top_k;
                const uint64_t total_k = block_sum(stays && part == 0 ? w : 0, sh.scan);
                stays = stays && (!by_p || before_w < reach(total_k)) && w >= least;
                if (is && part == 0 && !stays) { weights[i] = 0; }
                const uint64_t sum = block_sum(stays && part == 0 ? w : 0, sh.scan);          // (its barriers are between the writes above and the reads below)
                const uint64_t t = of_total(uni, sum);
                uint64_t upto_w = 0;
                constexpr uint64_t low = (1 << SA_INDEX_BITS) - 1;
                if (stays) {
                    for (int j = part; j < n_list; j += per) { if ((candidates[j] & low) > (key & low)) { upto_w += weights[j]; } }
                }
                upto_w = group_sum(upto_w);
                if (stays && part == 0 && upto_w <= t && t < upto_w + w) {
                    p.ids[row] = index_of(key);
                    if (p.probs) { p.probs[row] = (float)((double)w / (double)sum); }
                }
                return;
            }
            // sorted, cut from the end, put back into the order of indices, drawn
            sort_list(candidates, n_list);
            const int n1 = min(n_list, top_k);
            uint64_t w0 = 0, w1 = 0, k0 = 0, k1 = 0, all_w;
            if (2 * tid < n1) { k0 = candidates[2 * tid]; w0 = weight(value_of(k0)); }
            if (2 * tid + 1 < n1) { k1 = candidates[2 * tid + 1]; w1 = weight(value_of(k1)); }
            const uint64_t up = block_upto(w0 + w1, sh.scan, &all_w);
            const uint64_t stop = by_p ? reach(all_w) : ~0ull;
            bool in0 = 2 * tid < n1 && up - w1 - w0 < stop, in1 = 2 * tid + 1 < n1 && up - w1 < stop;
            if (fine) {
                const double floor = min_p > 0.f ? (double)fminf(min_p, 1.f) : 0.0, d0 = in0 ? fine_weight(value_of(k0), largest, temp) : 0.0, d1 = in1 ? fine_weight(value_of(k1), largest, temp) : 0.0;
                in0 = d0 > 0 && d0 >= floor; in1 = d1 > 0 && d1 >= floor;
                w0 = (uint64_t)__double_as_longlong(d0); w1 = (uint64_t)__double_as_longlong(d1);
            } else { in0 = in0 && w0 >= least; in1 = in1 && w1 >= least; }
            const uint64_t kept = block_sum((in0 ? 1 : 0) + (in1 ? 1 : 0), sh.scan);          // (a prefix of the list)
            const uint64_t sum = block_sum((in0 ? w0 : 0) + (in1 ? w1 : 0), sh.scan);
            // by index: the key's low bits, ascending as descending complements; the weights are found again from their place in the sorted list
            uint64_t *by_index = candidates;
            __syncthreads();
            constexpr uint64_t low = (1 << SA_INDEX_BITS) - 1;
            if (in0) { by_index[2 * tid] = ((k0 & low) << 11 | (2 * tid)) + 1; weights[2 * tid] = w0; }
            if (in1) { by_index[2 * tid + 1] = ((k1 & low) << 11 | (2 * tid + 1)) + 1; weights[2 * tid + 1] = w1; }
            sort_list(by_index, (int)kept);
            if (fine) {
                if (tid == 0) { fine_draw_list(p, row, by_index, weights, (int)kept, uni); }
                return;
            }
            uint64_t v0 = 0, v1 = 0, p0 = 0, p1 = 0, ignore;
            if (2 * tid < (int)kept) { p0 = by_index[2 * tid] - 1; v0 = weights[p0 & 2047]; }
            if (2 * tid + 1 < (int)kept) { p1 = by_index[2 * tid + 1] - 1; v1 = weights[p1 & 2047]; }
            const uint64_t upto2 = block_upto(v0 + v1, sh.scan, &ignore);
            const uint64_t t = of_total(uni, sum);
            const bool hit0 = v0 > 0 && upto2 - v1 - v0 <= t && t < upto2 - v1, hit1 = v1 > 0 && upto2 - v1 <= t && t < upto2;
            if (hit0 || hit1) {
                p.ids[row] = (int)(low - ((hit0 ? p0 : p1) >> 11));
                if (p.probs) { p.probs[row] = (float)((double)(hit0 ? v0 : v1) / (double)sum); }
            }
            return;
        }
        search = true;
    } else if (by_p) {
        sh.limb[0][tid] = sh.limb[1][tid] = sh.limb[2][tid] = 0;
        count_all();
        const uint2 n2 = counts();
        // what the bins weigh, to 1.6 %: the bins in which top_p may be reached
        const float step = -(float)(p.frac_bits + 1) / SA_BINS;     // log2 of a weight, a bin
        uint64_t all;
        const uint64_t m0 = (uint64_t)((double)exp2f(step * (2 * tid + 0.5f)) * n2.x * 1099511627776.0), m1 = (uint64_t)((double)exp2f(step * (2 * tid + 1.5f)) * n2.y * 1099511627776.0);   // x 2^40
        const uint64_t upto = block_upto(m0 + m1, sh.scan, &all), before_b = upto - m0 - m1;
        const double   goal = (double)max(top_p, 0.f) * (double)all;
        const uint64_t lo = (uint64_t)(0.965 * goal), hi = min((uint64_t)(1.035 * goal), all);
        if (tid == 0) { sh.found = 0; sh.found2 = SA_BINS - 1; }
        __syncthreads();
        if (before_b < lo && lo <= upto) { sh.found = lo <= before_b + m0 ? 2 * tid : 2 * tid + 1; }
        if (before_b < hi && hi <= upto) { sh.found2 = min(hi <= before_b + m0 ? 2 * tid + 1 : 2 * tid + 2, SA_BINS - 1); }
        __syncthreads();
        const float first = (float)sh.found, behind = (float)(sh.found2 + 1);
        const float sub_scale = (float)SA_SUB / (behind - first);
        auto sub_of = [&](float b) { return min(SA_SUB - 1, (int)((b - first) * sub_scale)); };
        uint64_t front = 0, total = 0;
        x.fours([&](const float (&v)[4], int) {
            uint64_t ww[4];
            weight.of(v, ww);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float b = bin_of(v[e]);
                total += ww[e];
                front += b < first ? ww[e] : 0;
                if (b >= first && b < behind) {
                    const int s = sub_of(b);
                    atomicAdd(&sh.limb[0][s], (uint32_t)(ww[e] & 0x7fff));
                    atomicAdd(&sh.limb[1][s], (uint32_t)(ww[e] >> 15) & 0x7fff);
                    if (ww[e] >> 30) { atomicAdd(&sh.limb[2][s], (uint32_t)(ww[e] >> 30)); }
                }
            }
        });
        front = block_sum(front, sh.scan);
        total = block_sum(total, sh.scan);
        if (tid < (int)ctas) { cluster_store64(cluster_map(smem_u32(sh.share[1] + rank), tid), front); cluster_store64(cluster_map(smem_u32(sh.share2 + rank), tid), total); }
        cluster_sync();
        front = total = 0;
        for (uint32_t r = 0; r < ctas; ++r) { front += sh.share[1][r]; total += sh.share2[r]; }
        uint64_t mass = 0;                               // of this thread's bin of the bracket
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            uint32_t v[SA_MAX_CLUSTER];
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) { v[r] = r < ctas ? cluster_load32(cluster_map(smem_u32(sh.limb[i]) + tid * 4, r)) : 0; }
#pragma unroll
            for (uint32_t r = 0; r < SA_MAX_CLUSTER; ++r) { mass += (uint64_t)v[r] << 15 * i; }
        }
        const uint64_t stop = reach(total);
        const uint64_t upto_s = front + block_upto(mass, sh.scan, &all);
        if (tid == 0) { sh.found = -1; }
        __syncthreads();
        if (upto_s - mass < stop && stop <= upto_s) { sh.found = tid; sh.total = upto_s - mass; }
        __syncthreads();
        const int sub = sh.found;
        if (sub < 0) { search = true; }              // (not reached inside the bracket)
        else {
            const uint32_t n_in_bin = gather(bin_of(own) < behind, [&](float v) { const float b = bin_of(v); return b >= first && b < behind && sub_of(b) == sub; });
            // the first CTA finds the last one that stays and tells all
            if (rank == 0) {
                const int nn = (int)n_in_bin;
                uint64_t found = 0;
                if (nn <= SA_LIST) {
                    sort_list(candidates, nn);
                    uint64_t w0 = 0, w1 = 0, ignore;
                    if (2 * tid < nn) { w0 = weight(value_of(candidates[2 * tid])); }
                    if (2 * tid + 1 < nn) { w1 = weight(value_of(candidates[2 * tid + 1])); }
                    const uint64_t up = sh.total + block_upto(w0 + w1, sh.scan, &ignore);
                    const uint64_t n_in = block_sum((2 * tid < nn && up - w1 - w0 < stop ? 1 : 0) + (2 * tid + 1 < nn && up - w1 < stop ? 1 : 0), sh.scan);
                    found = n_in > 0 ? candidates[n_in - 1] : 0;
                }
                if (tid < (int)ctas) { cluster_store64(cluster_map(smem_u32(&sh.cut), tid), found); }
            }
            cluster_sync();
            cut = sh.cut;
            search = cut == 0;
        }
    }
    if (search) {
        int turn = 0;
        cluster_sync();                                   // (nobody reads the shares of an earlier exchange any more)
        if (by_k) {
            for (int bit = 31 + SA_INDEX_BITS; bit >= 0; --bit) {
                if (sum_from(cut | (uint64_t)1 << bit, true, turn++) >= (uint64_t)top_k) { cut |= (uint64_t)1 << bit; }
            }
        }
        if (by_p) {
            const uint64_t floor = cut, stop = reach(sum_from(floor, false, turn++));
            cut = 0;
            for (int bit = 31 + SA_INDEX_BITS; bit >= 0; --bit) {
                if (sum_from(max(floor, cut | (uint64_t)1 << bit), false, turn++) >= stop) { cut |= (uint64_t)1 << bit; }
            }
            cut = max(cut, floor);
        }
    }

    // draw: warps have contiguous stretches
    const int stretch = ((x.n + SA_WARPS - 1) / SA_WARPS + 127) & ~127, from = min(warp * stretch, x.n), to = min(from + stretch, x.n);
    const float cut_value = cut == 0 ? -CUDART_INF_F : value_of(cut);
    const int   cut_index = cut == 0 ? p.n_vocab : index_of(cut);
    if (fine) { fine_draw<T, KEPT>(p, sh, x, row, largest, temp, min_p, uni, cut_value, cut_index, rank, ctas); return; }
    auto stays = [&](float v, int i, uint64_t w) {
        return v >= cut_value && !(v == cut_value && x.base + i > cut_index) && w >= least ? w : (uint64_t)0;
    };
    uint64_t s = 0;
    if (cut == 0 && least == 1) {                         // (all of them)
        x.stretch(from, to, lane, 32, [&](const float (&v)[4], int) {
            uint64_t w[4];
            weight.of(v, w);
            s += (w[0] + w[1]) + (w[2] + w[3]);
        });
    } else {
        x.stretch(from, to, lane, 32, [&](const float (&v)[4], int i) {
            if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) < cut_value) { return; }
            uint64_t w[4];
            weight.of(v, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) { s += stays(v[e], i + e, w[e]); }
        });
    }
    s = warp_sum64(s);
    __syncthreads();
    if (lane == 0) { sh.scan[warp] = s; }
    __syncthreads();
    uint64_t mine = 0, before = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) { const uint64_t u = sh.scan[w]; before += w < warp ? u : 0; mine += u; }
    cluster_sync();                                       // (shares of earlier exchanges are read)
    const uint64_t total = cluster_total(mine, sh.share[0], ctas, rank);
    for (uint32_t r = 0; r < rank; ++r) { before += sh.share[0][r]; }
    const uint64_t t = of_total(uni, total);
    if (before <= t && t < before + s) {
        uint64_t c = before;
        for (int i0 = from; i0 < to; i0 += 32) {
            const int i = i0 + lane;
            const uint64_t w = i < to ? stays(x(i), i, weight(x(i))) : 0, upto = c + warp_upto64(w);
            const unsigned hit = __ballot_sync(0xffffffffu, t < upto);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    p.ids[row] = x.base + i;
                    if (p.probs) { p.probs[row] = (float)((double)w / (double)total); }
                }
                break;
            }
            c = __shfl_sync(0xffffffffu, upto, 31);
        }
    }
}

__global__ void weights_kernel(const uint64_t *powers, const float *logits, int n, float largest, float temp, int bits, uint64_t *weights) {
    const double c = Weight::factor(temp);
    Weight w;
    w.set(powers, largest, c, 56 / c, bits);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) { weights[i] = w(logits[i]); }
}
int weight_bits(int n_vocab) {
    int log2_vocab = 0;
    while ((1 << log2_vocab) < n_vocab) { ++log2_vocab; }
    return std::min(45, 62 - log2_vocab);
}

template <class T, bool KEPT>
cudaError_t launch_sample(SampleParams &p, int n_rows, int ctas, const LaunchCfg &cfg) {
    const size_t smem = sizeof(SampleShared) + (KEPT ? (size_t)p.per * 4 : 0);
    const void *kernel = reinterpret_cast<const void *>(sample_kernel<T, KEPT>);
    const cudaError_t err = allow_dynamic_smem(kernel, smem);
    if (err != cudaSuccess) { return err; }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)n_rows * ctas); lc.blockDim = dim3(SA_THREADS); lc.dynamicSmemBytes = smem; lc.stream = cfg.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr; lc.numAttrs = cfg.pdl ? 2 : 1;
    void *args[] = {&p};
    return cudaLaunchKernelExC(&lc, kernel, args);
}
template <class T>
cudaError_t launch_sample(SampleParams &p, int n_rows, int sms, const LaunchCfg &cfg) {
    // slices of up to 16384 logits, so that an SM holds two CTAs; smaller ones while there are SMs without a CTA (one row of 32 000 at a temperature alone 8.6 us on
    // eight CTAs, 16.7 on two)
    int ctas = 1;
    while (ctas < SA_MAX_CLUSTER && (p.n_vocab > 16384 * ctas || (n_rows * ctas < sms && p.n_vocab > 2048 * ctas))) { ctas *= 2; }
    p.per = ((p.n_vocab + ctas - 1) / ctas + 127) & ~127;
    return (size_t)p.per <= SA_MAX_SLICE ? launch_sample<T, true>(p, n_rows, ctas, cfg) : launch_sample<T, false>(p, n_rows, ctas, cfg);
}

}  // namespace
}  // namespace spyb

using namespace spyb;

static spyb_status check_sample(Refusal &no, const spyb_sample_desc &d) {
    if (!value_type(d.number_type)) { return no.because("sample: logits of type %d", d.number_type); }
    if (d.n_rows < 0 || d.n_rows > (1 << 24) || d.n_vocab < 1 || d.n_vocab > (1 << SA_INDEX_BITS) || (d.n_rows > 1 && d.row_stride < d.n_vocab)) {
        return no.because("sample: %d rows of %d logits, %lld apart", d.n_rows, d.n_vocab, (long long)d.row_stride);
    }
    if (d.logits == nullptr || d.ids == nullptr) { return no.because("sample: logits and ids must be there"); }
    const void *const words[] = {d.temperature, d.top_k, d.top_p, d.min_p, d.uniform, d.ids, d.probs};
    bool aligned = aligned_to(d.logits, d.number_type == SPYB_FP32 ? 4 : 2);
    for (const void *w : words) { aligned &= aligned_to(w, 4); }
    if (!aligned) { return no.because("sample: operands must be aligned to their elements"); }
    return SPYB_SUCCESS;
}

extern "C" spyb_status spyb_sample_check(const spyb_sample_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_sample(no, *d), message, size);
}

extern "C" spyb_status spyb_sample(spyb_backend *be, const spyb_sample_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_sample(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    SampleParams p;
    p.logits = d->logits; p.row_stride = d->row_stride; p.n_vocab = d->n_vocab;
    p.frac_bits = weight_bits(d->n_vocab);
    p.temperature = d->temperature; p.top_k = d->top_k; p.top_p = d->top_p; p.min_p = d->min_p; p.uniform = d->uniform; p.ids = d->ids; p.probs = d->probs;
    p.powers = be->d_power_table; p.error_flag = be->d_error_flag; p.wait_limit = be->wait_limit_ns;
    const LaunchCfg cfg = be->launch_cfg(be->config.use_pdl != 0);
    SPYB_CUDA(be, d->number_type == SPYB_FP32 ? launch_sample<float>(p, d->n_rows, be->num_sms_total, cfg) : launch_sample<__half>(p, d->n_rows, be->num_sms_total, cfg));
    return SPYB_SUCCESS;
}

// The weights as the sampler's kernels make them: in units of 2^-S of the largest, S as for n_vocab logits. Host arrays.
extern "C" spyb_status spyb_sample_weights(spyb_backend *be, const float *logits_host, int32_t n, float largest, float temperature, int32_t n_vocab, uint64_t *weights_host) {
    if (be == nullptr || logits_host == nullptr || weights_host == nullptr || n < 1 || n_vocab < 1 || n_vocab > (1 << SA_INDEX_BITS) || !(temperature > 0.f)) { return SPYB_FAIL; }
    use_device(be->config.device_id);
    uint8_t *mem = nullptr;
    SPYB_CUDA(be, cudaMalloc(&mem, (size_t)n * 12));
    uint64_t *weights = reinterpret_cast<uint64_t *>(mem);
    float    *logits  = reinterpret_cast<float *>(weights + n);
    cudaError_t err = upload(logits, logits_host, (size_t)n * 4);
    if (err == cudaSuccess) {
        weights_kernel<<<64, 256, 0, be->stream>>>(be->d_power_table, logits, n, largest, temperature, weight_bits(n_vocab), weights);
        err = cudaGetLastError();
    }
    if (err == cudaSuccess) { err = cudaMemcpyAsync(weights_host, weights, (size_t)n * 8, cudaMemcpyDeviceToHost, be->stream); }
    if (err == cudaSuccess) { err = cudaStreamSynchronize(be->stream); }
    cudaFree(mem);
    SPYB_CUDA(be, err);
    return SPYB_SUCCESS;
}
