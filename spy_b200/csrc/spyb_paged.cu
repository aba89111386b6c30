// Caches in pages: appending a step's keys and values with the position rotation on the way, attention of few rows a sequence (single tokens, guessed tokens,
// head dimensions without a tensor-memory kernel), and the entry points of both operators.

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <vector>

#include <math_constants.h>

#include "spyb_internal.h"
#include "spyb_paged.cuh"

namespace spyb {
namespace {

// ---------------------------------------------------------------------------------------------- append
// Memory bound: every element is read once and written once, (4 + 2) or (2 + 2) bytes. A CTA has one row; a thread has eight elements of a head - a 16-byte piece of
// the output, or half of two pieces where the pairs are halves - in every 8th or 16th head, so that its (up to) four angles are made once a row. Angles are
// position x share of a circle in 64 bits, reduced to half a turn either way: in f32 a position of 100 000 leaves an angle 0.004 of uncertainty.
// Measured: 9246 rows of 120 heads of 128 elements (f32, 852 MB) 149 us, 5.7 TB/s; one row 3.5 us and 96 rows 6 to 7 us, a launch and a chain of dependent loads
// (whose row, which position, which page), beside which the row's first elements come.
constexpr int AP_THREADS = 256;

__device__ __forceinline__ int sequence_of(const PagedView &v, int row) {   // the last s with row_start[s] <= row, by a whole warp; -1 and n_seq: nobody's
    const int lane = threadIdx.x & 31;
    int lo = 0, n = v.n_seq + 1;
    while (n > 32) {
        const int step = (n + 31) / 32, i = lo + lane * step;
        const int c = __popc(__ballot_sync(0xffffffffu, lane * step < n && v.row_start[min(i, v.n_seq)] <= row));
        if (c == 0) { return -1; }
        lo += (c - 1) * step;
        n = min(step, v.n_seq + 1 - lo);
    }
    const int c = __popc(__ballot_sync(0xffffffffu, lane < n && v.row_start[min(lo + lane, v.n_seq)] <= row));
    return lo + c - 1;
}
__device__ __forceinline__ void load4(const float *p, float *v) { const float4 x = __ldcs(reinterpret_cast<const float4 *>(p)); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
__device__ __forceinline__ void load4(const __half *p, float *v) {
    const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&x.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&x.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ void store4(float *p, const float *v) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__half *p, const float *v) { *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3])); }

// AHEAD: a head's elements are fetched while the one before is turned, for calls whose CTAs run all at once: 96 rows of 56 heads 6.8 us against 7.9, 700 rows 10.1 against 11.1.
// (Where CTAs follow one another the registers cost more than it gives: 9246 rows of 120 heads 152 us against 149, in fp16 155 against 139.)
template <class TIn, class TQ, bool AHEAD>
__global__ void __launch_bounds__(AP_THREADS) paged_append_kernel(const __grid_constant__ PagedAppend p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    const int per = p.head_dim / 8, slots = AP_THREADS / per;       // threads of a head, heads at a time
    const int slot = threadIdx.x / per, item = threadIdx.x - slot * per, total = p.n_head + 2 * p.n_head_kv;
    const bool turned = item < p.rot / 8;
    const int  e0 = turned && p.halves ? 4 * item : 8 * item, e1 = turned && p.halves ? e0 + p.rot / 2 : e0 + 4;
    int  h = blockIdx.y * slots + slot;
    const int step = slots * gridDim.y;
    auto fetch = [&](int head, float (&x)[8]) {
        const bool is_q = head < p.n_head, is_k = !is_q && head < p.n_head + p.n_head_kv;
        const int  hh = is_q ? head : is_k ? head - p.n_head : head - p.n_head - p.n_head_kv;
        const TIn *src = static_cast<const TIn *>(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride) + (int64_t)hh * p.head_dim;
        load4(src + e0, x);
        load4(src + e1, x + 4);
    };
    // (the first head's elements are on their way while the row's place is found)
    float x[8];
    const bool works = slot < slots && h < total;
    if (works) { fetch(h, x); }
    const int s = sequence_of(p.view, row);
    if (s < 0 || s >= p.view.n_seq || !works) { return; }
    const int end = p.view.row_start[s + 1];
    const int pos = p.view.n_kv[s] - end + row;
    if (row >= end || pos < 0) { return; }
    int64_t cell = -1;
    if (pos < p.view.n_kv_most) {
        const int page = p.view.page_table[(int64_t)s * p.view.table_stride + pos / p.view.page_size];
        if (page >= 0 && page < p.view.n_pages) { cell = page * p.view.page_stride + (pos % p.view.page_size) * p.view.token_stride; }
    }
    float co[4], si[4];
    if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double t = (double)pos * p.turns[4 * item + i];
            sincospif(2.0f * (float)(t - rint(t)), &si[i], &co[i]);
        }
    }
    for (;;) {
        const bool is_q = h < p.n_head, is_k = !is_q && h < p.n_head + p.n_head_kv;
        const int  hh = is_q ? h : is_k ? h - p.n_head : h - p.n_head - p.n_head_kv;
        const int  next = h + step;
        float ahead[8];
        if (AHEAD && next < total) { fetch(next, ahead); }
        if (turned && (is_q || is_k)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int a = p.halves ? i : 2 * i, b = p.halves ? i + 4 : 2 * i + 1;
                const float u = x[a], w = x[b];
                x[a] = u * co[i] - w * si[i];
                x[b] = u * si[i] + w * co[i];
            }
        }
        if (is_q) {
            TQ *dst = static_cast<TQ *>(p.q_out) + row * p.q_out_stride + (int64_t)hh * p.head_dim;
            store4(dst + e0, x); store4(dst + e1, x + 4);
        } else if (cell >= 0) {
            __half *dst = (is_k ? p.k_cache : p.v_cache) + cell + hh * p.view.head_stride;
            store4(dst + e0, x); store4(dst + e1, x + 4);
        }
        if (next >= total) { break; }
        h = next;
        if (AHEAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = ahead[i]; }
        } else { fetch(h, x); }
    }
}

// ---------------------------------------------------------------------------------------------- attention of few rows
// Memory bound: the positions of a sequence are read once a K/V head, 4 head_dim bytes each. Every warp works for itself on blocks of 16 positions - its own ring of
// asynchronous copies, scores and values by mma.sync on up to 32 rows, a running maximum and sum in registers - and the warps of a CTA, then the CTAs
// of an item are joined at the end. The maximum that probabilities are taken against follows the true one only when that is 2^8 above it: the
// accumulators are hardly ever rescaled, and p <= 2^8 is as exact in fp16 as p <= 1.
// Measured: three sequences of 100 000 positions, 40 query heads on 8 of 128 elements (1.2 GB) 192 to 199 us, 6.1 to 6.3 TB/s; 64 sequences of up to 4096, 32 on 8: 91 us,
// 6.0 TB/s, heads of 64: 54 us, 5.1 TB/s; one of 4000, 32 on 32 (66 MB): 19.7 us. What is above the memory's time: some 6 us until the first block is there (lengths, the
// plan, the page table, the block, one after the other), the join of items on a cut (2 to 3 us), and each warp's chain of copy, scores, powers and values with
// eight to twelve warps an SM.
constexpr int PR_WARPS = 4, PR_BLOCK = 16, PR_UNIT = PR_WARPS * PR_BLOCK;

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool there) {   // zeros where it is not
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ bool not_finite2(uint32_t h2) { return (h2 & 0x7c00u) == 0x7c00u || (h2 & 0x7c000000u) == 0x7c000000u; }

template <int HD> struct RowsShape {
    static constexpr int ROW = HD <= 64 ? 128 : 256;                 // bytes of a position in shared memory (16-byte pieces swizzled within eight)
    static constexpr int STAGE = 2 * PR_BLOCK * ROW;
    static constexpr int STAGES = ROW == 128 ? 4 : 3;                // (short positions: three CTAs an SM; a warp's time a block is what their instructions wait for one another)
    static constexpr int RING = PR_WARPS * STAGES * STAGE;
};
template <int HD, int MT> struct RowsSmem {       // the ring; what the warps found: beside it for up to EARLY rows, in its place for more; the masks of the ring's stages
    static constexpr int EARLY = MT == 1 ? 8 : 0, FOUND = PR_WARPS * 16 * MT * (HD + 2) * 4, RING = RowsShape<HD>::RING > FOUND ? RowsShape<HD>::RING : FOUND;
    static constexpr int CTAS = MT == 1 && HD <= 64 ? 3 : 2;         // of an SM (64 single tokens, heads of 64, before the cut counted items' beginnings: 65 us with three, 79 with two; longer heads' rings leave room for two)
    static constexpr int MASKS = RING + PR_WARPS * EARLY * (HD + 2) * 4, BYTES = MASKS + PR_WARPS * RowsShape<HD>::STAGES * 4;
};
// IN_PAGE: a block's positions lie in one page (pages of a multiple of 16), heads of up to 64: 64 single tokens 64.8 us against 66.6. (Longer heads' blocks take longer than
// the table's latency: 103.2 us against 102.8, they go without.)
template <int HD, int MT, bool IN_PAGE>
__global__ void __launch_bounds__(PR_WARPS * 32) paged_rows_kernel(const __grid_constant__ PagedAttention p) {
    constexpr int PR_STAGES = RowsShape<HD>::STAGES, TILE = 16 * MT, ROW = RowsShape<HD>::ROW, STAGE = RowsShape<HD>::STAGE, NT = PR_WARPS * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PagedPlanShared plan;
    __shared__ int last_one;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t *there = reinterpret_cast<uint32_t *>(smem + RowsSmem<HD, MT>::MASKS) + warp * PR_STAGES;
    const uint32_t ring = smem_u32(smem) + warp * PR_STAGES * STAGE;
    pdl_launch_dependents();
    pdl_wait();
    PagedPlace at = paged_plan<NT, PR_UNIT, PR_BLOCK>(p, true, 1, plan);
    if (at.unit >= at.end) { return; }
    PagedSeq q = paged_seq(p.view, at.seq);
    int seq = at.seq, head = at.head, tile = at.tile, off = at.off;
    PagedItem it;
    int todo, ka, kb, n_block, packed;        // of the item that comes next: units of this CTA, positions [ka, kb), blocks of them; rows of the tile
    const int32_t *table;
    const __half *kbase, *vbase;
    auto describe = [&]() {
        it = paged_item<PR_UNIT, PR_BLOCK>(p, q, tile);
        todo = (int)min((int64_t)(it.units - off), at.end - at.unit);
        ka = it.lo + off * PR_UNIT; kb = min(it.hi, ka + todo * PR_UNIT);
        n_block = kb > ka ? (kb - ka + PR_BLOCK - 1) / PR_BLOCK : 0;
        packed = min(TILE, q.rows * p.group - tile * TILE);
        table = p.view.page_table + (int64_t)seq * p.view.table_stride;
        kbase = p.k + head * p.view.head_stride; vbase = p.v + head * p.view.head_stride;
    };
        auto page_of = [&](int b) {          // page of block b, or (lanes 0..15 and 16..31 alike) of this lane's position in it; -1: none
            const int j = ka + b * PR_BLOCK + (IN_PAGE ? 0 : lane & 15);
            return b < n_block && j < kb ? table[p.page_shift >= 0 ? j >> p.page_shift : j / p.view.page_size] : -1;
        };
        auto issue = [&](int b, int stage, int page) {
            const int j = ka + b * PR_BLOCK + (IN_PAGE ? 0 : lane & 15);
            const bool ok = page >= 0 && page < p.view.n_pages;
            const int in_page = p.page_shift >= 0 ? j & (p.view.page_size - 1) : j % p.view.page_size;
            const int64_t cell = ok ? page * p.view.page_stride + in_page * p.view.token_stride : 0;
            const unsigned mask = IN_PAGE ? (ok ? (kb - j >= PR_BLOCK ? 0xffffu : (1u << (kb - j)) - 1) : 0u) : __ballot_sync(0xffffffffu, ok) & 0xffffu;
            const uint32_t dst = ring + stage * STAGE;
            constexpr int PIECES = HD / 8;
            if constexpr (IN_PAGE) {
                static_assert(32 % PIECES == 0, "a row's pieces are lanes side by side");
                constexpr int AT_ONCE = 32 / PIECES;
                const int r0 = lane / PIECES, c = lane % PIECES;
                int64_t o = cell + r0 * p.view.token_stride + c * 8;
                const int64_t more = AT_ONCE * p.view.token_stride;
#pragma unroll
                for (int i = 0; i < PIECES / 2; ++i) {
                    const int r = i * AT_ONCE + r0;
                    const bool in = (mask >> r) & 1;
                    const uint32_t d = dst + r * ROW + ((c ^ (r & 7)) << 4);
                    const int64_t at = in ? o : 0;
                    cp_async16(d, kbase + at, in);
                    cp_async16(d + PR_BLOCK * ROW, vbase + at, in);
                    o += more;
                }
            } else {
#pragma unroll
                for (int i = 0; i < PIECES / 2; ++i) {
                    const int x = i * 32 + lane, r = x / PIECES, c = x - r * PIECES;
                    const bool in = (mask >> r) & 1;
                    const int64_t row = __shfl_sync(0xffffffffu, cell, r), o = in ? row + c * 8 : 0;
                    const uint32_t d = dst + r * ROW + ((c ^ (r & 7)) << 4);
                    cp_async16(d, kbase + o, in);
                    cp_async16(d + PR_BLOCK * ROW, vbase + o, in);
                }
            }
            if (lane == 0) { there[stage] = mask; }
            cp_commit();
        };

    // IN_PAGE: a lane has the page of every 32nd block of this warp, the next 32 are read while these are in use; a block's is told by its lane
    int page = -1, ids = -1, ids_next = -1, issued = 0;   // (page: of the block that is issued next)
    auto next_page = [&](int b) {             // of block b, the `issued`-th of this warp
        if (!IN_PAGE) { return page_of(b); }
        const int l = issued & 31;
        if (l == 0) { ids = ids_next; ids_next = page_of(warp + (issued + 32 + lane) * PR_WARPS); }
        ++issued;
        return __shfl_sync(0xffffffffu, ids, l);
    };
    uint32_t qf[MT][HD / 16][4];
    int pos[MT][2];
    auto start = [&]() {                      // the item's first blocks are on their way while its Q comes
        issued = 0;
        if (IN_PAGE) { ids_next = page_of(warp + lane * PR_WARPS); }
        page = next_page(warp);
#pragma unroll
        for (int i = 0; i < PR_STAGES - 1; ++i) {
            const int next = next_page(warp + (i + 1) * PR_WARPS);
            if (warp + i * PR_WARPS < n_block) { issue(warp + i * PR_WARPS, i, page); } else { cp_commit(); }
            page = next;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int r = m * 16 + hf * 8 + (lane >> 2), pr = tile * TILE + min(r, packed - 1);
                const int token = (int)((unsigned)pr / (unsigned)p.group), g = pr - token * p.group;
                pos[m][hf] = q.first + token;
                const uint32_t *src = reinterpret_cast<const uint32_t *>(p.q + (int64_t)(q.row0 + token) * p.q_stride + (head * p.group + g) * HD) + (lane & 3);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    qf[m][ks][hf] = r < packed ? src[ks * 8] : 0u;
                    qf[m][ks][2 + hf] = r < packed ? src[ks * 8 + 4] : 0u;
                }
            }
        }
    };
    describe();
    start();
    for (;;) {
        const int pos_first = q.first + (int)((unsigned)(tile * TILE) / (unsigned)p.group), pos_last = q.first + (int)((unsigned)(tile * TILE + packed - 1) / (unsigned)p.group);
        float o[MT][HD / 8][4], mx[MT][2], sum[MT][2], base[MT][2], over[MT][2];   // (base: the maximum, or 0 for none; over: scores beyond it move the maximum)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            mx[m][0] = mx[m][1] = over[m][0] = over[m][1] = -CUDART_INF_F; sum[m][0] = sum[m][1] = base[m][0] = base[m][1] = 0.f;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) { o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f; }
        }
        int stage = 0;
        for (int b = warp; b < n_block; b += PR_WARPS) {
            {
                const int ahead = b + (PR_STAGES - 1) * PR_WARPS, next = next_page(ahead + PR_WARPS);
                const int to = stage == 0 ? PR_STAGES - 1 : stage - 1;
                __syncwarp();
                if (ahead < n_block) { issue(ahead, to, page); } else { cp_commit(); }
                page = next;
            }
            cp_wait<PR_STAGES - 1>();
            __syncwarp();
            const uint32_t ks_addr = ring + stage * STAGE, vs_addr = ks_addr + PR_BLOCK * ROW;
            const uint32_t mask = there[stage];
            const int j0 = ka + b * PR_BLOCK;
            const bool whole = mask == 0xffffu && (!p.causal || (j0 + PR_BLOCK - 1 <= pos_first && (p.window <= 0 || j0 > pos_last - p.window)));
            float sc[MT][2][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int n = 0; n < 2; ++n) { sc[m][n][0] = sc[m][n][1] = sc[m][n][2] = sc[m][n][3] = 0.f; }
            }
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                uint32_t kf[4];
                const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
                ldsm4(ks_addr + r * ROW + ((c ^ (r & 7)) << 4), kf);
#pragma unroll
                for (int m = 0; m < MT; ++m) { mma16816(sc[m][0], qf[m][ks], kf[0], kf[1]); mma16816(sc[m][1], qf[m][ks], kf[2], kf[3]); }
            }
            // scores against the maximum, in powers of two
            bool above = false;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float &x = sc[m][n][e];
                        x = fmaf(x, p.scale_log2, -base[m][e >> 1]);
                        if (!whole) {
                            const int jj = n * 8 + (lane & 3) * 2 + (e & 1), d = pos[m][e >> 1] - (j0 + jj);
                            const bool seen = ((mask >> jj) & 1) && (!p.causal || (d >= 0 && (p.window <= 0 || d < p.window)));
                            x = seen ? x : -CUDART_INF_F;
                        }
                        above |= x > over[m][e >> 1];
                    }
                }
            }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float v = fmaxf(fmaxf(sc[m][0][2 * hf], sc[m][0][2 * hf + 1]), fmaxf(sc[m][1][2 * hf], sc[m][1][2 * hf + 1]));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                        const float to = fmaxf(mx[m][hf], base[m][hf] + v), f = to == mx[m][hf] ? 1.f : ex2(mx[m][hf] - to);   // (2^-inf = 0 at the first)
                        const float from = base[m][hf];
                        mx[m][hf] = to; sum[m][hf] *= f;
                        base[m][hf] = to == -CUDART_INF_F ? 0.f : to;
                        over[m][hf] = to == -CUDART_INF_F ? to : 8.f;
#pragma unroll
                        for (int n = 0; n < 2; ++n) { sc[m][n][2 * hf] += from - base[m][hf]; sc[m][n][2 * hf + 1] += from - base[m][hf]; }
#pragma unroll
                        for (int n = 0; n < HD / 8; ++n) { o[m][n][2 * hf] *= f; o[m][n][2 * hf + 1] *= f; }
                    }
                }
            }
            uint32_t pf[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float a = ex2(sc[m][n][2 * hf]), c = ex2(sc[m][n][2 * hf + 1]);
                        sum[m][hf] += a + c;
                        pf[m][2 * n + hf] = pack2(a, c);
                    }
                }
            }
            uint32_t bad = 0;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t vf[4];
                const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * d + (lane >> 4);
                ldsm4t(vs_addr + r * ROW + ((c ^ (r & 7)) << 4), vf);
                if (!whole) { bad |= not_finite2(vf[0]) | not_finite2(vf[1]) | not_finite2(vf[2]) | not_finite2(vf[3]); if (__any_sync(0xffffffffu, bad)) { break; } }
#pragma unroll
                for (int m = 0; m < MT; ++m) { mma16816(o[m][2 * d], pf[m], vf[0], vf[1]); mma16816(o[m][2 * d + 1], pf[m], vf[2], vf[3]); }
            }
            if (__any_sync(0xffffffffu, bad)) {
                // 0 x inf: a position that some rows see and others do not holds a value that is not finite. Products of what is seen alone, for the rest of the columns
                // (those in front of the bad one are done; a column whose values are finite gets the same sums either way)
                int d0 = 0;
                for (; d0 < HD / 16; ++d0) {   // the first piece with such a value, as the loop above found it
                    uint32_t vf[4];
                    const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * d0 + (lane >> 4);
                    ldsm4t(vs_addr + r * ROW + ((c ^ (r & 7)) << 4), vf);
                    if (__any_sync(0xffffffffu, not_finite2(vf[0]) | not_finite2(vf[1]) | not_finite2(vf[2]) | not_finite2(vf[3]))) { break; }
                }
                for (int j = 0; j < PR_BLOCK; ++j) {
                    const int src = (lane & ~3) | ((j & 7) >> 1);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const uint32_t h = __shfl_sync(0xffffffffu, j < 8 ? pf[m][hf] : pf[m][2 + hf], src);
                            const float pj = h2f((uint16_t)(j & 1 ? h >> 16 : h & 0xffffu));
                            const int d = pos[m][hf] - (j0 + j);
                            const bool seen = ((mask >> j) & 1) && (!p.causal || (d >= 0 && (p.window <= 0 || d < p.window)));
#pragma unroll
                            for (int n = 0; n < HD / 8; ++n) {
                                if (n >= 2 * d0 && seen) {
                                    const uint32_t v2 = lds32(vs_addr + j * ROW + ((n ^ (j & 7)) << 4) + (lane & 3) * 4);
                                    o[m][n][2 * hf] += pj * h2f((uint16_t)(v2 & 0xffffu));
                                    o[m][n][2 * hf + 1] += pj * h2f((uint16_t)(v2 >> 16));
                                }
                            }
                        }
                    }
                }
            }
            stage = stage == PR_STAGES - 1 ? 0 : stage + 1;
        }
        cp_wait<0>();
        __syncwarp();
        // What is known of this item; the next one's copies start before its findings are joined, where these have a place of their own
        const int done = packed, done_tile = tile, done_row0 = q.row0, done_head = head;
        const PagedCut cut = paged_cut(at, at.unit - off, it.units);
        at.unit += todo + p.start_units;
        off = 0;
        const bool more = at.unit < at.end && paged_next(p, true, q, seq, head, tile), early = done <= RowsSmem<HD, MT>::EARLY;
        if (more) { describe(); }
        if (more && early) { start(); }
        if (!early) { __syncthreads(); }
        const int room = early ? RowsSmem<HD, MT>::EARLY : TILE;              // rows of a warp's findings
        float *mo = reinterpret_cast<float *>(smem + (early ? RowsSmem<HD, MT>::RING : 0)), *mm = mo + PR_WARPS * room * HD, *ml = mm + PR_WARPS * room;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                float l = sum[m][hf];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int r = m * 16 + hf * 8 + (lane >> 2);
                if (r < done) {
                    float *dst = mo + (warp * room + r) * HD + (lane & 3) * 2;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) { *reinterpret_cast<float2 *>(dst + n * 8) = make_float2(o[m][n][2 * hf], o[m][n][2 * hf + 1]); }
                    if ((lane & 3) == 0) { mm[warp * room + r] = mx[m][hf]; ml[warp * room + r] = l; }
                }
            }
        }
        __syncthreads();
        constexpr int PART = TILE * (HD + 2);
        float *part = p.partial + paged_slot(blockIdx.x, cut.c0) * PART;
        auto put = [&](int r, int c, float4 v) {   // four elements of a finished row
            const int pr = done_tile * TILE + r, token = (int)((unsigned)pr / (unsigned)p.group), g = pr - token * p.group;
            const int64_t o2 = (int64_t)(done_row0 + token) * p.out_stride + (done_head * p.group + g) * HD + c;
            const float w[4] = {v.x, v.y, v.z, v.w};
            if (p.out_f32) { store4(static_cast<float *>(p.out) + o2, w); } else { store4(static_cast<__half *>(p.out) + o2, w); }
        };
        for (int x = tid; x < done * (HD / 4); x += NT) {
            const int r = x / (HD / 4), c = (x - r * (HD / 4)) * 4;
            float m = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < PR_WARPS; ++w) { m = fmaxf(m, mm[w * room + r]); }
            const float base = m == -CUDART_INF_F ? 0.f : m;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < PR_WARPS; ++w) {
                const float f = ex2(mm[w * room + r] - base);
                const float4 u = *reinterpret_cast<const float4 *>(mo + (w * room + r) * HD + c);
                v.x += f * u.x; v.y += f * u.y; v.z += f * u.z; v.w += f * u.w;
                l += f * ml[w * room + r];
            }
            if (cut.parts == 1) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                put(r, c, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            } else {
                *reinterpret_cast<float4 *>(part + r * HD + c) = v;
                if (c == 0) { part[TILE * HD + r] = m; part[TILE * HD + TILE + r] = l; }
            }
        }
        if (cut.parts > 1) {
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                const unsigned n = atomicAdd(p.arrived + cut.c0, 1u);
                last_one = n == (unsigned)cut.parts - 1;
                if (last_one) { p.arrived[cut.c0] = 0; __threadfence(); }
            }
            __syncthreads();
            if (last_one) {
                for (int x = tid; x < done * (HD / 4); x += NT) {
                    const int r = x / (HD / 4), c = (x - r * (HD / 4)) * 4;
                    float m = -CUDART_INF_F, l = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    // eight CTAs' findings are in flight together; what came before is scaled to the new maximum
#pragma unroll 1
                    for (int i0 = 0; i0 < cut.parts; i0 += 8) {
                        float  pm[8], pl[8], top = m;
                        float4 u[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const bool is = i0 + j < cut.parts;
                            const float *from = p.partial + paged_slot(cut.c0 + (is ? i0 + j : 0), cut.c0) * PART;
                            pm[j] = is ? __ldcg(from + TILE * HD + r) : -CUDART_INF_F;
                            pl[j] = is ? __ldcg(from + TILE * HD + TILE + r) : 0.f;
                            u[j] = is ? __ldcg(reinterpret_cast<const float4 *>(from + r * HD + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) { top = fmaxf(top, pm[j]); }
                        const float base = top == -CUDART_INF_F ? 0.f : top, before = ex2(m - base);
                        m = top; l *= before;
                        v = make_float4(v.x * before, v.y * before, v.z * before, v.w * before);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float f = ex2(pm[j] - base);
                            v.x += f * u[j].x; v.y += f * u[j].y; v.z += f * u[j].z; v.w += f * u[j].w;
                            l += f * pl[j];
                        }
                    }
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    put(r, c, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }
        if (!more) { return; }
        __syncthreads();                      // (the findings' place is free again)
        if (!early) { start(); }
    }
}

template <int HD, int MT, bool IN_PAGE>
cudaError_t launch_rows_as(const PagedAttention &p, int sms, const LaunchCfg &cfg) {
    const void *kernel = reinterpret_cast<const void *>(paged_rows_kernel<HD, MT, IN_PAGE>);
    const cudaError_t err = allow_dynamic_smem(kernel, (size_t)RowsSmem<HD, MT>::BYTES);
    if (err != cudaSuccess) { return err; }
    return launch_maybe_pdl(paged_rows_kernel<HD, MT, IN_PAGE>, dim3(RowsSmem<HD, MT>::CTAS * sms), PR_WARPS * 32, (size_t)RowsSmem<HD, MT>::BYTES, cfg.stream, cfg.pdl, p);
}
template <int HD, int MT>
cudaError_t launch_rows(PagedAttention p, int sms, const LaunchCfg &cfg) {
    const int page = p.view.page_size;
    p.page_shift = -1; p.start_units = PA_START;
    for (int s = 0; s < 31; ++s) { if (page == 1 << s) { p.page_shift = s; } }
    if constexpr (HD <= 64) {
        if (page % PR_BLOCK == 0) { return launch_rows_as<HD, MT, true>(p, sms, cfg); }
    }
    return launch_rows_as<HD, MT, false>(p, sms, cfg);
}

}  // namespace

template <class TIn, class TQ>
static cudaError_t launch_append(const PagedAppend &p, int sms, const LaunchCfg &cfg) {
    const int total = p.n_head + 2 * p.n_head_kv, slots = AP_THREADS / (p.head_dim / 8), loops = (total + slots - 1) / slots;
    // few rows: a row's heads are spread over CTAs (one row of 96 heads 5.8 us against 6.0 in one CTA, 300 rows of 56 heads 9.7 against 9.9)
    const int  split = std::max(1, std::min(loops, 2 * sms / std::max(1, p.view.n_rows)));
    const dim3 grid(p.view.n_rows, split);
    return (int64_t)p.view.n_rows * split <= 5 * sms ? launch_maybe_pdl(paged_append_kernel<TIn, TQ, true>, grid, AP_THREADS, 0, cfg.stream, cfg.pdl, p)      // (five of its CTAs fit an SM)
                                                     : launch_maybe_pdl(paged_append_kernel<TIn, TQ, false>, grid, AP_THREADS, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_append(const PagedAppend &p, int in_type, int q_out_type, int sms, const LaunchCfg &cfg) {
    if (in_type == SPYB_FP32) { return q_out_type == SPYB_FP32 ? launch_append<float, float>(p, sms, cfg) : launch_append<float, __half>(p, sms, cfg); }
    return q_out_type == SPYB_FP32 ? launch_append<__half, float>(p, sms, cfg) : launch_append<__half, __half>(p, sms, cfg);
}

cudaError_t launch_paged_attention_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg) {
    switch (head_dim * 2 + row_tiles - 1) {
    case 64: return launch_rows<32, 1>(p, sms, cfg);
    case 65: return launch_rows<32, 2>(p, sms, cfg);
    case 128: return launch_rows<64, 1>(p, sms, cfg);
    case 129: return launch_rows<64, 2>(p, sms, cfg);
    case 192: return launch_rows<96, 1>(p, sms, cfg);
    case 193: return launch_rows<96, 2>(p, sms, cfg);
    case 256: return launch_rows<128, 1>(p, sms, cfg);
    case 257: return launch_rows<128, 2>(p, sms, cfg);
    default: return cudaErrorInvalidValue;
    }
}

namespace {

int stride_unit(int t) { return t == SPYB_FP32 ? 4 : 8; }

// what both operators ask of the cache and the batch
spyb_status check_view(Refusal &no, const char *what, const spyb_paged_cache &c, const spyb_paged_batch &b) {
    if (c.number_type != SPYB_FP16) { return no.because("%s: a cache of type %d (fp16 it has to be)", what, c.number_type); }
    if (c.k == nullptr || c.v == nullptr || !aligned_to(c.k, 16) || !aligned_to(c.v, 16)) { return no.because("%s: the cache's k and v must be there and 16-byte aligned", what); }
    if (c.n_pages < 1 || c.page_size < 1 || c.n_head_kv < 1 || c.n_head_kv > 65535 || c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8 != 0) {
        return no.because("%s: %d pages of %d positions, %d heads of %d elements", what, c.n_pages, c.page_size, c.n_head_kv, c.head_dim);
    }
    if (c.page_stride < 0 || c.token_stride < 0 || c.head_stride < 0 || ((c.page_stride | c.token_stride | c.head_stride) & 7)) {
        return no.because("%s: the cache's strides (%lld, %lld, %lld) must be multiples of 8 elements, not negative", what, (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride);
    }
    if (b.n_seq < 0 || b.n_rows < 0 || b.max_rows < 0 || b.table_stride < 0 || b.n_seq >= (1 << 24) || b.n_rows >= (1 << 24)) {
        return no.because("%s: %d sequences, %d rows (most %d), table rows of %d", what, b.n_seq, b.n_rows, b.max_rows, b.table_stride);
    }
    if (b.n_seq > 0 && (b.row_start == nullptr || b.n_kv == nullptr || (b.table_stride > 0 && b.page_table == nullptr) || !aligned_to(b.row_start, 4) || !aligned_to(b.n_kv, 4) || !aligned_to(b.page_table, 4))) {
        return no.because("%s: row_start, n_kv and page_table must be there and 4-byte aligned", what);
    }
    return SPYB_SUCCESS;
}
spyb_status check_append(Refusal &no, const spyb_paged_append_desc &d) {
    const spyb_status st = check_view(no, "paged_append", d.cache, d.batch);
    if (st != SPYB_SUCCESS) { return st; }
    const bool has_q = d.q != nullptr;
    if (!value_type(d.in_type) || (has_q && !value_type(d.q_out_type))) { return no.because("paged_append: input of type %d, Q of type %d", d.in_type, d.q_out_type); }
    if (d.n_head < 0 || d.n_head > 65535 || has_q != (d.n_head > 0)) { return no.because("paged_append: %d query heads, Q %s", d.n_head, has_q ? "given" : "left out"); }
    if (d.k == nullptr || d.v == nullptr || (has_q && d.q_out == nullptr) || !aligned_to(d.q, 16) || !aligned_to(d.k, 16) || !aligned_to(d.v, 16) || (has_q && !aligned_to(d.q_out, 16))) {
        return no.because("paged_append: q, k, v and q_out must be there and 16-byte aligned");
    }
    if (((d.k_stride | d.v_stride | (has_q ? d.q_stride : 0)) & (stride_unit(d.in_type) - 1)) || (has_q && (d.q_out_stride & (stride_unit(d.q_out_type) - 1)))) {
        return no.because("paged_append: row strides must be multiples of 16 bytes");
    }
    if (d.rope_mode != SPYB_ROPE_NONE && d.rope_mode != SPYB_ROPE_PAIRS && d.rope_mode != SPYB_ROPE_HALVES) { return no.because("paged_append: rope mode %d", d.rope_mode); }
    if (d.rope_mode != SPYB_ROPE_NONE && (d.rope_dim < 8 || d.rope_dim > d.cache.head_dim || d.rope_dim % 8 != 0 || !(d.freq_base > 0.f) || !std::isfinite(d.freq_base) || !std::isfinite(d.freq_scale))) {
        return no.because("paged_append: %d rotated elements of %d, base %g, scale %g", d.rope_dim, d.cache.head_dim, d.freq_base, d.freq_scale);
    }
    return SPYB_SUCCESS;
}
spyb_status check_attention(Refusal &no, const spyb_paged_attention_desc &d) {
    const spyb_status st = check_view(no, "paged_attention", d.cache, d.batch);
    if (st != SPYB_SUCCESS) { return st; }
    const int hd = d.cache.head_dim;
    if (hd != 32 && hd != 64 && hd != 96 && hd != 128) { return no.because("paged_attention: heads of %d elements (32, 64, 96 or 128)", hd); }
    if (!value_type(d.out_type)) { return no.because("paged_attention: output of type %d", d.out_type); }
    if (d.n_head < 1 || d.n_head % d.cache.n_head_kv != 0 || d.n_head > 65535) { return no.because("paged_attention: %d query heads over %d K/V heads", d.n_head, d.cache.n_head_kv); }
    if (d.q == nullptr || d.out == nullptr || !aligned_to(d.q, 16) || !aligned_to(d.out, 16) || (d.q_stride & 7) || (d.out_stride & (stride_unit(d.out_type) - 1))) {
        return no.because("paged_attention: q and out must be there and 16-byte aligned, their row strides multiples of 16 bytes");
    }
    if (d.window < 0 || (d.window > 0 && d.causal == 0)) { return no.because("paged_attention: a window of %d positions%s", d.window, d.causal == 0 ? " without causal" : ""); }
    if (!std::isfinite(d.scale)) { return no.because("paged_attention: scale %g", d.scale); }
    if ((int64_t)d.batch.n_rows * (d.n_head / d.cache.n_head_kv) >= (1ll << 30)) { return no.because("paged_attention: %d rows of %d heads", d.batch.n_rows, d.n_head); }
    return SPYB_SUCCESS;
}
PagedView view_of(const spyb_paged_cache &c, const spyb_paged_batch &b) {
    PagedView v;
    v.row_start = b.row_start; v.n_kv = b.n_kv; v.page_table = b.page_table;
    v.n_seq = b.n_seq; v.n_rows = b.n_rows; v.table_stride = b.table_stride; v.n_pages = c.n_pages; v.page_size = c.page_size;
    v.n_kv_most = (int)std::min<int64_t>((int64_t)b.table_stride * c.page_size, 1 << 30);
    v.page_stride = c.page_stride; v.token_stride = c.token_stride; v.head_stride = c.head_stride;
    return v;
}

}  // namespace

// unit `rest` of a sequence whose K/V heads have `one` units each, one tile after the other (paged_plan looks at 32 at a time)
template <int UNIT, int ALIGN> static void paged_find(const PagedAttention &p, const PagedSeq &q, int64_t one, int64_t rest, int &head, int &tile, int &off) {
    head = (int)paged_div(rest, one); rest -= head * one;
    for (tile = 0;; ++tile) {
        const int u = paged_item<UNIT, ALIGN>(p, q, tile).units + p.start_units;
        if (rest < u) { break; }
        rest -= u;
    }
    off = (int)rest;                                      // (of the item with its beginning)
}
// Host check of how the work is cut: on any lengths, also ones that make no sense, the CTAs' pieces cover every unit of every item once, and every CTA of an item has a place of
// its own for what it finds. (Items, shares, cuts and places are the kernels' own functions; where a CTA begins is searched here one by one, by the kernels with all threads.)
// 0 = passed.
template <int UNIT, int ALIGN> static int cut_selftest(uint32_t seed, int tile_rows) {
    auto rnd = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (uint32_t)n); };
    for (int turn = 0; turn < 400; ++turn) {
        const int n_seq = 1 + rnd(12), most_rows = 1 + rnd(turn % 3 == 0 ? 3 : 60), most_kv = 1 + rnd(3000);
        std::vector<int32_t> start(n_seq + 1), kv(n_seq);
        for (int s = 0; s < n_seq; ++s) { start[s + 1] = start[s] + rnd(most_rows + 1); kv[s] = rnd(most_kv) - (turn % 5 == 0 ? most_kv / 2 : 0); }
        if (turn % 7 == 0) { start[rnd(n_seq + 1)] = rnd(200) - 100; }
        PagedAttention p;
        p.view.row_start = start.data(); p.view.n_kv = kv.data(); p.view.n_seq = n_seq; p.view.n_rows = std::max(1, start[n_seq] - rnd(2)); p.view.page_size = 1 + rnd(40);
        p.view.table_stride = 1 + rnd(80); p.view.n_kv_most = p.view.table_stride * p.view.page_size;
        p.n_head_kv = 1 + rnd(5); p.group = 1 + rnd(8); p.tile_rows = tile_rows > 0 ? tile_rows : 2 * (128 / p.group) * p.group; p.causal = rnd(4) != 0; p.window = p.causal && rnd(2) ? 1 + rnd(500) : 0; p.few_rows = rnd(3) == 0 ? 1 << 30 : rnd(40);
        p.start_units = rnd(2) * rnd(5);
        const bool all_seen = p.window > 0 && turn % 4 == 1;   // a window as long as an int can say is none
        if (all_seen) { p.window = paged_window(INT_MAX - rnd(3)); }
        const int grid = 1 + rnd(300), least = 1 + rnd(4);
        for (int few = 0; few < 2; ++few) {
            PagedPlace at = {};
            int64_t total = 0;
            for (int s = 0; s < n_seq; ++s) { total += paged_seq_units<UNIT, ALIGN>(p, s, few) * p.n_head_kv; }
            if (total == 0) { continue; }
            const int ctas = paged_ctas(total, grid, least);
            at.share = paged_share(total, ctas);
            std::vector<uint8_t> seen((size_t)total), real((size_t)total), place((size_t)2 * ctas);
            std::vector<int> arrived(ctas), wanted(ctas);
            for (int c = 0; c < ctas; ++c) {
                at.unit = paged_cta_unit(at.share, c); at.end = paged_cta_unit(at.share, c + 1);
                if (at.unit >= at.end) { return 1; }
                int64_t rest = at.unit;
                int s = 0;
                for (;; ++s) {
                    const int64_t n = s < n_seq ? paged_seq_units<UNIT, ALIGN>(p, s, few) * p.n_head_kv : 0;
                    if (s >= n_seq) { return 2; }
                    if (rest < n) { break; }
                    rest -= n;
                }
                PagedSeq q = paged_seq(p.view, s);
                int head, tile;
                paged_find<UNIT, ALIGN>(p, q, paged_seq_units<UNIT, ALIGN>(p, s, few), rest, head, tile, at.off);
                paged_begin(p, at);
                if (at.unit >= at.end) { continue; }
                int off = at.off;
                for (;;) {
                    const PagedItem it = paged_item<UNIT, ALIGN>(p, q, tile);
                    if (q.row0 < 0 || q.rows < 1 || q.row0 + q.rows > p.view.n_rows || head >= p.n_head_kv || tile * p.tile_rows >= q.rows * p.group) { return 3; }
                    if (all_seen && it.lo != 0) { return 14; }
                    if (it.lo < 0 || it.lo % ALIGN != 0 || it.hi > p.view.n_kv_most || off >= it.units || (int64_t)it.units * UNIT + it.lo < it.hi) { return 4; }
                    const int todo = (int)std::min<int64_t>(it.units - off, at.end - at.unit);
                    const PagedCut cut = paged_cut(at, at.unit - off, it.units);
                    if ((cut.parts == 1) != (todo == it.units) || cut.c0 < 0 || cut.c0 + cut.parts > ctas || c < cut.c0 || c >= cut.c0 + cut.parts) { return 5; }
                    if (cut.parts > 1) {
                        if (place[(size_t)paged_slot(c, cut.c0)]++) { return 6; }
                        if ((c == cut.c0) != (off == 0)) { return 7; }
                        ++arrived[cut.c0]; wanted[cut.c0] = cut.parts;
                    }
                    if (at.unit - off + it.units > total) { return 12; }
                    for (int u = 0; u < it.units; ++u) { real[(size_t)(at.unit - off + u)] = 1; }
                    for (int u = 0; u < todo; ++u) { if (seen[(size_t)(at.unit + u)]++) { return 8; } }
                    at.unit += todo + p.start_units;
                    if (at.unit >= at.end) { break; }
                    off = 0;
                    if (!paged_next(p, few, q, s, head, tile)) { return 9; }
                }
            }
            int64_t items = 0, work = 0;
            for (int s = 0; s < n_seq; ++s) {
                const PagedSeq q = paged_seq(p.view, s);
                if (paged_mine(p, q, few)) { items += (int64_t)((q.rows * p.group + p.tile_rows - 1) / p.tile_rows) * p.n_head_kv; }
            }
            for (size_t u = 0; u < seen.size(); ++u) { work += seen[u]; if (seen[u] != real[u]) { return 10; } }
            if (work != total - items * p.start_units) { return 13; }
            for (int c = 0; c < ctas; ++c) { if (arrived[c] != wanted[c]) { return 11; } }
        }
    }
    return 0;
}
int paged_cut_selftest() {
    int bad = cut_selftest<64, 16>(1, 16);
    if (bad == 0) { bad = cut_selftest<64, 16>(2, 32); }
    if (bad == 0) { bad = cut_selftest<128, 128>(3, 0); }
    return bad == 0 ? 0 : 100 + bad;
}

}  // namespace spyb

using namespace spyb;

// The public call, and with a role that is late the self-checks'
static spyb_status paged_attention(spyb_backend *be, const spyb_paged_attention_desc &desc, int late, uint64_t wait_limit) {
    const spyb_paged_attention_desc *d = &desc;
    Refusal no;
    if (check_attention(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->batch.n_seq == 0 || d->batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    if (!be->paged_workspace()) { return SPYB_FAIL; }
    const int hd = d->cache.head_dim;
    PagedAttention p;
    p.view = view_of(d->cache, d->batch);
    p.q = static_cast<const __half *>(d->q); p.out = d->out;
    p.k = static_cast<const __half *>(d->cache.k); p.v = static_cast<const __half *>(d->cache.v);
    p.q_stride = d->q_stride; p.out_stride = d->out_stride; p.n_head_kv = d->cache.n_head_kv; p.group = d->n_head / d->cache.n_head_kv;
    p.causal = d->causal != 0; p.window = paged_window(d->window); p.out_f32 = d->out_type == SPYB_FP32;
    const float scale = d->scale == 0.f ? 1.0f / std::sqrt((float)hd) : d->scale;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634073599);
    p.late = late; p.partial = be->paged_partial; p.arrived = be->paged_arrived;
    const int64_t most = (int64_t)(d->batch.max_rows > 0 ? std::min(d->batch.max_rows, d->batch.n_rows) : d->batch.n_rows) * p.group;
    const LaunchCfg cfg = be->launch_cfg(be->config.use_pdl != 0);
    p.few_rows = 1 << 30;
    if (most > PA_FEW_ROWS && scale >= 0.f) {
        cudaError_t err = cudaSuccess;
        p.few_rows = p.view.n_seq == 1 ? 0 : PA_FEW_ROWS;
        if (!launch_paged_attention_tc(p, hd, d->n_head, be->num_sms_total, cfg, wait_limit, &err)) { p.few_rows = 1 << 30; }
        SPYB_CUDA(be, err);
    }
    const int row_tiles = std::min<int64_t>(most, p.few_rows) <= 16 ? 1 : 2;
    p.tile_rows = 16 * row_tiles;
    if (p.few_rows > 0) { SPYB_CUDA(be, launch_paged_attention_rows(p, hd, row_tiles, be->num_sms_total, cfg)); }
    return SPYB_SUCCESS;
}

extern "C" {

spyb_status spyb_paged_append_check(const spyb_paged_append_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_append(no, *d), message, size);
}
spyb_status spyb_paged_attention_check(const spyb_paged_attention_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_attention(no, *d), message, size);
}

spyb_status spyb_paged_append(spyb_backend *be, const spyb_paged_append_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_append(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->batch.n_seq == 0 || d->batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    PagedAppend p;
    p.view = view_of(d->cache, d->batch);
    p.q = d->q; p.k = d->k; p.v = d->v; p.q_out = d->q_out;
    p.k_cache = static_cast<__half *>(d->cache.k); p.v_cache = static_cast<__half *>(d->cache.v);
    p.q_stride = d->q_stride; p.k_stride = d->k_stride; p.v_stride = d->v_stride; p.q_out_stride = d->q_out_stride;
    p.n_head = d->n_head; p.n_head_kv = d->cache.n_head_kv; p.head_dim = d->cache.head_dim;
    if (d->rope_mode != SPYB_ROPE_NONE) {
        // the shares of a circle of one setting are kept: every layer of every step asks for the same ones
        auto &t = be->paged_turns;
        if (t.base != d->freq_base || t.scale != d->freq_scale || t.rot != d->rope_dim) {
            for (int i = 0; i < d->rope_dim / 2; ++i) { t.turns[i] = (double)d->freq_scale * std::pow((double)d->freq_base, -2.0 * i / d->rope_dim) / 6.283185307179586476925286766559; }
            t.base = d->freq_base; t.scale = d->freq_scale; t.rot = d->rope_dim;
        }
        p.rot = d->rope_dim; p.halves = d->rope_mode == SPYB_ROPE_HALVES;
        std::copy(t.turns, t.turns + d->rope_dim / 2, p.turns);
    }
    SPYB_CUDA(be, launch_paged_append(p, d->in_type, d->q_out_type, be->num_sms_total, be->launch_cfg(be->config.use_pdl != 0)));
    return SPYB_SUCCESS;
}

spyb_status spyb_paged_attention(spyb_backend *be, const spyb_paged_attention_desc *d) {
    return be == nullptr || d == nullptr ? SPYB_FAIL : paged_attention(be, *d, PA_ON_TIME, be->wait_limit_ns);
}

// Self-check of the tensor-memory kernel's hand-overs: a chunk at the end of a long conversation and a short one, on time and with one of its roles late. A role that is late within
// the limit of the waits changes nothing; copies that come three limits late make waits give up: the kernel ends by itself, when they have landed, says so, and leaves nothing for
// the next launch.
spyb_status spyb_paged_selftest_late(spyb_backend *be, int32_t who, uint64_t limit_ns, int32_t *error_code_out) {
    if (be == nullptr || limit_ns == 0 || who < PA_LATE_CHECKS || who > PA_LATE_Q) { return SPYB_FAIL; }
    use_device(be->config.device_id);
    SPYB_CUDA(be, cudaStreamSynchronize(be->stream));
    if (be->device_error()) { return SPYB_FAIL; }
    constexpr int heads = 2, group = 3, page = 16, pages = 1300, rows[2] = {300, 70}, kv[2] = {20000, 70}, n_rows = rows[0] + rows[1];
    const int32_t words[5] = {0, rows[0], n_rows, kv[0], kv[1]};
    std::vector<int32_t> table(2 * pages);
    for (int i = 0; i < 2 * pages; ++i) { table[i] = i % pages; }
    int code = 0;
    for (const int hd : {64, 128}) {
        const size_t n_pool = (size_t)pages * page * heads * hd, n_q = (size_t)n_rows * heads * group * hd;
        std::vector<uint16_t> host(2 * n_pool + n_q);
        uint32_t seed = 1;
        for (uint16_t &x : host) { seed = seed * 1664525u + 1013904223u; x = (uint16_t)(0x3000 + (seed >> 18) % 0x0c00 + (seed & 0x80000000u ? 0x8000 : 0)); }   // 0.125 to 1, either sign
        std::vector<float> want(n_q), got(n_q);
        uint8_t *mem = nullptr;
        const size_t at_out = host.size() * 2, at_words = at_out + n_q * 4, at_table = at_words + sizeof words, size = at_table + table.size() * 4;
        SPYB_CUDA(be, cudaMalloc(&mem, size));
        spyb_paged_attention_desc d = {};
        d.cache.k = mem; d.cache.v = mem + n_pool * 2; d.cache.number_type = SPYB_FP16; d.cache.n_pages = pages; d.cache.page_size = page; d.cache.n_head_kv = heads; d.cache.head_dim = hd;
        d.cache.page_stride = page * heads * hd; d.cache.token_stride = heads * hd; d.cache.head_stride = hd;
        d.batch.row_start = reinterpret_cast<int32_t *>(mem + at_words); d.batch.n_kv = d.batch.row_start + 3; d.batch.page_table = reinterpret_cast<int32_t *>(mem + at_table);
        d.batch.n_seq = 2; d.batch.n_rows = n_rows; d.batch.table_stride = pages;
        d.q = mem + n_pool * 4; d.out = mem + at_out; d.q_stride = d.out_stride = heads * group * hd; d.n_head = heads * group; d.out_type = SPYB_FP32; d.causal = 1;
        cudaError_t err = upload(mem, host.data(), host.size() * 2);
        if (err == cudaSuccess) { err = upload(mem + at_words, words, sizeof words); }
        if (err == cudaSuccess) { err = upload(mem + at_table, table.data(), table.size() * 4); }
        spyb_status st = SPYB_SUCCESS;
        auto run = [&](int late, uint64_t limit, std::vector<float> &to) {
            if (err == cudaSuccess) { err = cudaMemsetAsync(d.out, 0xff, n_q * 4, be->stream); }
            if (err == cudaSuccess && st == SPYB_SUCCESS) { st = paged_attention(be, d, late, limit); }
            if (err == cudaSuccess) { err = cudaMemcpyAsync(to.data(), d.out, n_q * 4, cudaMemcpyDeviceToHost, be->stream); }
            if (err == cudaSuccess) { err = cudaStreamSynchronize(be->stream); }   // returns: the kernels ended by themselves
            return be->clear_device_error();
        };
        const int expected = who == PA_LATE_CHECKS ? 0 : 7, before = run(PA_ON_TIME, be->wait_limit_ns, want);
        int after = 0;
        if (before == 0) { code = run(who, limit_ns, got); }
        if (expected != 0) { after = run(PA_ON_TIME, be->wait_limit_ns, got); }
        cudaFree(mem);
        SPYB_CUDA(be, err);
        if (st != SPYB_SUCCESS) { return st; }
        if (error_code_out != nullptr) { *error_code_out = code; }
        if (before != 0 || code != expected || after != 0) { be->set_error("paged selftest: heads of %d: codes %d, %d, %d where 0, %d, 0 were expected", hd, before, code, after, expected); return SPYB_FAIL; }
        if (std::memcmp(want.data(), got.data(), n_q * 4) != 0) { be->set_error("paged selftest: heads of %d: a late role changed the output, its own or the next launch's", hd); return SPYB_FAIL; }
    }
    return SPYB_SUCCESS;
}

}  // extern "C"
