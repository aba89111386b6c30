// Caches in pages, what goes beyond fp16 ones whose sequences have nothing in common: storing with norms and in bytes, reading back, who shares what, and the kernels of attention of few rows
// that are built for these.

#include <algorithm>

#include "spyb_internal.h"
#include "spyb_paged.cuh"
#include "spyb_paged_rows.cuh"

namespace spyb {
namespace {

struct RowPlace { int64_t cell, pair; int pos; bool mine; };        // of a row: where its position lies (cell -1: not there) and its scales; mine: a sequence's
__device__ __forceinline__ RowPlace row_place(const PagedView &v, const PagedScales &scales, int row) {   // by one thread
    RowPlace a = {-1, 0, -1, false};
    if (row >= v.n_rows) { return a; }
    int q = -1, n = v.n_seq + 1;                                    // the last one that begins at the row or in front of it
    for (int lo = 0; n > 0;) {
        const int half = n / 2;
        if (v.row_start[lo + half] <= row) { q = lo + half; lo += half + 1; n -= half + 1; } else { n = half; }
    }
    if (q < 0 || q >= v.n_seq) { return a; }
    const int end = v.row_start[q + 1];
    a.pos = v.n_kv[q] - end + row; a.mine = row < end;
    if (a.mine && a.pos >= 0 && a.pos < v.n_kv_most) {
        const int page = v.page_table[(int64_t)q * v.table_stride + a.pos / v.page_size], at = a.pos % v.page_size;
        if (page >= 0 && page < v.n_pages) { a.cell = page * v.page_stride + at * v.token_stride; a.pair = page * scales.page_stride + at * scales.token_stride; }
    }
    return a;
}
__device__ __forceinline__ void store8(float *p, const float *v) { store4(p, v); store4(p + 4, v + 4); }
__device__ __forceinline__ void store8(__half *p, const float *v) { *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])); }

// ---------------------------------------------------------------------------------------------- store
// An element is read once (4 or 2 bytes) and written once (2, or 1 and a 64th of a scale); beside that the instructions count, some 100 for eight elements, so all that can be done once is: a CTA has up to
// ST_ROWS rows, whose places a lane each finds; their cosines and sines are made a pair a thread and go through shared memory; a thread has eight elements of a head in all of these rows, so that kinds of heads, weights and
// addresses are found once a head. A head's threads lie side by side in a warp (as many as the next power of two): the mean of squares and the largest magnitude are shuffles.
// An element is rounded once: norm, rotation and scale are f32, angles 64 bits.
constexpr int ST_THREADS = 256, ST_ROWS = 8;
struct StorePlace { int pos; int64_t cell, pair; };                 // pos -1: nobody's row, or one in front of position 0; cell -1: its page is not there
__device__ __forceinline__ float larger(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float one_over(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }   // (off by a step at most)
// x / scale to the nearest whole number, a half to the even one. A product with the reciprocal may be wrong beside a half; what is left over of x then says which it is, without an error: x - q scale, at most
// half a scale or a bit more, is a multiple of x's last place or of the scale's (11 bits), which 24 bits hold
__device__ __forceinline__ float nearest_byte(float x, float scale, float per_one) {
    const float q = rintf(x * per_one), left = fmaf(-q, scale, x), twice = 2.f * fabsf(left);
    const bool odd = ((int)q & 1) != 0;
    return twice > scale || (twice == scale && odd) ? q + copysignf(1.f, left) : q;
}

template <class TIn, class TQ, bool EIGHT, bool HALVES>
__global__ void __launch_bounds__(ST_THREADS, 4) paged_store_kernel(const __grid_constant__ PagedStore s, const int width, const int rows_each) {
    const PagedAppend &p = s.append;
    __shared__ __align__(16) float2 turn[ST_ROWS][128];             // cosine and sine of a pair
    __shared__ StorePlace places[ST_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int row0 = blockIdx.x * rows_each, rows = min(rows_each, p.view.n_rows - row0);
    const int per = p.head_dim / 8, slots = ST_THREADS / width;     // threads of a head that have elements, heads at a time
    const int slot = threadIdx.x / width, item = threadIdx.x & (width - 1), total = p.n_head + 2 * p.n_head_kv, keys_end = p.n_head + p.n_head_kv;
    const bool turned = item < p.rot / 8;
    const int  e0 = HALVES && turned ? 4 * item : 8 * item, e1 = HALVES && turned ? e0 + p.rot / 2 : e0 + 4;
    struct Head { const TIn *src; int64_t stride; bool is_q, is_k, mine; int hh; };
    auto head_of = [&](int h) {
        Head a;
        a.is_q = h < p.n_head; a.is_k = !a.is_q && h < keys_end; a.mine = item < per && h < total;
        a.hh = a.is_q ? h : a.is_k ? h - p.n_head : h - keys_end;
        a.stride = a.is_q ? p.q_stride : a.is_k ? p.k_stride : p.v_stride;
        a.src = static_cast<const TIn *>(a.is_q ? p.q : a.is_k ? p.k : p.v) + row0 * a.stride + (int64_t)a.hh * p.head_dim;
        return a;
    };
    auto fetch = [&](const Head &a, int r, float (&x)[8]) {
        if (a.mine && r < rows) { load4(a.src + r * a.stride + e0, x); load4(a.src + r * a.stride + e1, x + 4); }
    };
    // (the first head's elements are on their way while the rows' places are found)
    int  h0 = blockIdx.y * slots;                                   // (the same for all threads: they meet in shuffles)
    Head head = head_of(h0 + slot);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    fetch(head, 0, x);
    if (threadIdx.x < rows) {
        const RowPlace at = row_place(p.view, s.scales, row0 + threadIdx.x);
        places[threadIdx.x] = {at.mine ? at.pos : -1, at.cell, at.pair};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (p.rot / 2); i += ST_THREADS) {
        const int r = i / (p.rot / 2), k = i - r * (p.rot / 2);
        const double t = (double)places[r].pos * p.turns[k];
        sincospif(2.0f * (float)(t - rint(t)), &turn[r][k].y, &turn[r][k].x);
    }
    __syncthreads();
    const float mean = 1.f / (float)p.head_dim;
    for (;;) {
        const float *weight = head.is_q ? s.q_norm : head.is_k ? s.k_norm : nullptr;
        const bool some_norm = (h0 < p.n_head && s.q_norm != nullptr) || (h0 < keys_end && h0 + slots > p.n_head && s.k_norm != nullptr), some_cache = h0 + slots > p.n_head;   // of the CTA's heads
        float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (weight != nullptr && head.mine) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(weight + e0)), c = __ldg(reinterpret_cast<const float4 *>(weight + e1));
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
        }
        const int64_t to = head.is_q ? (int64_t)row0 * p.q_out_stride + (int64_t)head.hh * p.head_dim : head.hh * p.view.head_stride;
        for (int r = 0; r < rows; ++r) {
            float ahead[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};   // (a lane without elements takes part in its head's sum and maximum with zeros)
            fetch(head, r + 1, ahead);
            const StorePlace at = places[r];
            if (some_norm) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) { sum = fmaf(x[i], x[i], sum); }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) { if (o < width) { sum += __shfl_xor_sync(0xffffffffu, sum, o); } }
                if (weight != nullptr) {
                    const float f = rsqrtf(fmaf(sum, mean, s.eps));
#pragma unroll
                    for (int i = 0; i < 8; ++i) { x[i] = x[i] * f * w[i]; }
                }
            }
            if (turned && (head.is_q || head.is_k)) {
                const float4 c0 = *reinterpret_cast<const float4 *>(&turn[r][4 * item]), c1 = *reinterpret_cast<const float4 *>(&turn[r][4 * item + 2]);
                const float co[4] = {c0.x, c0.z, c1.x, c1.z}, si[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    constexpr int STEP = HALVES ? 1 : 2, SECOND = HALVES ? 4 : 1;
                    const float u = x[STEP * i], v = x[STEP * i + SECOND];
                    x[STEP * i] = u * co[i] - v * si[i];
                    x[STEP * i + SECOND] = u * si[i] + v * co[i];
                }
            }
            float most = 0.f;
            if (EIGHT && some_cache) {
#pragma unroll
                for (int i = 0; i < 8; ++i) { most = larger(most, fabsf(x[i])); }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) { if (o < width) { most = larger(most, __shfl_xor_sync(0xffffffffu, most, o)); } }
            }
            if (head.is_q) {
                if (head.mine && at.pos >= 0) {
                    TQ *dst = static_cast<TQ *>(p.q_out) + r * p.q_out_stride + to;
                    store4(dst + e0, x); store4(dst + e1, x + 4);
                }
            } else if (head.mine && at.pos >= 0 && at.cell >= 0) {
                if constexpr (EIGHT) {
                    const bool   fine = most <= 65468.f;
                    const __half scale = fine ? __float2half_ru(__fdiv_rn(most, 127.f)) : __ushort_as_half(0x7fff);
                    const float  per_one = fine && most > 0.f ? one_over(__half2float(scale)) : 0.f;
                    // (two products, 2^-21 to either side: where they agree, which is nearly always, that is the nearest. 1.5 x 2^23: the integer is the low byte. Beside a scale that is NaN the bytes are any)
                    const float  more = per_one * (1.f + 0x1p-21f), less = per_one * (1.f - 0x1p-21f), ones = 12582912.f;
                    uint8_t *dst = (head.is_k ? s.k8 : s.v8) + at.cell + to;
                    uint32_t b[8], differ = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) { b[i] = __float_as_uint(fmaf(x[i], more, ones)); differ |= b[i] ^ __float_as_uint(fmaf(x[i], less, ones)); }
                    if (differ != 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) { b[i] = __float_as_uint(nearest_byte(x[i], __half2float(scale), per_one) + ones); }
                    }
                    *reinterpret_cast<uint32_t *>(dst + e0) = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
                    *reinterpret_cast<uint32_t *>(dst + e1) = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
                    if (item == 0) { reinterpret_cast<__half *>(const_cast<uint32_t *>(s.scales.pairs))[2 * (at.pair + head.hh * s.scales.head_stride) + (head.is_k ? 0 : 1)] = scale; }
                } else {
                    __half *dst = (head.is_k ? p.k_cache : p.v_cache) + at.cell + to;
                    store4(dst + e0, x); store4(dst + e1, x + 4);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = ahead[i]; }
        }
        h0 += slots * gridDim.y;
        if (h0 >= total) { break; }
        head = head_of(h0 + slot);
#pragma unroll
        for (int i = 0; i < 8; ++i) { x[i] = 0.f; }
        fetch(head, 0, x);
    }
}

// ---------------------------------------------------------------------------------------------- load
// Memory bound: a byte (or two) read and two (or four) written an element. A CTA has 32 rows, whose places the lanes of its first warp find, one each (four dependent loads, which as many rows share); a thread
// has eight elements of one head in all of them.
constexpr int LD_THREADS = 256;

template <class T, bool EIGHT, int LD_ROWS>
__global__ void __launch_bounds__(LD_THREADS) paged_load_kernel(const __grid_constant__ PagedLoad p) {
    __shared__ int64_t cells[LD_ROWS], pairs[LD_ROWS];             // -1: nothing there; -2: nobody's row
    pdl_launch_dependents();
    pdl_wait();
    const int row0 = blockIdx.x * LD_ROWS;
    if (threadIdx.x < LD_ROWS) {
        const RowPlace at = row_place(p.view, p.scales, row0 + threadIdx.x);
        cells[threadIdx.x] = at.mine ? at.cell : -2; pairs[threadIdx.x] = at.pair;
    }
    __syncthreads();
    const int per = p.head_dim / 8, each = p.n_head_kv * per, first = p.k_out != nullptr ? 0 : each, items = (p.v_out != nullptr ? 2 * each : each) - first;
    const int sub = items < LD_THREADS ? threadIdx.x / items : 0, rows_at_once = items < LD_THREADS ? LD_THREADS / items : 1;
    if (sub >= rows_at_once) { return; }
    for (int it = threadIdx.x - sub * items; it < items; it += LD_THREADS) {
        const int i = it + first, is_v = i >= each, j = i - (is_v ? each : 0), head = j / per, e = (j - head * per) * 8;
        const int64_t in = head * p.view.head_stride + e, out = head * p.head_dim + e, stride = is_v ? p.v_stride : p.k_stride;
        T *dst = static_cast<T *>(is_v ? p.v_out : p.k_out) + (int64_t)row0 * stride + out;
        const int64_t of_pair = head * p.scales.head_stride;
        constexpr int TOGETHER = 4;                                 // rows whose bytes are on their way at a time
        for (int r0 = sub; r0 < LD_ROWS; r0 += TOGETHER * rows_at_once) {
            uint4    w[TOGETHER];
            uint32_t pair[TOGETHER];
            int64_t  cell[TOGETHER];
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                const int r = r0 + k * rows_at_once;
                cell[k] = r < LD_ROWS ? cells[r] : -2;
                if (cell[k] >= 0) {
                    if constexpr (EIGHT) {
                        const uint2 y = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(is_v ? p.v : p.k) + cell[k] + in));
                        w[k].x = y.x; w[k].y = y.y;
                        pair[k] = p.scales.pairs[pairs[r] + of_pair];
                    } else { w[k] = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const __half *>(is_v ? p.v : p.k) + cell[k] + in)); }
                }
            }
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                const int r = r0 + k * rows_at_once;
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (cell[k] >= 0) {
                    uint32_t h[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                    float scale = 1.f;
                    if constexpr (EIGHT) {
                        const float2 s = half2_bits(pair[k]);
                        scale = is_v ? s.y : s.x;
                        halves_of(w[k].x, h[0], h[1]); halves_of(w[k].y, h[2], h[3]);
                    }
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) { const float2 u = half2_bits(h[i4]); x[2 * i4] = EIGHT ? u.x * scale : u.x; x[2 * i4 + 1] = EIGHT ? u.y * scale : u.y; }
                }
                if (cell[k] != -2) { store8(dst + r * stride, x); }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- who shares what
// A warp for each sequence: its group, what all of the group's sequences that have rows see whole, and the first of these, which stands for all in the first pass.
// Groups and beginnings of rows are the caller's, on the device: where they are not ascending, a sequence may find a group that its first sequence is not in, or have rows that are not among that one's in the
// first pass. Such a sequence shares nothing, so that a row whose sequence has a `from` is a row of the first pass.
constexpr int SH_WARPS = 8;
__global__ void __launch_bounds__(SH_WARPS * 32) paged_shared_kernel(const __grid_constant__ PagedShared p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, s = blockIdx.x * SH_WARPS + (threadIdx.x >> 5), n_seq = p.view.n_seq;
    if (s >= n_seq) { return; }
    PagedView groups;                                               // (sequence_of's search, over groups)
    groups.row_start = p.group_start; groups.n_seq = p.n_group;
    const int g = sequence_of(groups, s);
    int common = 0, leader = -1, with_rows = 0, group_end = 0;
    if (g >= 0 && g < p.n_group && s < p.group_start[g + 1]) {
        const int a = max(0, p.group_start[g]);
        group_end = min(n_seq, p.group_start[g + 1]);
        common = min(max(0, p.n_shared[g]), p.view.n_kv_most);
        leader = n_seq;
        for (int i = a + lane; i < group_end; i += 32) {
            const PagedSeq q = paged_seq(p.view, i);
            if (q.rows > 0) {
                common = min(common, max(0, p.causal ? min(q.first, q.kv) : q.kv));
                leader = min(leader, i);
                ++with_rows;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            common = min(common, __shfl_xor_sync(0xffffffffu, common, o));
            leader = min(leader, __shfl_xor_sync(0xffffffffu, leader, o));
            with_rows += __shfl_xor_sync(0xffffffffu, with_rows, o);
        }
        common = with_rows > 1 && common >= PA_SHARED ? common / p.align * p.align : 0;
        if (common > 0) {                                           // (the same for all lanes)
            const int32_t *start = p.view.row_start;
            const int end = start[group_end];
            if (sequence_of(groups, leader) != g || start[leader + 1] > end || start[s] < start[leader] || start[s + 1] > end) { common = 0; }
        }
    }
    if (lane == 0) {
        const int begin = p.view.row_start[s];
        p.from[s] = common;
        p.kv[s] = common;
        p.row_end[s] = s == leader && common > 0 ? p.view.row_start[group_end] : begin;
        p.lead[s] = common > 0 ? p.view.row_start[leader] : begin;
    }
}

// Rows of two query heads a warp: the pieces of their tiles that the first pass's CTAs left, joined in their order. (In the first pass itself one CTA would have to read them all, 18 pieces of 64 KB where 64 requests
// share 6000 positions: 25 us of its 51.) A piece has its rows side by side, four elements of each: two rows are what a sector of memory holds.
constexpr int SJ_WARPS = 8, SJ_TILE = 128;    // (rows of a tile of the tensor-memory kernel)
template <int HD>
__global__ void __launch_bounds__(SJ_WARPS * 32) paged_shared_join_kernel(const __grid_constant__ PagedSharedJoin p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, n_head = p.n_head_kv * p.group;
    const int64_t cell = ((int64_t)blockIdx.x * SJ_WARPS + (threadIdx.x >> 5)) * 2 + (lane & 1);
    const int row = (int)(cell / n_head), head = (int)(cell - (int64_t)row * n_head), kv = (int)((unsigned)head / (unsigned)p.group);
    if (row >= p.view.n_rows) { return; }
    int s = -1, n = p.view.n_seq + 1;                               // the last one that begins at the row or in front of it
    for (int lo = 0; n > 0;) {
        const int half = n / 2;
        if (p.view.row_start[lo + half] <= row) { s = lo + half; lo += half + 1; n -= half + 1; } else { n = half; }
    }
    if (s < 0 || s >= p.view.n_seq || row >= p.view.row_end[s] || p.from[s] == 0) { return; }
    const int lead = max(0, p.lead[s]), tokens = SJ_TILE / p.group, half = (int)((unsigned)(row - lead) / (unsigned)tokens), first = lead + half * tokens;
    if (row < lead) { return; }                                     // (no group that makes sense)
    const int2 cut = p.cuts[(int64_t)kv * p.view.n_rows + first];
    if (cut.y < 2 || cut.x < 0 || cut.x > p.ctas - cut.y) { return; }   // (a pass that gave up may have left any word there; pieces are read from places of CTAs alone)
    const int r = (row - first) * p.group + head - kv * p.group;
    constexpr int PIECE = SJ_TILE * (HD + 2), FOURS = HD / 64;      // of a lane: four elements, 64 apart
    const float *const place = p.partial + (half & 1) * PIECE;
    float  m = -INFINITY, l = 0.f;
    float4 v[FOURS];
#pragma unroll
    for (int c = 0; c < FOURS; ++c) { v[c] = make_float4(0.f, 0.f, 0.f, 0.f); }
#pragma unroll 1
    for (int i0 = 0; i0 < cut.y; i0 += 8) {                         // eight pieces are in flight together; what came before is scaled to the new maximum
        float  pm[8], pl[8], top = m;
        float4 u[8][FOURS];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool is = i0 + j < cut.y;
            const float *from = place + paged_slot(cut.x + (is ? i0 + j : 0), cut.x) * 2 * PIECE;
            pm[j] = is ? __ldcg(from + SJ_TILE * HD + r) : -INFINITY;
            pl[j] = is ? __ldcg(from + SJ_TILE * HD + SJ_TILE + r) : 0.f;
#pragma unroll
            for (int c = 0; c < FOURS; ++c) { u[j][c] = is ? __ldcg(reinterpret_cast<const float4 *>(from) + (16 * c + lane / 2) * SJ_TILE + r) : make_float4(0.f, 0.f, 0.f, 0.f); }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) { top = fmaxf(top, pm[j]); }
        const float base = top == -INFINITY ? 0.f : top, before = exp2f(m - base);
        m = top; l *= before;
#pragma unroll
        for (int c = 0; c < FOURS; ++c) { v[c] = make_float4(v[c].x * before, v[c].y * before, v[c].z * before, v[c].w * before); }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = exp2f(pm[j] - base);
            l += f * pl[j];
#pragma unroll
            for (int c = 0; c < FOURS; ++c) { v[c].x += f * u[j][c].x; v[c].y += f * u[j][c].y; v[c].z += f * u[j][c].z; v[c].w += f * u[j][c].w; }
        }
    }
#pragma unroll
    for (int c = 0; c < FOURS; ++c) { reinterpret_cast<float4 *>(p.out + cell * HD)[16 * c + lane / 2] = v[c]; }
    if (lane < 2) { p.stats[cell] = make_float2(m, l); }
}

template <int ROWS>
cudaError_t launch_load(const PagedLoad &p, int out_type, const LaunchCfg &cfg) {
    const auto kernel = p.scales.pairs != nullptr ? (out_type == SPYB_FP32 ? paged_load_kernel<float, true, ROWS> : paged_load_kernel<__half, true, ROWS>)
                                                  : out_type == SPYB_FP32 ? paged_load_kernel<float, false, ROWS> : paged_load_kernel<__half, false, ROWS>;
    return launch_maybe_pdl(kernel, dim3((p.view.n_rows + ROWS - 1) / ROWS), LD_THREADS, 0, cfg.stream, cfg.pdl, p);
}
template <class TIn, class TQ, bool EIGHT>
cudaError_t launch_store(const PagedStore &p, int sms, const LaunchCfg &cfg) {
    int width = 1;
    while (width < p.append.head_dim / 8) { width *= 2; }
    const int total = p.append.n_head + 2 * p.append.n_head_kv, slots = ST_THREADS / width, loops = (total + slots - 1) / slots;
    // few rows: a row's heads are spread over CTAs; many: several rows a CTA, as long as there are CTAs for four an SM
    const int n_rows = p.append.view.n_rows, each = std::max(1, std::min(ST_ROWS, n_rows / (4 * sms))), split = std::max(1, std::min(loops, 2 * sms / std::max(1, n_rows)));
    const auto kernel = p.append.halves ? paged_store_kernel<TIn, TQ, EIGHT, true> : paged_store_kernel<TIn, TQ, EIGHT, false>;
    return launch_maybe_pdl(kernel, dim3((n_rows + each - 1) / each, split), ST_THREADS, 0, cfg.stream, cfg.pdl, p, width, each);
}
template <class TIn, class TQ>
cudaError_t launch_store(const PagedStore &p, int sms, const LaunchCfg &cfg) {
    return p.scales.pairs != nullptr ? launch_store<TIn, TQ, true>(p, sms, cfg) : launch_store<TIn, TQ, false>(p, sms, cfg);
}

}  // namespace

cudaError_t launch_paged_store(const PagedStore &p, int in_type, int q_out_type, int sms, const LaunchCfg &cfg) {
    if (in_type == SPYB_FP32) { return q_out_type == SPYB_FP32 ? launch_store<float, float>(p, sms, cfg) : launch_store<float, __half>(p, sms, cfg); }
    return q_out_type == SPYB_FP32 ? launch_store<__half, float>(p, sms, cfg) : launch_store<__half, __half>(p, sms, cfg);
}
cudaError_t launch_paged_load(const PagedLoad &p, int out_type, int sms, const LaunchCfg &cfg) {
    // (few rows: on as many CTAs as there are. 1 of 300, before the loads were made together: 5.2 us with eight rows each, 8.6 with 32; 4.1 now)
    return p.view.n_rows >= 32 * 4 * sms ? launch_load<32>(p, out_type, cfg) : launch_load<8>(p, out_type, cfg);
}
cudaError_t launch_paged_shared(const PagedShared &p, const LaunchCfg &cfg) {
    return launch_maybe_pdl(paged_shared_kernel, dim3((p.view.n_seq + SH_WARPS - 1) / SH_WARPS), SH_WARPS * 32, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_shared_join(const PagedSharedJoin &p, int head_dim, const LaunchCfg &cfg) {
    const int64_t cells = (int64_t)p.view.n_rows * p.n_head_kv * p.group;
    return launch_maybe_pdl(head_dim == 128 ? paged_shared_join_kernel<128> : paged_shared_join_kernel<64>, dim3((unsigned)((cells + 2 * SJ_WARPS - 1) / (2 * SJ_WARPS))), SJ_WARPS * 32, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_shared_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg) { return launch_rows_kind<PK_SHARED>(p, head_dim, row_tiles, sms, cfg); }

}  // namespace spyb
