// Caches in pages, what goes beyond fp16 ones whose sequences have nothing in common: storing with norms and in bytes, reading back, who shares what, and the kernels of attention of few rows
// that are built for these.

#include <algorithm>

#include "spyb_internal.h"
#include "spyb_paged.cuh"
#include "spyb_paged_rows.cuh"

namespace spyb {
namespace {

// ---------------------------------------------------------------------------------------------- store
// Memory bound, as append: an element is read once (4 or 2 bytes) and written once (2, or 1 and a 64th of a scale). A CTA has one row; a head's threads, eight elements each, lie side by side in
// a warp (as many as the next power of two), so that the mean of squares and the largest magnitude are shuffles. An element is rounded once: norm, rotation and scale are f32, angles 64 bits.
constexpr int ST_THREADS = 256;

template <class TIn, class TQ, bool EIGHT, bool AHEAD>
__global__ void __launch_bounds__(ST_THREADS) paged_store_kernel(const __grid_constant__ PagedStore s, const int width) {
    const PagedAppend &p = s.append;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    const int per = p.head_dim / 8, slots = ST_THREADS / width;     // threads of a head that have elements, heads at a time
    const int slot = threadIdx.x / width, item = threadIdx.x & (width - 1), total = p.n_head + 2 * p.n_head_kv;
    const bool turned = item < p.rot / 8;
    const int  e0 = turned && p.halves ? 4 * item : 8 * item, e1 = turned && p.halves ? e0 + p.rot / 2 : e0 + 4;
    const int  step = slots * gridDim.y;
    auto fetch = [&](int head, float (&x)[8]) {
        const bool is_q = head < p.n_head, is_k = !is_q && head < p.n_head + p.n_head_kv;
        const int  hh = is_q ? head : is_k ? head - p.n_head : head - p.n_head - p.n_head_kv;
        const TIn *src = static_cast<const TIn *>(is_q ? p.q : is_k ? p.k : p.v) + row * (is_q ? p.q_stride : is_k ? p.k_stride : p.v_stride) + (int64_t)hh * p.head_dim;
        load4(src + e0, x);
        load4(src + e1, x + 4);
    };
    auto works = [&](int h) { return item < per && h < total; };
    // (the first head's elements are on their way while the row's place is found)
    int   h0 = blockIdx.y * slots;                                  // (the same for all threads: they meet in shuffles)
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, q_weight[8], k_weight[8];
    if (works(h0 + slot)) { fetch(h0 + slot, x); }
#pragma unroll
    for (int i = 0; i < 8; ++i) { q_weight[i] = k_weight[i] = 1.f; }
    if (item < per && s.q_norm != nullptr) { load4(s.q_norm + e0, q_weight); load4(s.q_norm + e1, q_weight + 4); }
    if (item < per && s.k_norm != nullptr) { load4(s.k_norm + e0, k_weight); load4(s.k_norm + e1, k_weight + 4); }
    const int q = sequence_of(p.view, row);
    if (q < 0 || q >= p.view.n_seq) { return; }
    const int end = p.view.row_start[q + 1];
    const int pos = p.view.n_kv[q] - end + row;
    if (row >= end || pos < 0) { return; }
    int64_t cell = -1, pair = 0;
    if (pos < p.view.n_kv_most) {
        const int page = p.view.page_table[(int64_t)q * p.view.table_stride + pos / p.view.page_size], at = pos % p.view.page_size;
        if (page >= 0 && page < p.view.n_pages) {
            cell = page * p.view.page_stride + at * p.view.token_stride;
            pair = page * s.scales.page_stride + at * s.scales.token_stride;
        }
    }
    float co[4], si[4];
    if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double t = (double)pos * p.turns[4 * item + i];
            sincospif(2.0f * (float)(t - rint(t)), &si[i], &co[i]);
        }
    }
    const float mean = 1.f / (float)p.head_dim;
    for (;;) {
        const int  h = h0 + slot, next = h0 + step;
        const bool is_q = h < p.n_head, is_k = !is_q && h < p.n_head + p.n_head_kv, mine = works(h);
        const int  hh = is_q ? h : is_k ? h - p.n_head : h - p.n_head - p.n_head_kv;
        float ahead[8];
        if (AHEAD && works(next + slot)) { fetch(next + slot, ahead); }
        if (is_q ? s.q_norm != nullptr : is_k && s.k_norm != nullptr) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) { sum = fmaf(x[i], x[i], sum); }
            const unsigned all = width == 32 ? 0xffffffffu : ((1u << width) - 1) << (threadIdx.x & 31 & ~(width - 1));   // a head's threads: others may have another kind of head
            for (int o = width / 2; o > 0; o >>= 1) { sum += __shfl_xor_sync(all, sum, o); }
            const float f = rsqrtf(fmaf(sum, mean, s.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = x[i] * f * (is_q ? q_weight[i] : k_weight[i]); }
        }
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
            if (mine) {
                TQ *dst = static_cast<TQ *>(p.q_out) + row * p.q_out_stride + (int64_t)hh * p.head_dim;
                store4(dst + e0, x); store4(dst + e1, x + 4);
            }
        } else if constexpr (EIGHT) {
            uint32_t most = 0;                                      // (as bits: NaN is above everything)
#pragma unroll
            for (int i = 0; i < 8; ++i) { most = max(most, __float_as_uint(x[i]) & 0x7fffffffu); }
            const unsigned all = width == 32 ? 0xffffffffu : ((1u << width) - 1) << (threadIdx.x & 31 & ~(width - 1));
            for (int o = width / 2; o > 0; o >>= 1) { most = max(most, __shfl_xor_sync(all, most, o)); }
            const bool   fine = most <= __float_as_uint(65468.f);
            const __half scale = fine ? __float2half_ru(__fdiv_rn(__uint_as_float(most), 127.f)) : __ushort_as_half(0x7fff);
            if (mine && cell >= 0) {
                const float per_one = fine && most > 0 ? 1.f / __half2float(scale) : 0.f;
                uint8_t *dst = (is_k ? s.k8 : s.v8) + cell + hh * p.view.head_stride;
                uint32_t b[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { b[i] = fine ? __float_as_uint(fmaf(x[i], per_one, 12582912.f)) : 0u; }   // (1.5 x 2^23: the integer is the low byte)
                *reinterpret_cast<uint32_t *>(dst + e0) = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
                *reinterpret_cast<uint32_t *>(dst + e1) = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
                if (item == 0) { reinterpret_cast<__half *>(const_cast<uint32_t *>(s.scales.pairs))[2 * (pair + hh * s.scales.head_stride) + (is_k ? 0 : 1)] = scale; }
            }
        } else if (mine && cell >= 0) {
            __half *dst = (is_k ? p.k_cache : p.v_cache) + cell + hh * p.view.head_stride;
            store4(dst + e0, x); store4(dst + e1, x + 4);
        }
        if (next >= total) { break; }
        h0 = next;
        if (AHEAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { x[i] = ahead[i]; }
        } else if (works(h0 + slot)) { fetch(h0 + slot, x); }
    }
}

// ---------------------------------------------------------------------------------------------- load
// Memory bound: a byte (or two) read and two (or four) written an element. A CTA has eight rows, whose places its warps find, one each; a thread has eight elements of one head in all of them.
constexpr int LD_THREADS = 256, LD_ROWS = 8;

template <class T, bool EIGHT>
__global__ void __launch_bounds__(LD_THREADS) paged_load_kernel(const __grid_constant__ PagedLoad p) {
    __shared__ int64_t cells[LD_ROWS], pairs[LD_ROWS];             // -1: nothing there; -2: nobody's row
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row0 = blockIdx.x * LD_ROWS;
    {
        const int row = row0 + warp;
        int64_t cell = -2, pair = 0;
        const int q = row < p.view.n_rows ? sequence_of(p.view, row) : -1;
        if (q >= 0 && q < p.view.n_seq) {
            const int end = p.view.row_start[q + 1], pos = p.view.n_kv[q] - end + row;
            if (row < end) {
                cell = -1;
                if (pos >= 0 && pos < p.view.n_kv_most) {
                    const int page = p.view.page_table[(int64_t)q * p.view.table_stride + pos / p.view.page_size], at = pos % p.view.page_size;
                    if (page >= 0 && page < p.view.n_pages) {
                        cell = page * p.view.page_stride + at * p.view.token_stride;
                        pair = page * p.scales.page_stride + at * p.scales.token_stride;
                    }
                }
            }
        }
        if (lane == 0) { cells[warp] = cell; pairs[warp] = pair; }
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
#pragma unroll 4
        for (int r = sub; r < LD_ROWS; r += rows_at_once) {
            const int64_t cell = cells[r];
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (cell >= 0) {
                if constexpr (EIGHT) {
                    const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(is_v ? p.v : p.k) + cell + in));
                    const float2 s = half2_bits(p.scales.pairs[pairs[r] + of_pair]);
                    const float scale = is_v ? s.y : s.x;
                    uint32_t h[4];
                    halves_of(w.x, h[0], h[1]); halves_of(w.y, h[2], h[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) { const float2 u = half2_bits(h[k]); x[2 * k] = u.x * scale; x[2 * k + 1] = u.y * scale; }
                } else {
                    const __half *src = static_cast<const __half *>(is_v ? p.v : p.k) + cell + in;
                    load4(src, x); load4(src + 4, x + 4);
                }
            }
            if (cell != -2) { store4(dst + r * stride, x); store4(dst + r * stride + 4, x + 4); }
        }
    }
}

// ---------------------------------------------------------------------------------------------- who shares what
// A warp for each sequence: its group, what all of the group's sequences that have rows see whole, and the first of these, which stands for all in the first pass.
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
        common = with_rows > 1 ? common / PA_SHARED * PA_SHARED : 0;
    }
    if (lane == 0) {
        const int begin = p.view.row_start[s];
        p.from[s] = common;
        p.kv[s] = common;
        p.row_end[s] = s == leader && common > 0 ? p.view.row_start[group_end] : begin;
        p.lead[s] = common > 0 ? p.view.row_start[leader] : begin;
    }
}

// A row of a query head a warp: the pieces of its tile that the first pass's CTAs left, joined in their order. (In the first pass itself one CTA would have to read them all, 18 pieces of 64 KB where 64 requests
// share 6000 positions: 35 us of its 51.)
constexpr int SJ_WARPS = 8, SJ_TILE = 128;    // (rows of a tile of the tensor-memory kernel)
template <int HD>
__global__ void __launch_bounds__(SJ_WARPS * 32) paged_shared_join_kernel(const __grid_constant__ PagedSharedJoin p) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, n_head = p.n_head_kv * p.group;
    const int64_t cell = (int64_t)blockIdx.x * SJ_WARPS + (threadIdx.x >> 5);
    const int row = (int)(cell / n_head), head = (int)(cell - (int64_t)row * n_head), kv = (int)((unsigned)head / (unsigned)p.group);
    if (row >= p.view.n_rows) { return; }
    const int s = sequence_of(p.view, row);
    if (s < 0 || s >= p.view.n_seq || row >= p.view.row_end[s] || p.from[s] == 0) { return; }
    const int lead = max(0, p.lead[s]), tokens = SJ_TILE / p.group, half = (int)((unsigned)(row - lead) / (unsigned)tokens), first = lead + half * tokens;
    if (row < lead) { return; }                                     // (no group that makes sense)
    const int2 cut = p.cuts[(int64_t)kv * p.view.n_rows + first];
    if (cut.y < 2) { return; }
    const int r = (row - first) * p.group + head - kv * p.group;
    constexpr int PIECE = SJ_TILE * (HD + 2);
    auto piece = [&](int i) { return p.partial + (paged_slot(cut.x + i, cut.x) * 2 + (half & 1)) * PIECE; };
    float  m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = 0; i0 < cut.y; i0 += 8) {                         // eight pieces are in flight together; what came before is scaled to the new maximum
        float  pm[8], pl[8], top = m;
        float4 u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool is = i0 + j < cut.y;
            const float *from = piece(is ? i0 + j : 0);
            pm[j] = is ? __ldcg(from + SJ_TILE * HD + r) : -INFINITY;
            pl[j] = is ? __ldcg(from + SJ_TILE * HD + SJ_TILE + r) : 0.f;
            u[j] = is && lane < HD / 4 ? __ldcg(reinterpret_cast<const float4 *>(from) + lane * SJ_TILE + r) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) { top = fmaxf(top, pm[j]); }
        const float base = top == -INFINITY ? 0.f : top, before = exp2f(m - base);
        m = top; l *= before;
        v = make_float4(v.x * before, v.y * before, v.z * before, v.w * before);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = exp2f(pm[j] - base);
            v.x += f * u[j].x; v.y += f * u[j].y; v.z += f * u[j].z; v.w += f * u[j].w;
            l += f * pl[j];
        }
    }
    if (lane < HD / 4) { reinterpret_cast<float4 *>(p.out + cell * HD)[lane] = v; }
    if (lane == 0) { p.stats[cell] = make_float2(m, l); }
}

template <class TIn, class TQ, bool EIGHT>
cudaError_t launch_store(const PagedStore &p, int sms, const LaunchCfg &cfg) {
    int width = 1;
    while (width < p.append.head_dim / 8) { width *= 2; }
    const int total = p.append.n_head + 2 * p.append.n_head_kv, slots = ST_THREADS / width, loops = (total + slots - 1) / slots;
    // few rows: a row's heads are spread over CTAs
    const int  split = std::max(1, std::min(loops, 2 * sms / std::max(1, p.append.view.n_rows)));
    const dim3 grid(p.append.view.n_rows, split);
    return (int64_t)p.append.view.n_rows * split <= 4 * sms ? launch_maybe_pdl(paged_store_kernel<TIn, TQ, EIGHT, true>, grid, ST_THREADS, 0, cfg.stream, cfg.pdl, p, width)
                                                            : launch_maybe_pdl(paged_store_kernel<TIn, TQ, EIGHT, false>, grid, ST_THREADS, 0, cfg.stream, cfg.pdl, p, width);
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
cudaError_t launch_paged_load(const PagedLoad &p, int out_type, int, const LaunchCfg &cfg) {
    const dim3 grid((p.view.n_rows + LD_ROWS - 1) / LD_ROWS);
    const auto kernel = p.scales.pairs != nullptr ? (out_type == SPYB_FP32 ? paged_load_kernel<float, true> : paged_load_kernel<__half, true>)
                                                  : out_type == SPYB_FP32 ? paged_load_kernel<float, false> : paged_load_kernel<__half, false>;
    return launch_maybe_pdl(kernel, grid, LD_THREADS, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_shared(const PagedShared &p, const LaunchCfg &cfg) {
    return launch_maybe_pdl(paged_shared_kernel, dim3((p.view.n_seq + SH_WARPS - 1) / SH_WARPS), SH_WARPS * 32, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_shared_join(const PagedSharedJoin &p, int head_dim, const LaunchCfg &cfg) {
    const int64_t cells = (int64_t)p.view.n_rows * p.n_head_kv * p.group;
    return launch_maybe_pdl(head_dim == 128 ? paged_shared_join_kernel<128> : paged_shared_join_kernel<64>, dim3((unsigned)((cells + SJ_WARPS - 1) / SJ_WARPS)), SJ_WARPS * 32, 0, cfg.stream, cfg.pdl, p);
}
cudaError_t launch_paged_shared_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg) { return launch_rows_kind<PK_SHARED>(p, head_dim, row_tiles, sms, cfg); }

}  // namespace spyb
