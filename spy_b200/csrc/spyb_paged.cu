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
#include "spyb_paged_rows.cuh"

namespace spyb {
namespace {

// ---------------------------------------------------------------------------------------------- append
// Memory bound: every element is read once and written once, (4 + 2) or (2 + 2) bytes. A CTA has one row; a thread has eight elements of a head - a 16-byte piece of
// the output, or half of two pieces where the pairs are halves - in every 8th or 16th head, so that its (up to) four angles are made once a row. Angles are
// position x share of a circle in 64 bits, reduced to half a turn either way: in f32 a position of 100 000 leaves an angle 0.004 of uncertainty.
// Measured: 9246 rows of 120 heads of 128 elements (f32, 852 MB) 149 us, 5.7 TB/s; one row 3.5 us and 96 rows 6 to 7 us, a launch and a chain of dependent loads
// (whose row, which position, which page), beside which the row's first elements come.
constexpr int AP_THREADS = 256;

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

spyb_status paged_check_view(Refusal &no, const char *what, const spyb_paged_cache &c, const spyb_paged_batch &b, const spyb_paged_scales *scales) {
    const bool bytes = scales != nullptr && c.number_type == SPYB_INT8;
    if (c.number_type != SPYB_FP16 && !bytes) { return no.because("%s: a cache of type %d (fp16%s it has to be)", what, c.number_type, scales != nullptr ? " or int8" : ""); }
    if (c.k == nullptr || c.v == nullptr || !aligned_to(c.k, 16) || !aligned_to(c.v, 16)) { return no.because("%s: the cache's k and v must be there and 16-byte aligned", what); }
    if (c.n_pages < 1 || c.page_size < 1 || c.n_head_kv < 1 || c.n_head_kv > 65535 || c.head_dim < 8 || c.head_dim > 256 || c.head_dim % 8 != 0) {
        return no.because("%s: %d pages of %d positions, %d heads of %d elements", what, c.n_pages, c.page_size, c.n_head_kv, c.head_dim);
    }
    const int unit = bytes ? 16 : 8;
    if (c.page_stride < 0 || c.token_stride < 0 || c.head_stride < 0 || ((c.page_stride | c.token_stride | c.head_stride) & (unit - 1))) {
        return no.because("%s: the cache's strides (%lld, %lld, %lld) must be multiples of %d elements, not negative", what, (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride, unit);
    }
    if (bytes && (scales->pairs == nullptr || !aligned_to(scales->pairs, 4) || scales->page_stride < 0 || scales->token_stride < 0 || scales->head_stride < 0)) {
        return no.because("%s: the scales of an int8 cache must be there and 4-byte aligned, their strides (%lld, %lld, %lld) not negative", what, (long long)scales->page_stride,
                          (long long)scales->token_stride, (long long)scales->head_stride);
    }
    if (b.n_seq < 0 || b.n_rows < 0 || b.max_rows < 0 || b.table_stride < 0 || b.n_seq >= (1 << 24) || b.n_rows >= (1 << 24)) {
        return no.because("%s: %d sequences, %d rows (most %d), table rows of %d", what, b.n_seq, b.n_rows, b.max_rows, b.table_stride);
    }
    if (b.n_seq > 0 && (b.row_start == nullptr || b.n_kv == nullptr || (b.table_stride > 0 && b.page_table == nullptr) || !aligned_to(b.row_start, 4) || !aligned_to(b.n_kv, 4) || !aligned_to(b.page_table, 4))) {
        return no.because("%s: row_start, n_kv and page_table must be there and 4-byte aligned", what);
    }
    return SPYB_SUCCESS;
}
PagedView paged_view(const spyb_paged_cache &c, const spyb_paged_batch &b) {
    PagedView v;
    v.row_start = b.row_start; v.row_end = b.row_start + 1; v.n_kv = b.n_kv; v.page_table = b.page_table;
    v.n_seq = b.n_seq; v.n_rows = b.n_rows; v.table_stride = b.table_stride; v.n_pages = c.n_pages; v.page_size = c.page_size;
    v.n_kv_most = (int)std::min<int64_t>((int64_t)b.table_stride * c.page_size, 1 << 30);
    v.page_stride = c.page_stride; v.token_stride = c.token_stride; v.head_stride = c.head_stride;
    return v;
}
PagedScales paged_scales_of(const spyb_paged_cache &c, const spyb_paged_scales &s) {
    PagedScales got;
    if (c.number_type == SPYB_INT8) { got.pairs = static_cast<const uint32_t *>(s.pairs); got.page_stride = s.page_stride; got.token_stride = s.token_stride; got.head_stride = s.head_stride; }
    return got;
}
cudaError_t launch_paged_attention_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg) { return launch_rows_kind<PK_PLAIN>(p, head_dim, row_tiles, sms, cfg); }

namespace {

int stride_unit(int t) { return t == SPYB_FP32 ? 4 : 8; }

spyb_status check_append(Refusal &no, const spyb_paged_append_desc &d, const char *what = "paged_append", const spyb_paged_scales *scales = nullptr) {
    const spyb_status st = paged_check_view(no, what, d.cache, d.batch, scales);
    if (st != SPYB_SUCCESS) { return st; }
    const bool has_q = d.q != nullptr;
    if (!value_type(d.in_type) || (has_q && !value_type(d.q_out_type))) { return no.because("%s: input of type %d, Q of type %d", what, d.in_type, d.q_out_type); }
    if (d.n_head < 0 || d.n_head > 65535 || has_q != (d.n_head > 0)) { return no.because("%s: %d query heads, Q %s", what, d.n_head, has_q ? "given" : "left out"); }
    if (d.k == nullptr || d.v == nullptr || (has_q && d.q_out == nullptr) || !aligned_to(d.q, 16) || !aligned_to(d.k, 16) || !aligned_to(d.v, 16) || (has_q && !aligned_to(d.q_out, 16))) {
        return no.because("%s: q, k, v and q_out must be there and 16-byte aligned", what);
    }
    if (((d.k_stride | d.v_stride | (has_q ? d.q_stride : 0)) & (stride_unit(d.in_type) - 1)) || (has_q && (d.q_out_stride & (stride_unit(d.q_out_type) - 1)))) {
        return no.because("%s: row strides must be multiples of 16 bytes", what);
    }
    if (d.rope_mode != SPYB_ROPE_NONE && d.rope_mode != SPYB_ROPE_PAIRS && d.rope_mode != SPYB_ROPE_HALVES) { return no.because("%s: rope mode %d", what, d.rope_mode); }
    if (d.rope_mode != SPYB_ROPE_NONE && (d.rope_dim < 8 || d.rope_dim > d.cache.head_dim || d.rope_dim % 8 != 0 || !(d.freq_base > 0.f) || !std::isfinite(d.freq_base) || !std::isfinite(d.freq_scale))) {
        return no.because("%s: %d rotated elements of %d, base %g, scale %g", what, d.rope_dim, d.cache.head_dim, d.freq_base, d.freq_scale);
    }
    return SPYB_SUCCESS;
}
spyb_status check_attention(Refusal &no, const spyb_paged_attention_desc &d, const char *what = "paged_attention", const spyb_paged_scales *scales = nullptr) {
    const spyb_status st = paged_check_view(no, what, d.cache, d.batch, scales);
    if (st != SPYB_SUCCESS) { return st; }
    const int hd = d.cache.head_dim;
    if (hd != 32 && hd != 64 && hd != 96 && hd != 128) { return no.because("%s: heads of %d elements (32, 64, 96 or 128)", what, hd); }
    if (!value_type(d.out_type)) { return no.because("%s: output of type %d", what, d.out_type); }
    if (d.n_head < 1 || d.n_head % d.cache.n_head_kv != 0 || d.n_head > 65535) { return no.because("%s: %d query heads over %d K/V heads", what, d.n_head, d.cache.n_head_kv); }
    if (d.q == nullptr || d.out == nullptr || !aligned_to(d.q, 16) || !aligned_to(d.out, 16) || (d.q_stride & 7) || (d.out_stride & (stride_unit(d.out_type) - 1))) {
        return no.because("%s: q and out must be there and 16-byte aligned, their row strides multiples of 16 bytes", what);
    }
    if (d.window < 0 || (d.window > 0 && d.causal == 0)) { return no.because("%s: a window of %d positions%s", what, d.window, d.causal == 0 ? " without causal" : ""); }
    if (!std::isfinite(d.scale)) { return no.because("%s: scale %g", what, d.scale); }
    if ((int64_t)d.batch.n_rows * (d.n_head / d.cache.n_head_kv) >= (1ll << 30)) { return no.because("%s: %d rows of %d heads", what, d.batch.n_rows, d.n_head); }
    return SPYB_SUCCESS;
}
spyb_status check_store(Refusal &no, const spyb_paged_store_desc &d) {
    const spyb_status st = check_append(no, d.append, "paged_store", &d.scales);
    if (st != SPYB_SUCCESS) { return st; }
    if ((d.q_norm != nullptr && d.append.q == nullptr) || !aligned_to(d.q_norm, 16) || !aligned_to(d.k_norm, 16)) { return no.because("paged_store: norms must be 16-byte aligned, Q's has to have a Q"); }
    if (!(d.norm_eps >= 0.f) || !std::isfinite(d.norm_eps)) { return no.because("paged_store: norm_eps %g", d.norm_eps); }
    return SPYB_SUCCESS;
}
spyb_status check_load(Refusal &no, const spyb_paged_load_desc &d) {
    const spyb_status st = paged_check_view(no, "paged_load", d.cache, d.batch, &d.scales);
    if (st != SPYB_SUCCESS) { return st; }
    if (!value_type(d.out_type)) { return no.because("paged_load: output of type %d", d.out_type); }
    if ((d.k == nullptr && d.v == nullptr) || !aligned_to(d.k, 16) || !aligned_to(d.v, 16)) { return no.because("paged_load: k or v must be there, both 16-byte aligned"); }
    if (((d.k != nullptr ? d.k_stride : 0) | (d.v != nullptr ? d.v_stride : 0)) & (stride_unit(d.out_type) - 1)) { return no.because("paged_load: row strides must be multiples of 16 bytes"); }
    return SPYB_SUCCESS;
}
// What a call with groups keeps in its workspace: accumulators and statistics of the first pass, and who shares what
struct SharedRoom { uint64_t out, stats, cuts, words, bytes; };
SharedRoom shared_room(int64_t n_seq, int64_t n_rows, int64_t n_head, int64_t head_dim) {
    SharedRoom r;
    const uint64_t cells = (uint64_t)n_rows * n_head;
    r.out = 0; r.stats = cells * head_dim * sizeof(float); r.cuts = r.stats + cells * sizeof(float2); r.words = r.cuts + cells * sizeof(int2);
    r.bytes = (r.words + 4 * (uint64_t)n_seq * sizeof(int32_t) + 15) & ~15ull;
    return r;
}
spyb_status check_attend(Refusal &no, const spyb_paged_attend_desc &d) {
    const spyb_status st = check_attention(no, d.attention, "paged_attend", &d.scales);
    if (st != SPYB_SUCCESS) { return st; }
    const spyb_paged_shared &s = d.shared;
    if (s.n_group < 0 || s.n_group >= (1 << 24)) { return no.because("paged_attend: %d groups", s.n_group); }
    if (s.n_group == 0) { return SPYB_SUCCESS; }
    if (s.group_start == nullptr || s.n_shared == nullptr || !aligned_to(s.group_start, 4) || !aligned_to(s.n_shared, 4)) { return no.because("paged_attend: group_start and n_shared must be there and 4-byte aligned"); }
    const uint64_t need = shared_room(d.attention.batch.n_seq, d.attention.batch.n_rows, d.attention.n_head, d.attention.cache.head_dim).bytes;
    if (need > 0 && (s.workspace == nullptr || !aligned_to(s.workspace, 16) || s.workspace_bytes < need)) {
        return no.because("paged_attend: groups ask for a workspace of %llu bytes, 16-byte aligned (there are %llu)", (unsigned long long)need, (unsigned long long)(s.workspace == nullptr ? 0 : s.workspace_bytes));
    }
    return SPYB_SUCCESS;
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
        p.view.row_start = start.data(); p.view.row_end = start.data() + 1; p.view.n_kv = kv.data(); p.view.n_seq = n_seq; p.view.n_rows = std::max(1, start[n_seq] - rnd(2)); p.view.page_size = 1 + rnd(40);
        p.view.table_stride = 1 + rnd(80); p.view.n_kv_most = p.view.table_stride * p.view.page_size;
        p.n_head_kv = 1 + rnd(5); p.group = 1 + rnd(8); p.tile_rows = tile_rows > 0 ? tile_rows : 2 * (128 / p.group) * p.group; p.causal = rnd(4) != 0; p.window = p.causal && rnd(2) ? 1 + rnd(500) : 0; p.few_rows = rnd(3) == 0 ? 1 << 30 : rnd(40);
        p.start_units = rnd(2) * rnd(5);
        const bool all_seen = p.window > 0 && turn % 4 == 1;   // a window as long as an int can say is none
        if (all_seen) { p.window = paged_window(INT_MAX - rnd(3)); }
        std::vector<int32_t> from(n_seq);        // own positions of the second of two passes; of nonsense too
        if (turn % 2 == 1 && p.window == 0) {
            for (int32_t &x : from) { x = 16 * rnd(1 + most_kv / (turn % 3 == 1 ? 8 : 24)); }
            p.view.from = from.data();
        }
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
                    if (it.lo < 0 || (p.view.from != nullptr ? it.lo != q.from || it.lo % 16 != 0 : it.lo % ALIGN != 0) || it.hi > p.view.n_kv_most || off >= it.units || (int64_t)it.units * UNIT + it.lo < it.hi) { return 4; }
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
    for (const int tile : {8, 16, 24}) { if (bad == 0) { bad = cut_selftest<64, 64>(4 + tile, tile); } }
    if (bad == 0) { bad = cut_selftest<128, 128>(3, 0); }
    return bad == 0 ? 0 : 100 + bad;
}

}  // namespace spyb

using namespace spyb;

static PagedAppend append_of(spyb_backend *be, const spyb_paged_append_desc &given) {
    const spyb_paged_append_desc *d = &given;
    PagedAppend p;
    p.view = paged_view(d->cache, d->batch);
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
    return p;
}
// One pass over pages: sequences of many rows on tensor memory, the others on the kernel for few
static spyb_status attention_pass(spyb_backend *be, PagedAttention p, int head_dim, int n_head, int64_t most, uint64_t wait_limit, bool *on_tensor_memory = nullptr) {
    const LaunchCfg cfg = be->launch_cfg(be->config.use_pdl != 0);
    const bool bytes = p.kind() == PK_INT8;
    p.few_rows = 1 << 30;
    if (most > (bytes ? PB_FEW_ROWS : PA_FEW_ROWS) && p.scale_log2 >= 0.f) {
        cudaError_t err = cudaSuccess;
        // what single tokens beside the many rows have is the small kernel's in its narrowest tile. (Bytes, four query heads a K/V head, 1500 rows beside 24 sequences of 1, 3 and 5: tiles of 8 rows for
        // sequences of up to 8 377, 431 and 432 us; of 16 389, 393 and 434; of 24 408, 413 and 421. How many rows the others have is known on the device alone, and single tokens are what stands beside a prompt)
        p.few_rows = p.view.n_seq == 1 || p.stats != nullptr ? 0 : !bytes ? PA_FEW_ROWS : p.group > PB_FEW_ROWS ? 0 : (p.group + 7) / 8 * 8;
        const bool taken = launch_paged_attention_tc(p, head_dim, n_head, be->num_sms_total, cfg, wait_limit, &err);
        if (!taken) { p.few_rows = 1 << 30; }
        if (on_tensor_memory != nullptr) { *on_tensor_memory = taken; }
        SPYB_CUDA(be, err);
    }
    if (p.few_rows == 0) { return SPYB_SUCCESS; }
    const int64_t rows = std::min<int64_t>(most, p.few_rows);
    const int row_tiles = rows <= 16 ? 1 : 2;
    p.tile_rows = bytes ? (rows <= 8 ? 8 : rows <= 16 ? 16 : 24) : 16 * row_tiles;
    SPYB_CUDA(be, bytes ? launch_paged_attention_bytes(p, head_dim, be->num_sms_total, cfg, wait_limit)
                  : p.kind() == PK_SHARED ? launch_paged_shared_rows(p, head_dim, row_tiles, be->num_sms_total, cfg)
                                          : launch_paged_attention_rows(p, head_dim, row_tiles, be->num_sms_total, cfg));
    return SPYB_SUCCESS;
}
// The public calls (`scales`, `shared`: spyb_paged_attend's), and with a role that is late the self-checks'. The descriptors have been checked.
static spyb_status paged_attention(spyb_backend *be, const spyb_paged_attention_desc &d, int late, uint64_t wait_limit, const spyb_paged_scales *scales = nullptr, const spyb_paged_shared *shared = nullptr) {
    if (d.batch.n_seq == 0 || d.batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    if (!be->paged_workspace()) { return SPYB_FAIL; }
    const int hd = d.cache.head_dim;
    PagedAttention p;
    p.view = paged_view(d.cache, d.batch);
    p.q = static_cast<const __half *>(d.q); p.out = d.out;
    p.k = static_cast<const __half *>(d.cache.k); p.v = static_cast<const __half *>(d.cache.v);
    p.q_stride = d.q_stride; p.out_stride = d.out_stride; p.n_head_kv = d.cache.n_head_kv; p.group = d.n_head / d.cache.n_head_kv;
    p.causal = d.causal != 0; p.window = paged_window(d.window); p.out_f32 = d.out_type == SPYB_FP32;
    const float scale = d.scale == 0.f ? 1.0f / std::sqrt((float)hd) : d.scale;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634073599);
    p.late = late; p.partial = be->paged_partial; p.arrived = be->paged_arrived;
    if (scales != nullptr) { p.scales = paged_scales_of(d.cache, *scales); }
    const int64_t most = (int64_t)(d.batch.max_rows > 0 ? std::min(d.batch.max_rows, d.batch.n_rows) : d.batch.n_rows) * p.group;
    if (shared != nullptr && shared->n_group > 0 && d.window == 0 && d.batch.n_seq > 1) {
        // Two passes: over what the sequences of a group share, all of their rows as one sequence's, and over the rest, which joins the two
        const SharedRoom room = shared_room(d.batch.n_seq, d.batch.n_rows, d.n_head, hd);
        uint8_t *const mem = static_cast<uint8_t *>(shared->workspace);
        PagedShared g;
        g.view = p.view; g.group_start = shared->group_start; g.n_shared = shared->n_shared; g.n_group = shared->n_group; g.causal = p.causal; g.align = paged_shared_align(d.cache.page_size);
        g.from = reinterpret_cast<int32_t *>(mem + room.words); g.row_end = g.from + d.batch.n_seq; g.kv = g.row_end + d.batch.n_seq; g.lead = g.kv + d.batch.n_seq;
        SPYB_CUDA(be, launch_paged_shared(g, be->launch_cfg(be->config.use_pdl != 0)));
        PagedAttention first = p;
        first.view.row_end = g.row_end; first.view.n_kv = g.kv; first.causal = 0;
        first.out = mem + room.out; first.out_f32 = 1; first.out_stride = (int64_t)d.n_head * hd; first.stats = reinterpret_cast<float2 *>(mem + room.stats); first.cuts = reinterpret_cast<int2 *>(mem + room.cuts);
        bool on_tensor_memory = false;
        const spyb_status st = attention_pass(be, first, hd, d.n_head, (int64_t)d.batch.n_rows * p.group, wait_limit, &on_tensor_memory);
        if (st != SPYB_SUCCESS) { return st; }
        if (on_tensor_memory) {
            PagedSharedJoin j;
            j.view = p.view; j.from = g.from; j.lead = g.lead; j.cuts = first.cuts; j.partial = be->paged_partial; j.out = static_cast<float *>(first.out); j.stats = first.stats;
            j.n_head_kv = p.n_head_kv; j.group = p.group; j.ctas = be->num_sms_total;
            SPYB_CUDA(be, launch_paged_shared_join(j, hd, be->launch_cfg(be->config.use_pdl != 0)));
        }
        p.view.from = g.from; p.with_stats = first.stats; p.with_out = static_cast<const float *>(first.out);
    }
    return attention_pass(be, p, hd, d.n_head, most, wait_limit);
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

spyb_status spyb_paged_store_check(const spyb_paged_store_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_store(no, *d), message, size);
}
spyb_status spyb_paged_load_check(const spyb_paged_load_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_load(no, *d), message, size);
}
spyb_status spyb_paged_attend_check(const spyb_paged_attend_desc *d, char *message, int32_t size) {
    Refusal no;
    return d == nullptr ? SPYB_FAIL : no.answer(check_attend(no, *d), message, size);
}

spyb_status spyb_paged_append(spyb_backend *be, const spyb_paged_append_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_append(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->batch.n_seq == 0 || d->batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    SPYB_CUDA(be, launch_paged_append(append_of(be, *d), d->in_type, d->q_out_type, be->num_sms_total, be->launch_cfg(be->config.use_pdl != 0)));
    return SPYB_SUCCESS;
}
spyb_status spyb_paged_store(spyb_backend *be, const spyb_paged_store_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_store(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->append.batch.n_seq == 0 || d->append.batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    PagedStore p;
    p.append = append_of(be, d->append);
    p.scales = paged_scales_of(d->append.cache, d->scales);
    p.q_norm = d->q_norm; p.k_norm = d->k_norm; p.eps = d->norm_eps;
    p.k8 = static_cast<uint8_t *>(d->append.cache.k); p.v8 = static_cast<uint8_t *>(d->append.cache.v);
    SPYB_CUDA(be, launch_paged_store(p, d->append.in_type, d->append.q_out_type, be->num_sms_total, be->launch_cfg(be->config.use_pdl != 0)));
    return SPYB_SUCCESS;
}
spyb_status spyb_paged_load(spyb_backend *be, const spyb_paged_load_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_load(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    if (d->batch.n_seq == 0 || d->batch.n_rows == 0) { return SPYB_SUCCESS; }
    use_device(be->config.device_id);
    PagedLoad p;
    p.view = paged_view(d->cache, d->batch);
    p.k = d->cache.k; p.v = d->cache.v; p.scales = paged_scales_of(d->cache, d->scales);
    p.k_out = d->k; p.v_out = d->v; p.k_stride = d->k_stride; p.v_stride = d->v_stride; p.n_head_kv = d->cache.n_head_kv; p.head_dim = d->cache.head_dim;
    SPYB_CUDA(be, launch_paged_load(p, d->out_type, be->num_sms_total, be->launch_cfg(be->config.use_pdl != 0)));
    return SPYB_SUCCESS;
}

spyb_status spyb_paged_attention(spyb_backend *be, const spyb_paged_attention_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_attention(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    return paged_attention(be, *d, PA_ON_TIME, be->wait_limit_ns);
}
spyb_status spyb_paged_attend(spyb_backend *be, const spyb_paged_attend_desc *d) {
    if (be == nullptr || d == nullptr) { return SPYB_FAIL; }
    Refusal no;
    if (check_attend(no, *d) != SPYB_SUCCESS) { be->set_error("%s", no.text); return SPYB_UNSUPPORTED; }
    return paged_attention(be, d->attention, PA_ON_TIME, be->wait_limit_ns, &d->scales, &d->shared);
}
uint64_t spyb_paged_attend_workspace(int32_t n_seq, int32_t n_rows, int32_t n_head, int32_t head_dim) {
    if (n_seq < 0 || n_rows < 0 || n_head < 0 || head_dim < 0 || n_seq >= (1 << 24) || n_rows >= (1 << 24) || n_head > 65535 || head_dim > 256) { return 0; }
    return shared_room(n_seq, n_rows, n_head, head_dim).bytes;
}

// Self-check of the tensor-memory kernel's hand-overs: a chunk at the end of a long conversation and a short one, on time and with one of its roles late. A role that is late within
// the limit of the waits changes nothing; copies that come three limits late make waits give up: the kernel ends by itself, when they have landed, says so, and leaves nothing for
// the next launch.
spyb_status spyb_paged_selftest_late(spyb_backend *be, int32_t who, uint64_t limit_ns, int32_t *error_code_out) {
    if (be == nullptr || limit_ns == 0 || who < PA_LATE_CHECKS || who > PA_LATE_FEW) { return SPYB_FAIL; }
    use_device(be->config.device_id);
    SPYB_CUDA(be, cudaStreamSynchronize(be->stream));
    if (be->device_error()) { return SPYB_FAIL; }
    // (few rows: of the kernel for bytes)
    const bool few = who == PA_LATE_FEW;
    constexpr int heads = 2, group = 3, page = 16, pages = 1300, kv[2] = {20000, 70};
    const int rows[2] = {few ? 2 : 300, few ? 1 : 70}, n_rows = rows[0] + rows[1];
    const int32_t words[5] = {0, rows[0], n_rows, kv[0], kv[1]};
    std::vector<int32_t> table(2 * pages);
    for (int i = 0; i < 2 * pages; ++i) { table[i] = i % pages; }
    int code = 0;
    for (const int which : {0, 1, 2, 3}) {
        const int  hd = which & 1 ? 128 : 64;
        const bool bytes = which >= 2;
        if (few && !bytes) { continue; }
        const size_t n_pool = (size_t)pages * page * heads * hd, n_q = (size_t)n_rows * heads * group * hd;
        std::vector<uint16_t> host(2 * n_pool + n_q);
        uint32_t seed = 1;
        for (uint16_t &x : host) { seed = seed * 1664525u + 1013904223u; x = (uint16_t)(0x3000 + (seed >> 18) % 0x0c00 + (seed & 0x80000000u ? 0x8000 : 0)); }   // 0.125 to 1, either sign (bytes: any, and these numbers as their scales)
        std::vector<float> want(n_q), got(n_q);
        uint8_t *mem = nullptr;
        const size_t at_out = host.size() * 2, at_words = at_out + n_q * 4, at_table = at_words + sizeof words, size = at_table + table.size() * 4;
        SPYB_CUDA(be, cudaMalloc(&mem, size));
        spyb_paged_attention_desc d = {};
        d.cache.k = mem; d.cache.v = mem + n_pool * 2; d.cache.number_type = SPYB_FP16; d.cache.n_pages = pages; d.cache.page_size = page; d.cache.n_head_kv = heads; d.cache.head_dim = hd;
        d.cache.page_stride = page * heads * hd; d.cache.token_stride = heads * hd; d.cache.head_stride = hd;
        spyb_paged_scales scales = {};
        if (bytes) {                                          // (both pools of bytes in the place of the one of K in fp16, scales in V's)
            d.cache.number_type = SPYB_INT8; d.cache.v = mem + n_pool;
            scales.pairs = mem + n_pool * 2; scales.page_stride = page * heads; scales.token_stride = heads; scales.head_stride = 1;
        }
        d.batch.row_start = reinterpret_cast<int32_t *>(mem + at_words); d.batch.n_kv = d.batch.row_start + 3; d.batch.page_table = reinterpret_cast<int32_t *>(mem + at_table);
        d.batch.n_seq = 2; d.batch.n_rows = n_rows; d.batch.table_stride = pages;
        d.q = mem + n_pool * 4; d.out = mem + at_out; d.q_stride = d.out_stride = heads * group * hd; d.n_head = heads * group; d.out_type = SPYB_FP32; d.causal = 1;
        cudaError_t err = upload(mem, host.data(), host.size() * 2);
        if (err == cudaSuccess) { err = upload(mem + at_words, words, sizeof words); }
        if (err == cudaSuccess) { err = upload(mem + at_table, table.data(), table.size() * 4); }
        spyb_status st = SPYB_SUCCESS;
        auto run = [&](int late, uint64_t limit, std::vector<float> &to) {
            if (err == cudaSuccess) { err = cudaMemsetAsync(d.out, 0xff, n_q * 4, be->stream); }
            if (err == cudaSuccess && st == SPYB_SUCCESS) { st = paged_attention(be, d, late, limit, bytes ? &scales : nullptr); }
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
        if (before != 0 || code != expected || after != 0) { be->set_error("paged selftest: heads of %d%s: codes %d, %d, %d where 0, %d, 0 were expected", hd, bytes ? " in bytes" : "", before, code, after, expected); return SPYB_FAIL; }
        if (std::memcmp(want.data(), got.data(), n_q * 4) != 0) { be->set_error("paged selftest: heads of %d%s: a late role changed the output, its own or the next launch's", hd, bytes ? " in bytes" : ""); return SPYB_FAIL; }
    }
    return SPYB_SUCCESS;
}

}  // extern "C"
