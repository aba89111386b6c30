// What the kernels over paged caches share: parameters, how a call's work is cut among its CTAs, and the joining of what several CTAs found for one tile of rows.
#pragma once

#include "spyb_common.cuh"
#include "spyb_kernels.h"

namespace spyb {

struct PagedView {                        // a spyb_paged_cache and a spyb_paged_batch as the kernels read them
    const int32_t *row_start = nullptr, *n_kv = nullptr, *page_table = nullptr;
    int            n_seq = 0, n_rows = 0, table_stride = 0, n_pages = 0, page_size = 1;
    int            n_kv_most = 0;         // positions that a row of the table can name
    int64_t        page_stride = 0, token_stride = 0, head_stride = 0;
};
struct PagedAppend {
    PagedView    view;
    const void  *q = nullptr, *k = nullptr, *v = nullptr;
    void        *q_out = nullptr;
    __half      *k_cache = nullptr, *v_cache = nullptr;
    int64_t      q_stride = 0, k_stride = 0, v_stride = 0, q_out_stride = 0;
    int          n_head = 0, n_head_kv = 0, head_dim = 0, rot = 0, halves = 0;
    double       turns[128] = {};         // pair i turns by this share of a full circle a position
};
// the warps that check V stay a few microseconds behind everything else; one copy of a CTA's K and V, or its first of Q, comes three limits of the waits late
enum PagedLate { PA_ON_TIME = 0, PA_LATE_CHECKS = 1, PA_LATE_KV = 2, PA_LATE_Q = 3 };
struct PagedAttention {
    PagedView    view;
    const __half *q = nullptr, *k = nullptr, *v = nullptr;
    void        *out = nullptr;
    int64_t      q_stride = 0, out_stride = 0;
    int          n_head_kv = 0, group = 1, causal = 1, window = 0, out_f32 = 0;
    float        scale_log2 = 0.f;        // scale * log2(e): probabilities are powers of two
    int          tile_rows = 16;          // rows of a tile, counting every query head of its K/V head
    int          page_shift = -1;         // log2 of the page size, if it is a power of two
    int          start_units = 0;         // what going on to an item costs beside its units, in units (PA_START)
    int          few_rows = 0;            // sequences of up to so many rows (of all query heads of a K/V head) are the small kernel's
    float       *partial = nullptr;       // [CTAs][2][rows of a tile][head_dim + 2]
    unsigned    *arrived = nullptr;       // [CTAs], zero between launches
    int          late = PA_ON_TIME;       // self-checks of the tensor-memory kernel
};
int         paged_cut_selftest();   // host-only: 0 when the CTAs' pieces cover every item once, on any lengths
cudaError_t launch_paged_append(const PagedAppend &p, int in_type, int q_out_type, int sms, const LaunchCfg &cfg);
cudaError_t launch_paged_attention_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg);
// the kernel on tensor memory; false where it does not take these pages, heads or strides (nothing is launched then)
bool        launch_paged_attention_tc(const PagedAttention &p, int head_dim, int n_head, int sms, const LaunchCfg &cfg, uint64_t wait_limit, cudaError_t *err);
// Sequences of up to so many rows (times query heads of a K/V head) are the small kernel's, whose tile of 16 rows costs them nothing but the memory's time; a second tile
// doubles its instructions. 24 sequences of up to 9000 positions, four query heads a K/V head: 3 and 4 rows (12 and 16 in all) 95 and 98 us there against
// 118 and 118 on tensor memory, 5 and 8 rows (20 and 32) 144 and 156 against 118 and 118.
constexpr int PA_FEW_ROWS = 16;

// ---------------------------------------------------------------------------------------------- cutting the work
// The rows of a sequence that share a K/V head - token by token, its query heads side by side - are cut into tiles; a tile and a K/V head are an item, and the
// positions that its rows see are counted in units of UNIT. All units of a call, item after item, are cut evenly among the CTAs: whatever the
// lengths are, every SM has the same to read, and one long sequence uses the whole chip. An item on a cut is joined by the CTA that is done with it last.
// A CTA that goes on from one item to the next loses the time of some units (its findings go out, the next item's Q and first block come): an item counts PA_START units
// more than it has. Without them the CTAs with two pieces of items end 10 us behind the others. Small kernel, of 64 positions, none / 1 / 2 / 4: 64 single tokens of up to
// 4096 positions 103.1 / 97.8 / 91.3 / 92.8 us, heads of 64 65.1 / 61.9 / 53.5 / 53.4, 16 of up to 8000 64.0 / 53.3 / 51.0 / 50.4, 100 of up to 300 - / - / 27.5 / 29.0.
// Tensor memory, of 128: 24 x 5 rows of up to 9000 117.5 / 109.7 / 110.6 / 113.2, 512 rows at 3968 54.7 / 53.1 / 52.2 / 52.4, prompts of 6 under a window
// 225.8 / 209.0 / 211.3 / 218.9, 512 at 1024 34.5 / 27.3 / 28.4 / 30.0.
constexpr int PA_START = 2;
struct PagedSeq { int row0, rows, first, kv; };   // first row and number of rows, position of the first row, positions that are there
struct PagedItem { int lo, hi, units; };          // positions [lo, hi) that some row of the tile sees (lo a multiple of ALIGN)

__host__ __device__ __forceinline__ int pmin(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int pmax(int a, int b) { return a < b ? b : a; }
// Positions are below 2^30: a window of as many hides nothing, and a position minus a window stays in 32 bits also for rows in front of position 0
inline int paged_window(int window) { return pmin(window, 1 << 30); }
__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedView &v, int s) {
    const int a = pmax(0, pmin(v.row_start[s], v.n_rows)), end = pmax(a, pmin(v.row_start[s + 1], 1 << 24)), b = pmin(end, v.n_rows);
    const int kv = pmin(pmax(0, v.n_kv[s]), 1 << 30);
    return {a, b - a, kv - (end - a), pmin(kv, v.n_kv_most)};
}
template <int UNIT, int ALIGN>
__host__ __device__ __forceinline__ PagedItem paged_item(const PagedAttention &p, const PagedSeq &q, int tile) {
    const int last = pmin(q.rows * p.group, (tile + 1) * p.tile_rows) - 1;
    const int i0 = (int)((unsigned)(tile * p.tile_rows) / (unsigned)p.group), i1 = (int)((unsigned)last / (unsigned)p.group);
    PagedItem t;
    t.hi = p.causal ? pmin(q.kv, q.first + i1 + 1) : q.kv;
    t.lo = p.causal && p.window > 0 ? pmax(0, q.first + i0 - p.window + 1) / ALIGN * ALIGN : 0;
    t.units = pmax(1, (t.hi - t.lo + UNIT - 1) / UNIT);   // (an item without positions still has its zeros to write)
    return t;
}
__host__ __device__ __forceinline__ bool paged_mine(const PagedAttention &p, const PagedSeq &q, bool few) {
    return q.rows > 0 && ((int64_t)q.rows * p.group <= p.few_rows) == few;
}
template <int UNIT, int ALIGN>
__host__ __device__ __forceinline__ int64_t paged_seq_units(const PagedAttention &p, int s, bool few, int first = 0, int step = 1) {   // of one K/V head; of every step-th tile
    const PagedSeq q = paged_seq(p.view, s);
    if (!paged_mine(p, q, few)) { return 0; }
    const int tiles = (q.rows * p.group + p.tile_rows - 1) / p.tile_rows;
    int64_t n = 0;
    for (int t = first; t < tiles; t += step) { n += paged_item<UNIT, ALIGN>(p, q, t).units + p.start_units; }
    return n;
}

__host__ __device__ __forceinline__ int64_t paged_div(int64_t a, int64_t b) {   // (a division of 64 bits costs some 100 instructions)
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// All units cut into `ctas` stretches, the first `longer` of them one longer than the others
struct PagedShare { int64_t total, each; int ctas, longer; };
__host__ __device__ __forceinline__ PagedShare paged_share(int64_t total, int ctas) {
    const int64_t each = paged_div(total, ctas);
    return {total, each, ctas, (int)(total - each * ctas)};
}
__host__ __device__ __forceinline__ int64_t paged_cta_unit(const PagedShare &s, int c) { return s.each * c + pmin(c, s.longer); }
__host__ __device__ __forceinline__ int paged_unit_cta(const PagedShare &s, int64_t u) {
    const int64_t head = (s.each + 1) * s.longer;
    return u < head ? (int)paged_div(u, s.each + 1) : s.longer + (int)paged_div(u - head, s.each);
}
struct PagedPlace { PagedShare share; int seq, head, tile, off; int64_t unit, end; };   // where a CTA begins, its first unit and the one behind its last
// A CTA's stretch begins at a unit that is work: beginnings of items, which are counted but nobody's, are stepped over (in the middle of a stretch by whoever goes on to the
// next item). A stretch of nothing else is empty.
__host__ __device__ __forceinline__ void paged_begin(const PagedAttention &p, PagedPlace &at) {
    at.unit += pmax(0, p.start_units - at.off);
    at.off = pmax(0, at.off - p.start_units);
}
struct PagedPlanShared { int64_t warp[32], one, rest; int seq; };
__host__ __device__ __forceinline__ int paged_ctas(int64_t total, int grid, int least) { const int64_t n = paged_div(total, least); return n < 1 ? 1 : n < grid ? (int)n : grid; }

// all NT threads of the CTA; `least`: units that a CTA takes at least
template <int NT, int UNIT, int ALIGN>
__device__ PagedPlace paged_plan(const PagedAttention &p, bool few, int least, PagedPlanShared &sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NT / 32;
    // few sequences have a warp each, whose lanes share the tiles; many have a thread each
    const bool by_warp = p.view.n_seq <= NW;
    int64_t total = 0, mine = 0;
    if (by_warp) {
        if (warp < p.view.n_seq) { mine = paged_seq_units<UNIT, ALIGN>(p, warp, few, lane, 32); }
        for (int o = 16; o > 0; o >>= 1) { mine += __shfl_xor_sync(0xffffffffu, mine, o); }
        mine *= p.n_head_kv;
        total = mine;
    } else {
        for (int base = 0; base < p.view.n_seq; base += NT) {
            const int s = base + tid;
            mine = s < p.view.n_seq ? paged_seq_units<UNIT, ALIGN>(p, s, few) * p.n_head_kv : 0;
            total += mine;
        }
        for (int o = 16; o > 0; o >>= 1) { total += __shfl_xor_sync(0xffffffffu, total, o); }
    }
    if (lane == 0) { sh.warp[warp] = total; }
    __syncthreads();
    total = 0;
    for (int w = 0; w < NW; ++w) { total += sh.warp[w]; }
    PagedPlace at;
    at.share = paged_share(total, paged_ctas(total, gridDim.x, least));
    at.unit = at.end = 0; at.seq = at.head = at.tile = at.off = 0;
    if (total == 0 || (int)blockIdx.x >= at.share.ctas) { return at; }
    at.unit = paged_cta_unit(at.share, blockIdx.x);
    at.end = paged_cta_unit(at.share, blockIdx.x + 1);
    if (by_warp) {
        int64_t from = 0;
        for (int w = 0; w < warp; ++w) { from += sh.warp[w]; }
        if (from <= at.unit && at.unit < from + mine && lane == 0) { sh.seq = warp; sh.one = paged_div(mine, p.n_head_kv); sh.rest = at.unit - from; }
    } else {
        int64_t before = 0;
        for (int base = 0; base < p.view.n_seq; base += NT) {
            const int s = base + tid;
            if (p.view.n_seq > NT) { mine = s < p.view.n_seq ? paged_seq_units<UNIT, ALIGN>(p, s, few) * p.n_head_kv : 0; }
            int64_t upto = mine;
            for (int o = 1; o < 32; o <<= 1) { const int64_t v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) { upto += v; } }
            __syncthreads();
            if (lane == 31) { sh.warp[warp] = upto; }
            __syncthreads();
            int64_t all = 0;
            for (int w = 0; w < NW; ++w) { const int64_t v = sh.warp[w]; upto += w < warp ? v : 0; all += v; }
            const int64_t from = before + upto - mine;
            if (from <= at.unit && at.unit < from + mine) { sh.seq = s; sh.one = paged_div(mine, p.n_head_kv); sh.rest = at.unit - from; }
            before += all;
            if (at.unit < before) { break; }   // (the same for all threads)
        }
    }
    __syncthreads();
    at.seq = sh.seq;
    at.head = (int)paged_div(sh.rest, sh.one);
    int64_t rest = sh.rest - at.head * sh.one;
    const PagedSeq q = paged_seq(p.view, at.seq);
    const int tiles = (q.rows * p.group + p.tile_rows - 1) / p.tile_rows;
    for (int base = 0; base < tiles; base += 32) {       // 32 tiles at a time, every warp for itself
        const int u = base + lane < tiles ? paged_item<UNIT, ALIGN>(p, q, base + lane).units + p.start_units : 0;
        int upto = u;
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) { upto += v; } }
        const unsigned hit = __ballot_sync(0xffffffffu, rest < upto);
        if (hit) {
            const int l = __ffs(hit) - 1;
            at.tile = base + l;
            at.off = (int)rest - (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, u, l));
            break;
        }
        rest -= __shfl_sync(0xffffffffu, upto, 31);
    }
    paged_begin(p, at);
    return at;
}

// The item behind an item, the same for all threads; false behind the last one.
__host__ __device__ __forceinline__ bool paged_next(const PagedAttention &p, bool few, PagedSeq &q, int &seq, int &head, int &tile) {
    if ((++tile) * p.tile_rows < q.rows * p.group) { return true; }
    tile = 0;
    if (++head < p.n_head_kv) { return true; }
    head = 0;
    while (++seq < p.view.n_seq) {
        q = paged_seq(p.view, seq);
        if (paged_mine(p, q, few)) { return true; }
    }
    return false;
}

// An item on a cut: its CTAs c0 .. c0 + parts - 1 leave what they found, and who is last joins it in their order. The first one's piece is the last of its own
// stretch (place 1), every other one's the first of its own (place 0).
struct PagedCut { int c0, parts; };
__host__ __device__ __forceinline__ PagedCut paged_cut(const PagedPlace &at, int64_t item_begin, int units) {
    const int a = paged_unit_cta(at.share, item_begin), b = paged_unit_cta(at.share, item_begin + units - 1);
    return {a, b - a + 1};
}
__host__ __device__ __forceinline__ int64_t paged_slot(int c, int c0) { return 2 * (int64_t)c + (c == c0 ? 1 : 0); }

}  // namespace spyb
