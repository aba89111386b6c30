// What the kernels over paged caches share: parameters, how a call's work is cut among its CTAs, and the joining of what several CTAs found for one tile of rows.
#pragma once

#include "spyb_common.cuh"
#include "spyb_kernels.h"
#include "../../include/spyb.h"

namespace spyb {

struct PagedView {                        // a spyb_paged_cache and a spyb_paged_batch as the kernels read them
    const int32_t *row_start = nullptr, *row_end = nullptr, *n_kv = nullptr, *page_table = nullptr;   // (row_end: row_start + 1, or an array of its own)
    const int32_t *from = nullptr;        // positions in front of it (paged_shared_align) are not this pass's; nullptr: all are
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
// the warps that check V (that make operands of bytes) stay a few microseconds behind everything else; one copy of a CTA's K and V, or its first of Q, comes three limits of the waits late; the same of a
// copy of K and V in the kernel for few rows of bytes
enum PagedLate { PA_ON_TIME = 0, PA_LATE_CHECKS = 1, PA_LATE_KV = 2, PA_LATE_Q = 3, PA_LATE_FEW = 4 };
// What a kernel of attention is built for: an fp16 cache whose sequences have nothing in common; one of the two passes where they have; bytes with scales, in passes or not
enum PagedKind { PK_PLAIN = 0, PK_SHARED = 1, PK_INT8 = 2 };
struct PagedScales { const uint32_t *pairs = nullptr; int64_t page_stride = 0, token_stride = 0, head_stride = 0; };   // fp16 pairs: K's scale below, V's above
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
    int          late = PA_ON_TIME;       // self-checks of the tensor-memory kernel and of the one for few rows of bytes
    PagedScales  scales;                  // of an 8-bit cache
    float2      *stats = nullptr;         // first pass of two, over what sequences share: every row's maximum and sum go here, its accumulators as they are to `out` (f32), both [row][head]
    int2        *cuts = nullptr;          // of the first pass on tensor memory, by K/V head and first row of a tile: first CTA and number of CTAs of its item. Several leave their findings where they are
    const float2 *with_stats = nullptr;   // second pass: these are joined with what is found
    const float  *with_out = nullptr;
    __host__ __device__ int kind() const { return scales.pairs != nullptr ? PK_INT8 : stats != nullptr || with_stats != nullptr ? PK_SHARED : PK_PLAIN; }
};
struct PagedStore {
    PagedAppend   append;
    const float  *q_norm = nullptr, *k_norm = nullptr;
    float         eps = 0.f;
    uint8_t      *k8 = nullptr, *v8 = nullptr;       // an 8-bit cache, in place of append's
    PagedScales   scales;                            // (written)
};
struct PagedLoad {
    PagedView    view;
    const void  *k = nullptr, *v = nullptr;
    PagedScales  scales;
    void        *k_out = nullptr, *v_out = nullptr;
    int64_t      k_stride = 0, v_stride = 0;
    int          n_head_kv = 0, head_dim = 0;
};
struct PagedShared {                      // which sequences share what, and what becomes of it
    PagedView      view;
    const int32_t *group_start = nullptr, *n_shared = nullptr;
    int            n_group = 0, causal = 1, align = 128;                 // align: what is shared is cut to a multiple of so many positions
    int32_t       *from = nullptr, *row_end = nullptr, *kv = nullptr, *lead = nullptr;   // [n_seq] each: where a sequence's own positions begin; rows and positions of the first pass's sequences; first row of the group
};
struct PagedSharedJoin {                  // cut items of the first pass on tensor memory
    PagedView      view;
    const int32_t *from = nullptr, *lead = nullptr;
    const int2    *cuts = nullptr;
    const float   *partial = nullptr;
    float         *out = nullptr;
    float2        *stats = nullptr;
    int            n_head_kv = 0, group = 1, ctas = 0;               // ctas: of the first pass
};
constexpr int PA_SHARED = 128;            // fewer positions than that are not shared
// A sequence's own positions begin where a box of the kernels' tensor maps and a block of 16 do: at a multiple of the largest power of two that divides the page size, 16 to 128
inline int paged_shared_align(int page_size) { int a = 128; while (a > 16 && page_size % a != 0) { a /= 2; } return a; }
int         paged_cut_selftest();   // host-only: 0 when the CTAs' pieces cover every item once, on any lengths
cudaError_t launch_paged_store(const PagedStore &p, int in_type, int q_out_type, int sms, const LaunchCfg &cfg);
cudaError_t launch_paged_load(const PagedLoad &p, int out_type, int sms, const LaunchCfg &cfg);
cudaError_t launch_paged_shared(const PagedShared &p, const LaunchCfg &cfg);
cudaError_t launch_paged_shared_join(const PagedSharedJoin &p, int head_dim, const LaunchCfg &cfg);
cudaError_t launch_paged_append(const PagedAppend &p, int in_type, int q_out_type, int sms, const LaunchCfg &cfg);
cudaError_t launch_paged_attention_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg);
cudaError_t launch_paged_shared_rows(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg);   // (PK_SHARED)
cudaError_t launch_paged_attention_bytes(const PagedAttention &p, int head_dim, int sms, const LaunchCfg &cfg, uint64_t wait_limit);   // (PK_INT8; tiles of 8, 16 or 24 rows)
// the kernel on tensor memory; false where it does not take these pages, heads or strides (nothing is launched then)
bool        launch_paged_attention_tc(const PagedAttention &p, int head_dim, int n_head, int sms, const LaunchCfg &cfg, uint64_t wait_limit, cudaError_t *err);
// Sequences of up to so many rows (times query heads of a K/V head) are the small kernel's, whose tile of 16 rows costs them nothing but the memory's time; a second tile
// doubles its instructions. 24 sequences of up to 9000 positions, four query heads a K/V head: 3 and 4 rows (12 and 16 in all) 95 and 98 us there against
// 118 and 118 on tensor memory, 5 and 8 rows (20 and 32) 144 and 156 against 118 and 118.
constexpr int PA_FEW_ROWS = 16;
// The same of the small kernel for bytes, whose tiles have 8, 16 or 24 rows: the 24 sequences at 3 and 4 rows (12 and 16 in all) 80 and 85 us, at 5 and 6 (20 and 24) 117 and 122, on tensor memory 155 to 159
// for any of these, 160 at 8 rows (32), where two small tiles take 208. 5 rows of 6 sequences of up to 600 18 us and 26, of 64 47 and 78, of one of 60 000 77 and 92 (3 rows 52 and 87).
constexpr int PB_FEW_ROWS = 24;

// What every operator asks of the cache and the batch; `scales`: those that may come with bytes (nullptr: an fp16 cache alone)
struct Refusal;
spyb_status paged_check_view(Refusal &no, const char *what, const spyb_paged_cache &c, const spyb_paged_batch &b, const spyb_paged_scales *scales = nullptr);
PagedView   paged_view(const spyb_paged_cache &c, const spyb_paged_batch &b);
PagedScales paged_scales_of(const spyb_paged_cache &c, const spyb_paged_scales &s);

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
struct PagedSeq { int row0, rows, first, kv, from; };   // first row and number of rows, position of the first row, positions that are there, and the first of them that this pass reads
struct PagedItem { int lo, hi, units; };          // positions [lo, hi) that some row of the tile sees (lo a multiple of ALIGN, or where own positions begin: of paged_shared_align, 16 to 128)

__host__ __device__ __forceinline__ int pmin(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int pmax(int a, int b) { return a < b ? b : a; }
// Positions are below 2^30: a window of as many hides nothing, and a position minus a window stays in 32 bits also for rows in front of position 0
inline int paged_window(int window) { return pmin(window, 1 << 30); }
__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedView &v, int s) {
    const int a = pmax(0, pmin(v.row_start[s], v.n_rows)), end = pmax(a, pmin(v.row_end[s], 1 << 24)), b = pmin(end, v.n_rows);
    const int kv = pmin(pmax(0, v.n_kv[s]), 1 << 30);
    return {a, b - a, kv - (end - a), pmin(kv, v.n_kv_most), v.from != nullptr ? v.from[s] : 0};
}
template <int UNIT, int ALIGN>
__host__ __device__ __forceinline__ PagedItem paged_item(const PagedAttention &p, const PagedSeq &q, int tile) {
    const int last = pmin(q.rows * p.group, (tile + 1) * p.tile_rows) - 1;
    const int i0 = (int)((unsigned)(tile * p.tile_rows) / (unsigned)p.group), i1 = (int)((unsigned)last / (unsigned)p.group);
    PagedItem t;
    t.hi = p.causal ? pmin(q.kv, q.first + i1 + 1) : q.kv;
    t.lo = p.causal && p.window > 0 ? pmax(0, q.first + i0 - p.window + 1) / ALIGN * ALIGN : q.from;   // (a window leaves nothing to share)
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

// What the first pass found for four elements of a row, into what the second one did (maxima in powers of two)
__device__ __forceinline__ void paged_join_pass(float4 &v, float &l, float m, float2 with, float4 u) {
    const float top = fmaxf(m, with.x), base = top == -INFINITY ? 0.f : top, f = exp2f(m - base), w = exp2f(with.x - base);
    v = make_float4(f * v.x + w * u.x, f * v.y + w * u.y, f * v.z + w * u.z, f * v.w + w * u.w);
    l = f * l + w * with.y;
}

// ---------------------------------------------------------------------------------------------- bytes
// Four signed bytes as fp16 numbers, without an error: the byte plus 128 is the low half of the mantissa of 1024 + it, and 1152 is taken off.
__device__ __forceinline__ uint32_t sub_1152(uint32_t h2) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h2), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ void halves_of(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w ^= 0x80808080u;
    lo = sub_1152(__byte_perm(w, 0x64646464u, 0x4140)); hi = sub_1152(__byte_perm(w, 0x64646464u, 0x4342));
}
// of two words, the pairs of bytes that have the same place
__device__ __forceinline__ void pairs_of(uint32_t a, uint32_t b, uint32_t (&h2)[4]) {
    a ^= 0x80808080u; b ^= 0x80808080u;
    const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
    h2[0] = sub_1152(__byte_perm(lo, 0x64646464u, 0x4140)); h2[1] = sub_1152(__byte_perm(lo, 0x64646464u, 0x4342));
    h2[2] = sub_1152(__byte_perm(hi, 0x64646464u, 0x4140)); h2[3] = sub_1152(__byte_perm(hi, 0x64646464u, 0x4342));
}
__device__ __forceinline__ float2 half2_bits(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }

// ---------------------------------------------------------------------------------------------- rows and elements
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

}  // namespace spyb
