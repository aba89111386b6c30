// Attention of few rows a sequence over 8-bit caches in pages.
// Half the bytes of fp16 a position and more instructions for each: what holds a warp is not the memory but its own work on a block, so everything here is about few registers (many warps) and few
// instructions a byte.
//   S^T = K Q^T and O^T += V^T P^T, mma.sync 16 x 8 x 16: positions or elements are the products' 16 rows, query rows their 8 columns. A tile of 8 rows - the single token of up to eight query heads -
//   costs half the products, scores and accumulators of one that has query rows in the 16.
//   Bytes become fp16 numbers without an error in registers (five instructions for four of K, six of V). A lane reads HD / 4 bytes of two positions of K and HD / 8 of four of V in
//   16-byte pieces: the products' inner order is the lane's own, the same for Q, whose elements it reads alike, and V's elements are where the accumulators' rows are.
//   Scales stay out of the products' operands: K's multiply scores (where scale and log2 e are a product anyway), V's the probabilities, in f32. What is rounded to fp16 is their product, the weight of a position: a
//   row's maximum is that of its scores plus log2 of V's scales, over what it sees, so that weights are rounded against the row's largest one, whatever the scales of other positions and other rows' are.
// Measured (heads of 128): 64 single tokens of up to 4096 positions, 32 query heads on 8 (277 MB), 61 us, 4.5 TB/s (heads of 64 52 us, 96 71, 32 41); three of 100 000, 40 on 8, 115 us, 5.3 TB/s, by head 108; one of 4000, 32 on 32 (33 MB),
// 15 us. Single tokens' loop runs at the memory's rate; beside it 7 us until the first stage is there (lengths, the plan, page table, bytes, one after the other) and 4 us for every item that is done, joins among them.
// Five rows of 24 sequences of up to 9000 (tiles of 24 rows) 117 us: 1.7 us a stage of 64 positions, a warp's chain of products and conversions with eight warps an SM (168 registers), and 5 us for a join.
// Slower: K by mma.sync on bytes, with Q as two bytes of a 16-bit number; bytes as 2^-24 times themselves with their 128 taken off the sums (8 %); 32 positions a warp at a time; two chains of scores; rings of four stages;
// what the warps found added up one after the other (61 -> 68 us); joins of two and four pieces of four elements at once (the same, and 2 %).

#include <cuda.h>

#include "spyb_internal.h"
#include "spyb_paged.cuh"
#include "spyb_paged_maps.h"
#include "spyb_paged_rows.cuh"
#include "spyb_tc.cuh"

namespace spyb {
namespace {

constexpr int PB_THREADS = (PR_WARPS + 1) * 32, PB_STAGE = PR_WARPS * PR_BLOCK;   // four warps that compute and one that copies; positions of a stage of the ring, 16 a warp
template <int HD> struct BytesShape {
    static constexpr int ROW = HD == 96 ? 128 : HD, TILE = PR_BLOCK * ROW;   // bytes of a position in shared memory, of 16
    static constexpr int V_AT = PB_STAGE * ROW, STAGE = 2 * V_AT;
    static constexpr int PIECES = HD / 16;                           // 16-byte pieces of a position
    // where byte 16 c of position r lies: the tensor maps' swizzles of 128 and 64 bytes
    static __device__ __forceinline__ int place(int r, int c) {
        return HD > 64 ? r * ROW + ((c ^ (r & 7)) << 4) : HD == 64 ? r * ROW + ((c ^ (r >> 1 & 3)) << 4) : r * ROW + (c << 4);
    }
};
// the ring, what the warps found, scales of the ring's stages
template <int HD, int NT> struct BytesSmem {
    using Shape = BytesShape<HD>;
    static constexpr int CTAS = NT == 1 ? 3 : 2;                     // of an SM
    static constexpr int STAGES = 3;
    static constexpr bool Q_SHARED = NT > 2;                         // Q's operands in shared memory, all warps' (they would not leave room for the sums in registers)
    static constexpr int FOUND = STAGES * Shape::STAGE, QUERY = FOUND + PR_WARPS * 8 * NT * (HD + 2) * 4, SCALES = QUERY + (Q_SHARED ? NT * HD * 16 : 0);
    static constexpr int BYTES = SCALES + STAGES * PB_STAGE * 4 + 1024;   // (+ alignment)
};
// N bytes of position r from byte N i on, as words
template <class Shape, int N> __device__ __forceinline__ void lds_row(uint32_t addr, int r, int i, uint32_t (&w)[N / 4]) {
    if constexpr (N % 16 == 0) {
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {
            const uint4 x = lds128(addr + Shape::place(r, i * (N / 16) + k));
            w[4 * k] = x.x; w[4 * k + 1] = x.y; w[4 * k + 2] = x.z; w[4 * k + 3] = x.w;
        }
    } else if constexpr (N % 8 == 0) {
#pragma unroll
        for (int k = 0; k < N / 8; ++k) {
            const int at = i * (N / 8) + k;
            const uint2 x = lds64(addr + Shape::place(r, at >> 1) + (at & 1) * 8);
            w[2 * k] = x.x; w[2 * k + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) { const int at = i * (N / 4) + k; w[k] = lds32(addr + Shape::place(r, at >> 2) + (at & 3) * 4); }
    }
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma_f(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // (not volatile: the compiler may move it)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // of an 8 x 8 matrix, two elements a lane
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float over_groups(float v, bool largest) {   // over the lanes that have the same query rows
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) { const float u = __shfl_xor_sync(0xffffffffu, v, o); v = largest ? fmaxf(v, u) : v + u; }
    return v;
}

__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void sts64(uint32_t addr, uint2 v) { asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory"); }
constexpr uint64_t PB_LANDING_NS = 1000000000;      // copies have this long to land (whatever the limit of the waits)
__device__ __noinline__ void stand_still(uint64_t ns) {
    const uint64_t t0 = global_timer_ns();
    for (int i = 0; i < (1 << 22) && global_timer_ns() - t0 < ns; ++i) { __nanosleep(200); }
}
__device__ __forceinline__ void tma_pages(uint32_t dst, const CUtensorMap *map, uint32_t bar, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3,%4,%5,%6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(token), "r"(head), "r"(page) : "memory");
}
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }   // of this lane's copies so far
// A CTA's part of an item, found by the copying warp for all: rows of the tile, stages of the ring, positions [ka, kb); rows 0: behind the last one
struct BytesEntry { int rows, n_stage, ka, kb, tile, head, row0, first, from, c0, parts; };
// What weights are taken against follows when one is 2^PB_SLACK times that: weights up to 2^15 are as exact in fp16 as those below 1
constexpr float PB_SLACK = 15.f;
constexpr float PB_LEAST = -24.f;             // log2 of the least scale; a scale of 0, or one that is not finite, counts as it (so that scores have a maximum, and sums of probabilities stay below 2^40 each)
constexpr int PB_ENTRIES = 4;                 // known ahead

// One warp copies for four that compute (with each its own copies a block's took a third of the warp's time on it: some hundred instructions of addresses).
// MAPS: K and V come by tensor maps, boxes of `box` positions that lie in one page (pages of a multiple of 16, heads of 64 and 128); otherwise by 16 bytes a lane.
template <int HD, int NT, bool MAPS>
__global__ void __launch_bounds__(PB_THREADS, BytesSmem<HD, NT>::CTAS) paged_bytes_kernel(const __grid_constant__ PagedAttention p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                                          const int box, int *error_flag, const uint64_t wait_limit) {
    using Shape = BytesShape<HD>;
    using Smem = BytesSmem<HD, NT>;
    constexpr int STAGES = Smem::STAGES, ROWS = 8 * NT, TILE = Shape::TILE, V_AT = Shape::V_AT, PIECES = Shape::PIECES;
    extern __shared__ uint8_t raw[];
    __shared__ PagedPlanShared plan;
    __shared__ int last_one;
    __shared__ uint64_t full_bars[STAGES], empty_bars[STAGES], known_bars[PB_ENTRIES], read_bars[PB_ENTRIES], joined_bar;
    __shared__ BytesEntry entries[PB_ENTRIES];
    __shared__ __align__(8) uint16_t there[STAGES][PR_WARPS];   // which positions of a stage are there
    uint8_t *const smem = raw + (-smem_u32(raw) & 1023);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t ring = smem_u32(smem), scales = ring + Smem::SCALES, full = smem_u32(full_bars), empty = smem_u32(empty_bars), known = smem_u32(known_bars), read = smem_u32(read_bars);
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(full + 8 * i, 33); mbar_init(empty + 8 * i, PR_WARPS); }
        mbar_init(smem_u32(&joined_bar), PR_WARPS);
        for (int i = 0; i < PB_ENTRIES; ++i) { mbar_init(known + 8 * i, 1); mbar_init(read + 8 * i, PR_WARPS); }
        mbar_init_fence();
    }
    if (MAPS && threadIdx.x == PR_WARPS * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    PagedPlace at = paged_plan<PB_THREADS, PB_STAGE, PB_STAGE>(p, true, 1, plan);
    if (at.unit >= at.end) { return; }
    uint64_t limit = wait_limit;              // (0: a wait of this warp has run out. It frees nothing and copies nothing any more, so the others' run out in turn)
    uint32_t stage = 0, phase = 0;
    auto advance = [&]() { if (++stage == STAGES) { stage = 0; phase ^= 1; } };
    if (warp == PR_WARPS) {
        // ---------------------------------------------------------------------------------- copies
        uint32_t issued = 0, entry = 0;
        PagedSeq q = paged_seq(p.view, at.seq);
        int seq = at.seq, head = at.head, tile = at.tile, off = at.off;
        auto put = [&](const BytesEntry &e) {                 // false: a wait has run out
            const uint32_t i = entry & (PB_ENTRIES - 1);
            mbar_wait_lean(read + 8 * i, ((entry / PB_ENTRIES) & 1) ^ 1, limit);
            if (!__all_sync(0xffffffffu, limit != 0)) { limit = 0; return false; }
            if (lane == 0) { entries[i] = e; mbar_arrive(known + 8 * i); }
            ++entry;
            return true;
        };
        for (bool more = true; more;) {
            const PagedItem it = paged_item<PB_STAGE, PB_STAGE>(p, q, tile);   // (stages begin where boxes do)
            const int todo = (int)min((int64_t)(it.units - off), at.end - at.unit), ka = it.lo + off * PB_STAGE, kb = min(it.hi, ka + todo * PB_STAGE), n_stage = kb > ka ? (kb - ka + PB_STAGE - 1) / PB_STAGE : 0;
            const PagedCut cut = paged_cut(at, at.unit - off, it.units);
            const BytesEntry e = {min(ROWS, q.rows * p.group - tile * ROWS), n_stage, ka, kb, tile, head, q.row0, q.first, q.from, cut.c0, cut.parts};
            if (!put(e)) { break; }
            const int32_t *table = p.view.page_table + (int64_t)seq * p.view.table_stride;
            const uint32_t *pairs = p.scales.pairs + head * p.scales.head_stride;
            const int seen_from = p.causal && p.window > 0 ? q.first + (int)((unsigned)(tile * ROWS) / (unsigned)p.group) - p.window + 1 : 0;   // what nobody sees is not there, its scales neither
            int page[2];                                      // of this lane's two positions of a stage, read a stage ahead. (No branch around the loads, or they are waited for where they stand)
            auto find = [&](int s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = min(ka + s * PB_STAGE + 32 * i + lane, kb - 1);
                    page[i] = table[p.page_shift >= 0 ? j >> p.page_shift : j / p.view.page_size];
                }
            };
            if (n_stage > 0) { find(0); }
            for (int s = 0; s < n_stage; ++s) {
                mbar_wait_lean(empty + 8 * stage, phase ^ 1, limit);
                if (!__all_sync(0xffffffffu, limit != 0)) { limit = 0; break; }
                if (p.late == PA_LATE_FEW && issued == 2) { stand_still(3 * wait_limit); }   // (the self-check's: issued all the same, with nobody waiting any more)
                const uint32_t bar = full + 8 * stage, dst = ring + stage * Shape::STAGE;
                int in[2], at[2];
                bool ok[2], seen[2];
                unsigned mask[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = ka + s * PB_STAGE + 32 * i + lane;
                    in[i] = p.page_shift >= 0 ? j & (p.view.page_size - 1) : j % p.view.page_size;
                    at[i] = page[i];
                    ok[i] = j < kb && at[i] >= 0 && at[i] < p.view.n_pages;
                    seen[i] = ok[i] && j >= seen_from;
                    mask[i] = __ballot_sync(0xffffffffu, seen[i]);
                }
                if (s + 1 < n_stage) { find(s + 1); }
                if (lane == 0) {
                    *reinterpret_cast<uint2 *>(there[stage]) = make_uint2(mask[0], mask[1]);
                    if (MAPS) { mbar_expect_tx(bar, Shape::STAGE); } else { mbar_arrive(bar); }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    cp_async4(scales + (stage * PB_STAGE + 32 * i + lane) * 4, pairs + (seen[i] ? at[i] * p.scales.page_stride + in[i] * p.scales.token_stride : 0), seen[i]);
                }
                if constexpr (MAPS) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = 32 * i + lane;
                        if ((r & (box - 1)) == 0) {           // (a box that is not there: a page behind the last one, which reads as zeros; positions behind kb are read, and masked)
                            const int from = ok[i] ? at[i] : p.view.n_pages, token = ok[i] ? in[i] : 0;
                            tma_pages(dst + r * Shape::ROW, &k_map, bar, token, head, from);
                            tma_pages(dst + V_AT + r * Shape::ROW, &v_map, bar, token, head, from);
                        }
                        __syncwarp();
                    }
                } else {
                    const uint8_t *kbase = reinterpret_cast<const uint8_t *>(p.k) + head * p.view.head_stride, *vbase = reinterpret_cast<const uint8_t *>(p.v) + head * p.view.head_stride;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int64_t cell = ok[h] ? at[h] * p.view.page_stride + in[h] * p.view.token_stride : 0;
#pragma unroll 2
                        for (int i = 0; i < PIECES; ++i) {
                            const int x = i * 32 + lane, r = x / PIECES, c = x - r * PIECES;
                            const bool is = (mask[h] >> r) & 1;
                            const int64_t from = __shfl_sync(0xffffffffu, cell, r), o = is ? from + c * 16 : 0;
                            const uint32_t d = dst + h * 32 * Shape::ROW + Shape::place(r, c);
                            cp_async16(d, kbase + o, is);
                            cp_async16(d + V_AT, vbase + o, is);
                        }
                    }
                }
                arrive_when_copied(bar);
                advance();
                ++issued;
            }
            if (limit == 0) { break; }
            at.unit += todo + p.start_units;
            off = 0;
            more = at.unit < at.end && paged_next(p, true, q, seq, head, tile);
        }
        if (limit != 0) { const BytesEntry over = {}; put(over); }
        // What is on its way lands before the CTA ends, also where those who waited for it have given up
        if (limit == 0 && lane == 0) { pf_report(error_flag, 7); }
        uint64_t again = PB_LANDING_NS;
        for (uint32_t i = 0; i < STAGES && i < issued; ++i) {
            if (stage == 0) { stage = STAGES; phase ^= 1; }
            --stage;
            mbar_wait_lean(full + 8 * stage, phase, again);
        }
        return;
    }
    // -------------------------------------------------------------------------------------- scores, probabilities, sums
    const int g = lane >> 2, t = lane & 3;
    uint2 qf[Smem::Q_SHARED ? 1 : NT][HD / 16];   // row g of each tile of eight, elements t HD / 4 on, four a product
    const uint32_t q_at = ring + Smem::QUERY + lane * 8;   // or [tile][product][lane]
    int pos[NT][2];                           // of rows 2 t, 2 t + 1
    uint32_t entry = 0, joined_phase = 0;
    auto meet = [&]() {                       // the four warps (a barrier whose wait ends: one of them may have given up)
        __syncwarp();
        if (lane == 0) { mbar_arrive(smem_u32(&joined_bar)); }
        mbar_wait_lean(smem_u32(&joined_bar), joined_phase, limit);
        if (!__all_sync(0xffffffffu, limit != 0)) { limit = 0; }
        joined_phase ^= 1;
    };
    BytesEntry e;
    auto next = [&]() {                       // the next item and its Q; false behind the last one, or when a wait has run out
        const uint32_t i = entry & (PB_ENTRIES - 1);
        mbar_wait_lean(known + 8 * i, (entry / PB_ENTRIES) & 1, limit);
        if (!__all_sync(0xffffffffu, limit != 0)) { limit = 0; return false; }
        e = entries[i];
        ++entry;
        __syncwarp();
        if (lane == 0) { mbar_arrive(read + 8 * i); }
        if (e.rows == 0) { return false; }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (!Smem::Q_SHARED || n % PR_WARPS == warp) {
                const int r = n * 8 + g, pr = e.tile * ROWS + min(r, e.rows - 1);
                const int token = (int)((unsigned)pr / (unsigned)p.group), h = pr - token * p.group;
                const uint2 *src = reinterpret_cast<const uint2 *>(p.q + (int64_t)(e.row0 + token) * p.q_stride + (e.head * p.group + h) * HD) + t * (HD / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint2 x = r < e.rows ? src[ks] : make_uint2(0, 0);
                    if (Smem::Q_SHARED) { sts64(q_at + (n * (HD / 16) + ks) * 256, x); } else { qf[Smem::Q_SHARED ? 0 : n][ks] = x; }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) { pos[n][i] = e.first + (int)((unsigned)(e.tile * ROWS + min(n * 8 + 2 * t + i, e.rows - 1)) / (unsigned)p.group); }
        }
        if (Smem::Q_SHARED) { meet(); }
        return true;
    };
    while (next()) {
        const int first_row = e.tile * ROWS, pos_first = e.first + (int)((unsigned)first_row / (unsigned)p.group), pos_last = e.first + (int)((unsigned)(first_row + e.rows - 1) / (unsigned)p.group);
        float o[NT][HD / 16][4], mx[NT][2], sum[NT][2], base[NT][2], over[NT][2];   // (mx: of the weights, in powers of two; base: that, or 0 for none; over: weights beyond it move the maximum)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mx[n][0] = mx[n][1] = over[n][0] = over[n][1] = -CUDART_INF_F; sum[n][0] = sum[n][1] = base[n][0] = base[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) { o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f; }
        }
        for (int s = 0; s < e.n_stage; ++s) {
            mbar_wait_lean(full + 8 * stage, phase, limit);
            if (!__all_sync(0xffffffffu, limit != 0)) { limit = 0; break; }
            const uint32_t k_addr = ring + stage * Shape::STAGE + warp * TILE, v_addr = k_addr + V_AT, s_addr = scales + (stage * PB_STAGE + warp * PR_BLOCK) * 4;
            const uint32_t mask = there[stage][warp];
            const int j0 = e.ka + s * PB_STAGE + warp * PR_BLOCK;
            const bool whole = mask == 0xffffu && (!p.causal || (j0 + PR_BLOCK - 1 <= pos_first && (p.window <= 0 || j0 > pos_last - p.window)));
            // scores of positions g and g + 8
            float sc[NT][4], v_scale[2], v_log[2], k_scale[2];
            {
#pragma unroll
                for (int n = 0; n < NT; ++n) { sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f; }
                uint32_t w0[HD / 16], w1[HD / 16];
                lds_row<Shape, HD / 4>(k_addr, g, t, w0);
                lds_row<Shape, HD / 4>(k_addr, g + 8, t, w1);
                const float2 s0 = half2_bits(lds32(s_addr + g * 4)), s1 = half2_bits(lds32(s_addr + (g + 8) * 4));
                k_scale[0] = fmaf(s0.x, 0.f, s0.x * p.scale_log2); k_scale[1] = fmaf(s1.x, 0.f, s1.x * p.scale_log2);   // (an infinite one is NaN: its elements' infinities do not add up to one)
                v_scale[0] = s0.y; v_scale[1] = s1.y;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    uint32_t a[4];
                    halves_of(w0[ks], a[0], a[2]);
                    halves_of(w1[ks], a[1], a[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 b = Smem::Q_SHARED ? lds64(q_at + (n * (HD / 16) + ks) * 256) : qf[Smem::Q_SHARED ? 0 : n][ks];
                        mma_f(sc[n], a, b.x, b.y);
                    }
                }
            }
            // against the maximum, in powers of two
            bool above = false, odd = false;                  // (odd: a scale of V is not finite)
            {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float size = fabsf(v_scale[i]);
                    const bool is = size < CUDART_INF_F;
                    v_log[i] = is ? fmaxf(lg2(size), PB_LEAST) : PB_LEAST;
                    above |= !is;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &x = sc[n][i];
                        x = fmaf(x, k_scale[i >> 1], -base[n][i & 1]);
                        if (!whole) {
                            const int jj = g + (i >> 1) * 8, d = pos[n][i & 1] - (j0 + jj);
                            const bool seen = ((mask >> jj) & 1) && (!p.causal || (d >= 0 && (p.window <= 0 || d < p.window)));
                            x = seen ? x : -CUDART_INF_F;
                        }
                        above |= x + v_log[i >> 1] > over[n][i & 1];
                    }
                }
            }
            if (__any_sync(0xffffffffu, above)) {
                odd = !__all_sync(0xffffffffu, fabsf(v_scale[0]) < CUDART_INF_F && fabsf(v_scale[1]) < CUDART_INF_F);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float v = fmaxf(sc[n][i] + v_log[0], sc[n][2 + i] + v_log[1]);
                        v = over_groups(v, true);
                        const float to = v > over[n][i] ? fmaxf(mx[n][i], base[n][i] + v) : mx[n][i], f = to == mx[n][i] ? 1.f : ex2(mx[n][i] - to);   // (2^-inf = 0 at the first)
                        const float from = base[n][i];
                        mx[n][i] = to; sum[n][i] *= f;
                        base[n][i] = to == -CUDART_INF_F ? 0.f : to;
                        over[n][i] = to == -CUDART_INF_F ? to : PB_SLACK;
                        sc[n][i] += from - base[n][i]; sc[n][2 + i] += from - base[n][i];
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) { o[n][k][i] *= f; o[n][k][2 + i] *= f; }
                    }
                }
            }
            {
                uint32_t pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float a = ex2(sc[n][2 * hf]), c = ex2(sc[n][2 * hf + 1]);
                        sum[n][0] += a; sum[n][1] += c;
                        float x = a * v_scale[hf], y = c * v_scale[hf];
                        if (odd) {                            // what is not seen is 0 whatever its scale is
                            x = sc[n][2 * hf] == -CUDART_INF_F ? 0.f : x;
                            y = sc[n][2 * hf + 1] == -CUDART_INF_F ? 0.f : y;
                        }
                        pf[n][hf] = transposed(pack2(x, y));
                    }
                }
                // a lane has elements g HD / 8 on of positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9: the i-th product's rows g and g + 8 are elements 2 i and 2 i + 1 of these
                uint32_t vw[4][HD / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) { lds_row<Shape, HD / 8>(v_addr, (i >> 1) * 8 + t * 2 + (i & 1), g, vw[i]); }
                __syncwarp();
                if (lane == 0) { mbar_arrive(empty + 8 * stage); }
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) {
                    uint32_t b0[4], b1[4];
                    pairs_of(vw[0][w], vw[1][w], b0);
                    pairs_of(vw[2][w], vw[3][w], b1);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a[4] = {b0[2 * i], b0[2 * i + 1], b1[2 * i], b1[2 * i + 1]};
#pragma unroll
                        for (int n = 0; n < NT; ++n) { mma_f(o[n][2 * w + i], a, pf[n][0], pf[n][1]); }
                    }
                }
            }
            advance();
        }
        // This warp's findings (the next item's copies are on their way)
        float *mo = reinterpret_cast<float *>(smem + Smem::FOUND), *mm = mo + PR_WARPS * ROWS * HD, *ml = mm + PR_WARPS * ROWS;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float l = over_groups(sum[n][i], false);
                const int r = n * 8 + 2 * t + i;
                if (r < e.rows) {
                    float *dst = mo + (warp * ROWS + r) * HD + g * (HD / 8);
#pragma unroll
                    for (int k = 0; k < HD / 16; k += 2) { *reinterpret_cast<float4 *>(dst + 2 * k) = make_float4(o[n][k][i], o[n][k][2 + i], o[n][k + 1][i], o[n][k + 1][2 + i]); }
                    if (g == 0) { mm[warp * ROWS + r] = mx[n][i]; ml[warp * ROWS + r] = l; }
                }
            }
        }
        meet();
        const RowsDone what = {e.rows, e.tile, e.row0, e.head, e.from};
        rows_finish<HD, ROWS, PK_INT8, PR_WARPS>(p, PagedCut{e.c0, e.parts}, what, mo, mm, ml, ROWS, last_one, meet);
        meet();                               // (the findings' place is free again)
    }
    if (limit == 0 && lane == 0) { pf_report(error_flag, 7); }
}

template <int HD, int NT, bool MAPS>
cudaError_t launch_bytes_as(const PagedAttention &p, const CUtensorMap &k, const CUtensorMap &v, int box, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    using Smem = BytesSmem<HD, NT>;
    const cudaError_t err = allow_dynamic_smem(reinterpret_cast<const void *>(paged_bytes_kernel<HD, NT, MAPS>), (size_t)Smem::BYTES);
    if (err != cudaSuccess) { return err; }
    return launch_maybe_pdl(paged_bytes_kernel<HD, NT, MAPS>, dim3(Smem::CTAS * sms), PB_THREADS, (size_t)Smem::BYTES, cfg.stream, cfg.pdl, p, k, v, box, cfg.error_flag, wait_limit);
}
template <int HD, int NT>
cudaError_t launch_bytes(PagedAttention p, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    const int page = p.view.page_size;
    p.page_shift = -1; p.start_units = PA_START;
    for (int s = 0; s < 31; ++s) { if (page == 1 << s) { p.page_shift = s; } }
    CUtensorMap k = {}, v = {};
    if constexpr (HD == 64 || HD == 128) {
        const int box = page % 64 == 0 ? 64 : page % 32 == 0 ? 32 : 16;
        if (page % 16 == 0 && paged_byte_map(&k, p.k, p.view, p.n_head_kv, HD, box) && paged_byte_map(&v, p.v, p.view, p.n_head_kv, HD, box)) { return launch_bytes_as<HD, NT, true>(p, k, v, box, sms, cfg, wait_limit); }
    }
    return launch_bytes_as<HD, NT, false>(p, k, v, 0, sms, cfg, wait_limit);
}
template <int NT>
cudaError_t launch_bytes(const PagedAttention &p, int head_dim, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    switch (head_dim) {
    case 32: return launch_bytes<32, NT>(p, sms, cfg, wait_limit);
    case 64: return launch_bytes<64, NT>(p, sms, cfg, wait_limit);
    case 96: return launch_bytes<96, NT>(p, sms, cfg, wait_limit);
    case 128: return launch_bytes<128, NT>(p, sms, cfg, wait_limit);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_paged_attention_bytes(const PagedAttention &p, int head_dim, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    return p.tile_rows == 8 ? launch_bytes<1>(p, head_dim, sms, cfg, wait_limit) : p.tile_rows == 16 ? launch_bytes<2>(p, head_dim, sms, cfg, wait_limit) : launch_bytes<3>(p, head_dim, sms, cfg, wait_limit);
}

}  // namespace spyb
