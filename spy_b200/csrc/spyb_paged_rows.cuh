// Attention of few rows a sequence over caches in pages: the kernel for fp16 ones, and what it shares with the one for bytes.
#pragma once

#include <math_constants.h>

#include "spyb_paged.cuh"

namespace spyb {
namespace {

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

struct RowsDone { int rows, tile, row0, head, from; };   // an item's rows that this tile holds, its tile, the sequence's first row, K/V head, and where its own positions begin
// What WARPS warps of a CTA found for an item ([warp][room][HD], maxima, sums), joined and put where it goes: to the output, or where other CTAs have pieces of the item to the workspace, and by the
// last of these, in their order, to the output. All threads, behind a barrier.
template <int HD, int TILE, int KIND, int WARPS, class Meet>
__device__ __forceinline__ void rows_finish(const PagedAttention &p, const PagedCut &cut, const RowsDone &what, const float *mo, const float *mm, const float *ml, int room, int &last_one, const Meet &meet) {
    constexpr int PART = TILE * (HD + 2), NT = PR_WARPS * 32;
    const int tid = threadIdx.x, done = what.rows;
    float *part = p.partial + paged_slot(blockIdx.x, cut.c0) * PART;
    // what the first pass found for four elements is read one turn ahead
    const bool with = KIND != PK_PLAIN && p.with_stats != nullptr && what.from > 0;
    struct First { float2 stats; float4 sums; };
    auto first_pass = [&](int x) {
        First f = {make_float2(-CUDART_INF_F, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        if (KIND != PK_PLAIN && with && x < done * (HD / 4)) {
            const int r = x / (HD / 4), pr = what.tile * TILE + r, token = (int)((unsigned)pr / (unsigned)p.group);
            const int64_t cell = (int64_t)(what.row0 + token) * (p.n_head_kv * p.group) + what.head * p.group + pr - token * p.group;
            f.stats = p.with_stats[cell]; f.sums = *reinterpret_cast<const float4 *>(p.with_out + cell * HD + (x - r * (HD / 4)) * 4);
        }
        return f;
    };
    First next = first_pass(tid);
    auto put = [&](int r, int c, float4 v, float m, float l, const First &f) {   // four elements of a row, its maximum and sum
        const int pr = what.tile * TILE + r, token = (int)((unsigned)pr / (unsigned)p.group), g = pr - token * p.group;
        const int64_t o2 = (int64_t)(what.row0 + token) * p.out_stride + (what.head * p.group + g) * HD + c;
        if constexpr (KIND != PK_PLAIN) {
            const int64_t cell = (int64_t)(what.row0 + token) * (p.n_head_kv * p.group) + what.head * p.group + g;
            if (p.stats != nullptr) {
                if (c == 0) { p.stats[cell] = make_float2(m, l); }
                *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + o2) = v;
                return;
            }
            if (with) { paged_join_pass(v, l, m, f.stats, f.sums); }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float w[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
        if (p.out_f32) { store4(static_cast<float *>(p.out) + o2, w); } else { store4(static_cast<__half *>(p.out) + o2, w); }
    };
    for (int x = tid; x < done * (HD / 4); x += NT) {
        const int r = x / (HD / 4), c = (x - r * (HD / 4)) * 4;
        const First found = next;
        if (cut.parts == 1) { next = first_pass(x + NT); }
        float m = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { m = fmaxf(m, mm[w * room + r]); }
        const float base = m == -CUDART_INF_F ? 0.f : m;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = ex2(mm[w * room + r] - base);
            const float4 u = *reinterpret_cast<const float4 *>(mo + (w * room + r) * HD + c);
            v.x += f * u.x; v.y += f * u.y; v.z += f * u.z; v.w += f * u.w;
            l += f * ml[w * room + r];
        }
        if (cut.parts == 1) { put(r, c, v, m, l, found); }
        else {
            *reinterpret_cast<float4 *>(part + r * HD + c) = v;
            if (c == 0) { part[TILE * HD + r] = m; part[TILE * HD + TILE + r] = l; }
        }
    }
    if (cut.parts > 1) {
        meet();
        if (tid == 0) {
            if (KIND == PK_INT8) {            // (one instruction orders what the CTA wrote before it and what the last one reads after it; 64 single tokens of up to 4096 positions: 59.7 us, 60.1 with two fences)
                unsigned n;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(n) : "l"(p.arrived + cut.c0), "r"(1u) : "memory");
                last_one = n == (unsigned)cut.parts - 1;
                if (last_one) { p.arrived[cut.c0] = 0; }
            } else {
                __threadfence();
                const unsigned n = atomicAdd(p.arrived + cut.c0, 1u);
                last_one = n == (unsigned)cut.parts - 1;
                if (last_one) { p.arrived[cut.c0] = 0; __threadfence(); }
            }
        }
        meet();
        if (last_one) {
            for (int x = tid; x < done * (HD / 4); x += NT) {
                const int r = x / (HD / 4), c = (x - r * (HD / 4)) * 4;
                const First found = next;
                next = first_pass(x + NT);
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
                put(r, c, v, m, l, found);
            }
        }
    }
}

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
template <int HD, int MT, bool IN_PAGE, int KIND>
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
        const RowsDone what = {packed, tile, q.row0, head, q.from};
        const int done = packed;
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
        rows_finish<HD, TILE, KIND, PR_WARPS>(p, cut, what, mo, mm, ml, room, last_one, [] { __syncthreads(); });
        if (!more) { return; }
        __syncthreads();                      // (the findings' place is free again)
        if (!early) { start(); }
    }
}

template <int HD, int MT, bool IN_PAGE, int KIND>
cudaError_t launch_rows_as(const PagedAttention &p, int sms, const LaunchCfg &cfg) {
    const void *kernel = reinterpret_cast<const void *>(paged_rows_kernel<HD, MT, IN_PAGE, KIND>);
    const cudaError_t err = allow_dynamic_smem(kernel, (size_t)RowsSmem<HD, MT>::BYTES);
    if (err != cudaSuccess) { return err; }
    return launch_maybe_pdl(paged_rows_kernel<HD, MT, IN_PAGE, KIND>, dim3(RowsSmem<HD, MT>::CTAS * sms), PR_WARPS * 32, (size_t)RowsSmem<HD, MT>::BYTES, cfg.stream, cfg.pdl, p);
}
template <int HD, int MT, int KIND>
cudaError_t launch_rows(PagedAttention p, int sms, const LaunchCfg &cfg) {
    const int page = p.view.page_size;
    p.page_shift = -1; p.start_units = PA_START;
    for (int s = 0; s < 31; ++s) { if (page == 1 << s) { p.page_shift = s; } }
    if constexpr (HD <= 64) {
        if (page % PR_BLOCK == 0) { return launch_rows_as<HD, MT, true, KIND>(p, sms, cfg); }
    }
    return launch_rows_as<HD, MT, false, KIND>(p, sms, cfg);
}

template <int KIND>
cudaError_t launch_rows_kind(const PagedAttention &p, int head_dim, int row_tiles, int sms, const LaunchCfg &cfg) {
    switch (head_dim * 2 + row_tiles - 1) {
    case 64: return launch_rows<32, 1, KIND>(p, sms, cfg);
    case 65: return launch_rows<32, 2, KIND>(p, sms, cfg);
    case 128: return launch_rows<64, 1, KIND>(p, sms, cfg);
    case 129: return launch_rows<64, 2, KIND>(p, sms, cfg);
    case 192: return launch_rows<96, 1, KIND>(p, sms, cfg);
    case 193: return launch_rows<96, 2, KIND>(p, sms, cfg);
    case 256: return launch_rows<128, 1, KIND>(p, sms, cfg);
    case 257: return launch_rows<128, 2, KIND>(p, sms, cfg);
    default: return cudaErrorInvalidValue;
    }
}
}  // namespace
}  // namespace spyb
