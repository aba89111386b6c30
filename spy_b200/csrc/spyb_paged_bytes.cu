// Attention of few rows a sequence over 8-bit caches in pages.
// Half the bytes of fp16 a position and more instructions for each: what holds a warp is not the memory but its own work on a block, so everything here is about few registers (many warps) and few
// instructions a byte.
//   S^T = K Q^T and O^T += V^T P^T, mma.sync 16 x 8 x 16: positions or elements are the products' 16 rows, query rows their 8 columns. A tile of 8 rows - the single token of up to eight query heads -
//   costs half the products, scores and accumulators of one that has query rows in the 16.
//   Bytes become fp16 numbers without an error in registers (five instructions for four of K, six of V). A lane reads HD / 4 bytes of two positions of K and HD / 8 of four of V in
//   16-byte pieces: the products' inner order is the lane's own, the same for Q, whose elements it reads alike, and V's elements are where the accumulators' rows are.
//   Scales stay out of the products' operands: K's multiply scores (where scale and log2 e are a product anyway), V's the probabilities, in f32. So that no probability leaves fp16's range,
//   V's scales are taken against the largest so far, rounded up to a power of two; like the maximum of the scores it moves a few times at the start and hardly ever after.

#include "spyb_internal.h"
#include "spyb_paged.cuh"
#include "spyb_paged_rows.cuh"

namespace spyb {
namespace {

template <int HD> struct BytesShape {
    static constexpr int ROW = HD == 96 ? 128 : HD;                  // bytes of a position in shared memory
    static constexpr int SCALES = 2 * PR_BLOCK * ROW, STAGE = SCALES + PR_BLOCK * 4;
    static constexpr int STAGES = HD <= 64 ? 4 : 3;
    static constexpr int RING = PR_WARPS * STAGES * STAGE;
    static constexpr int PIECES = HD / 16;                           // 16-byte pieces of a position
    // where byte 16 c of position r lies: what a quarter of a warp reads at a time - two positions side by side, or every second one - lies in other banks
    static __device__ __forceinline__ int place(int r, int c) {
        if (HD > 64) { return r * ROW + ((c ^ (r & 7)) << 4); }
        if (HD == 64) { return (r >> 1) * 128 + ((((r ^ (r >> 2)) & 1) * 4 + (c ^ (r & 2))) << 4); }
        return r * ROW + (c << 4);
    }
};
template <int HD, int NT> struct BytesSmem {       // the ring; what the warps found: beside it for up to EARLY rows, in its place for more; the masks of the ring's stages
    using Shape = BytesShape<HD>;
    static constexpr int CTAS = NT == 1 ? 4 : NT == 2 ? 3 : 2;        // of an SM
    static constexpr int EARLY = NT == 1 && HD <= 64 ? 8 : 0, FOUND = PR_WARPS * 8 * NT * (HD + 2) * 4, RING = Shape::RING > FOUND ? Shape::RING : FOUND;
    static constexpr int MASKS = RING + PR_WARPS * EARLY * (HD + 2) * 4, BYTES = MASKS + PR_WARPS * Shape::STAGES * 4;
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
__device__ __forceinline__ uint32_t transposed(uint32_t x) {   // of an 8 x 8 matrix, two elements a lane
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float over_groups(float v, bool largest) {   // over the lanes that have the same query rows
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) { const float u = __shfl_xor_sync(0xffffffffu, v, o); v = largest ? fmaxf(v, u) : v + u; }
    return v;
}

// IN_PAGE: a block's positions lie in one page (pages of a multiple of 16, but for heads of 96)
template <int HD, int NT, bool IN_PAGE>
__global__ void __launch_bounds__(PR_WARPS * 32, BytesSmem<HD, NT>::CTAS) paged_bytes_kernel(const __grid_constant__ PagedAttention p) {
    using Shape = BytesShape<HD>;
    using Smem = BytesSmem<HD, NT>;
    constexpr int STAGES = Shape::STAGES, TILE = 8 * NT, STAGE = Shape::STAGE, V_AT = PR_BLOCK * Shape::ROW, PIECES = Shape::PIECES;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PagedPlanShared plan;
    __shared__ int last_one;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint32_t *there = reinterpret_cast<uint32_t *>(smem + Smem::MASKS) + warp * STAGES;
    const uint32_t ring = smem_u32(smem) + warp * STAGES * STAGE;
    pdl_launch_dependents();
    pdl_wait();
    PagedPlace at = paged_plan<PR_WARPS * 32, PR_UNIT, PR_BLOCK>(p, true, 1, plan);
    if (at.unit >= at.end) { return; }
    PagedSeq q = paged_seq(p.view, at.seq);
    int seq = at.seq, head = at.head, tile = at.tile, off = at.off;
    PagedItem it;
    int todo, ka, kb, n_block, packed;        // of the item that comes next: units of this CTA, positions [ka, kb), blocks of them; rows of the tile
    const int32_t *table;
    const uint8_t *kbase, *vbase;
    const uint32_t *sbase;
    auto describe = [&]() {
        it = paged_item<PR_UNIT, PR_BLOCK>(p, q, tile);
        todo = (int)min((int64_t)(it.units - off), at.end - at.unit);
        ka = it.lo + off * PR_UNIT; kb = min(it.hi, ka + todo * PR_UNIT);
        n_block = kb > ka ? (kb - ka + PR_BLOCK - 1) / PR_BLOCK : 0;
        packed = min(TILE, q.rows * p.group - tile * TILE);
        table = p.view.page_table + (int64_t)seq * p.view.table_stride;
        kbase = reinterpret_cast<const uint8_t *>(p.k) + head * p.view.head_stride; vbase = reinterpret_cast<const uint8_t *>(p.v) + head * p.view.head_stride;
        sbase = p.scales.pairs + head * p.scales.head_stride;
    };
    auto page_of = [&](int b) {              // page of block b, or (lanes 0..15 and 16..31 alike) of this lane's position in it; -1: none
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
        {
            const int r = lane & 15;                          // (lanes 0..15: the scales of a position each)
            const bool in = (mask >> r) & 1;
            const int64_t o = in ? p.scales.page_stride * page + p.scales.token_stride * (in_page + (IN_PAGE ? r : 0)) : 0;
            if (lane < 16) { cp_async4(dst + Shape::SCALES + r * 4, sbase + o, in); }
        }
        if constexpr (IN_PAGE) {
            constexpr int AT_ONCE = 32 / PIECES;              // (a row's pieces are lanes side by side)
            const int r0 = lane / PIECES, c = lane % PIECES;
            int64_t o = cell + r0 * p.view.token_stride + c * 16;
            const int64_t more = AT_ONCE * p.view.token_stride;
#pragma unroll
            for (int i = 0; i < PIECES / 2; ++i) {
                const int r = i * AT_ONCE + r0;
                const bool in = (mask >> r) & 1;
                const uint32_t d = dst + Shape::place(r, c);
                const int64_t from = in ? o : 0;
                cp_async16(d, kbase + from, in);
                cp_async16(d + V_AT, vbase + from, in);
                o += more;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PIECES / 2; ++i) {
                const int x = i * 32 + lane, r = x / PIECES, c = x - r * PIECES;
                const bool in = (mask >> r) & 1;
                const int64_t row = __shfl_sync(0xffffffffu, cell, r), o = in ? row + c * 16 : 0;
                const uint32_t d = dst + Shape::place(r, c);
                cp_async16(d, kbase + o, in);
                cp_async16(d + V_AT, vbase + o, in);
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
    uint32_t qf[NT][HD / 16][2];              // row g of each tile of eight, elements t HD / 4 on, four a product
    int pos[NT][2];                           // of rows 2 t, 2 t + 1
    auto start = [&]() {                      // the item's first blocks are on their way while its Q comes
        issued = 0;
        if (IN_PAGE) { ids_next = page_of(warp + lane * PR_WARPS); }
        page = next_page(warp);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            const int next = next_page(warp + (i + 1) * PR_WARPS);
            if (warp + i * PR_WARPS < n_block) { issue(warp + i * PR_WARPS, i, page); } else { cp_commit(); }
            page = next;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            {
                const int r = n * 8 + g, pr = tile * TILE + min(r, packed - 1);
                const int token = (int)((unsigned)pr / (unsigned)p.group), h = pr - token * p.group;
                const uint2 *src = reinterpret_cast<const uint2 *>(p.q + (int64_t)(q.row0 + token) * p.q_stride + (head * p.group + h) * HD) + t * (HD / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint2 x = r < packed ? src[ks] : make_uint2(0, 0);
                    qf[n][ks][0] = x.x; qf[n][ks][1] = x.y;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) { pos[n][e] = q.first + (int)((unsigned)(tile * TILE + min(n * 8 + 2 * t + e, packed - 1)) / (unsigned)p.group); }
        }
    };
    describe();
    start();
    for (;;) {
        const int pos_first = q.first + (int)((unsigned)(tile * TILE) / (unsigned)p.group), pos_last = q.first + (int)((unsigned)(tile * TILE + packed - 1) / (unsigned)p.group);
        float o[NT][HD / 16][4], mx[NT][2], sum[NT][2], base[NT][2], over[NT][2];   // (base: the maximum, or 0 for none; over: scores beyond it move the maximum)
        float unit = 1099511627776.f;             // one over the power of two that V's scales are taken against: 2^-40 at first, below the least scale
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mx[n][0] = mx[n][1] = over[n][0] = over[n][1] = -CUDART_INF_F; sum[n][0] = sum[n][1] = base[n][0] = base[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) { o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f; }
        }
        int stage = 0;
        for (int b = warp; b < n_block; b += PR_WARPS) {
            {
                const int ahead = b + (STAGES - 1) * PR_WARPS, next = next_page(ahead + PR_WARPS);
                const int to = stage == 0 ? STAGES - 1 : stage - 1;
                __syncwarp();
                if (ahead < n_block) { issue(ahead, to, page); } else { cp_commit(); }
                page = next;
            }
            cp_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t k_addr = ring + stage * STAGE, v_addr = k_addr + V_AT;
            const uint32_t mask = there[stage];
            const int j0 = ka + b * PR_BLOCK;
            const bool whole = mask == 0xffffu && (!p.causal || (j0 + PR_BLOCK - 1 <= pos_first && (p.window <= 0 || j0 > pos_last - p.window)));
            // scores of positions g and g + 8
            float sc[NT][4], v_scale[2], k_scale[2];
#pragma unroll
            for (int n = 0; n < NT; ++n) { sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f; }
            {
                uint32_t w0[HD / 16], w1[HD / 16];
                lds_row<Shape, HD / 4>(k_addr, g, t, w0);
                lds_row<Shape, HD / 4>(k_addr, g + 8, t, w1);
                const float2 s0 = half2_bits(lds32(k_addr + Shape::SCALES + g * 4)), s1 = half2_bits(lds32(k_addr + Shape::SCALES + g * 4 + 32));
                k_scale[0] = fmaf(s0.x, 0.f, s0.x * p.scale_log2); k_scale[1] = fmaf(s1.x, 0.f, s1.x * p.scale_log2);   // (an infinite one is NaN: its elements' infinities do not add up to one)
                v_scale[0] = s0.y; v_scale[1] = s1.y;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    uint32_t a[4];
                    halves_of(w0[ks], a[0], a[2]);
                    halves_of(w1[ks], a[1], a[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) { mma16816(sc[n], a, qf[n][ks][0], qf[n][ks][1]); }
                }
            }
            // against the maximum, in powers of two
            bool above = false, odd = false;                  // (odd: a scale of V is not finite)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float &x = sc[n][e];
                    x = fmaf(x, k_scale[e >> 1], -base[n][e & 1]);
                    if (!whole) {
                        const int jj = g + (e >> 1) * 8, d = pos[n][e & 1] - (j0 + jj);
                        const bool seen = ((mask >> jj) & 1) && (!p.causal || (d >= 0 && (p.window <= 0 || d < p.window)));
                        x = seen ? x : -CUDART_INF_F;
                    }
                    above |= x > over[n][e & 1];
                }
            }
            v_scale[0] *= unit; v_scale[1] *= unit;
            if (__any_sync(0xffffffffu, above || !(fmaxf(fabsf(v_scale[0]), fabsf(v_scale[1])) <= 1.f) || v_scale[0] != v_scale[0] || v_scale[1] != v_scale[1])) {
                const bool fine0 = fabsf(v_scale[0]) < CUDART_INF_F, fine1 = fabsf(v_scale[1]) < CUDART_INF_F;
                odd = __any_sync(0xffffffffu, !fine0 || !fine1);
                const float most = over_groups(fmaxf(fmaxf(fine0 ? fabsf(v_scale[0]) : 0.f, fine1 ? fabsf(v_scale[1]) : 0.f), 1.f), true);
                const uint32_t up = (__float_as_uint(most) + 0x7fffffu) & 0x7f800000u;      // the next power of two, 2^56 at most
                const float f_scale = __uint_as_float(0x7f000000u - up);                    // one over it
                unit *= f_scale; v_scale[0] *= f_scale; v_scale[1] *= f_scale;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = over_groups(fmaxf(sc[n][e], sc[n][2 + e]), true);
                        const bool  moves = v > over[n][e];
                        const float to = moves ? fmaxf(mx[n][e], base[n][e] + v) : mx[n][e], f = to == mx[n][e] ? 1.f : ex2(mx[n][e] - to);   // (2^-inf = 0 at the first)
                        const float from = base[n][e], f_o = f * f_scale;
                        mx[n][e] = to; sum[n][e] *= f;
                        base[n][e] = to == -CUDART_INF_F ? 0.f : to;
                        over[n][e] = to == -CUDART_INF_F ? to : 8.f;
                        sc[n][e] += from - base[n][e]; sc[n][2 + e] += from - base[n][e];
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) { o[n][i][e] *= f_o; o[n][i][2 + e] *= f_o; }
                    }
                }
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float a = ex2(sc[n][2 * hf]), c = ex2(sc[n][2 * hf + 1]);
                    sum[n][0] += a; sum[n][1] += c;
                    float u = a * v_scale[hf], w = c * v_scale[hf];
                    if (odd) {                                // what is not seen is 0 whatever its scale is
                        u = sc[n][2 * hf] == -CUDART_INF_F ? 0.f : u;
                        w = sc[n][2 * hf + 1] == -CUDART_INF_F ? 0.f : w;
                    }
                    pf[n][hf] = transposed(pack2(u, w));
                }
            }
            // a lane has elements g HD / 8 on of positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9: the i-th product's rows g and g + 8 are elements 2 i and 2 i + 1 of these
            uint32_t vw[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) { lds_row<Shape, HD / 8>(v_addr, (i >> 1) * 8 + t * 2 + (i & 1), g, vw[i]); }
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {
                uint32_t b0[4], b1[4];
                pairs_of(vw[0][w], vw[1][w], b0);
                pairs_of(vw[2][w], vw[3][w], b1);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t a[4] = {b0[2 * i], b0[2 * i + 1], b1[2 * i], b1[2 * i + 1]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) { mma16816(o[n][2 * w + i], a, pf[n][0], pf[n][1]); }
                }
            }
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        cp_wait<0>();
        __syncwarp();
        // What is known of this item; the next one's copies start before its findings are joined, where these have a place of their own
        const RowsDone what = {packed, tile, q.row0, head, q.from};
        const PagedCut cut = paged_cut(at, at.unit - off, it.units);
        at.unit += todo + p.start_units;
        off = 0;
        const bool more = at.unit < at.end && paged_next(p, true, q, seq, head, tile), early = what.rows <= Smem::EARLY;
        if (more) { describe(); }
        if (more && early) { start(); }
        if (!early) { __syncthreads(); }
        const int room = early ? Smem::EARLY : TILE;              // rows of a warp's findings
        float *mo = reinterpret_cast<float *>(smem + (early ? Smem::RING : 0)), *mm = mo + PR_WARPS * room * HD, *ml = mm + PR_WARPS * room;
        const float f = 1.f / unit;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float l = over_groups(sum[n][e], false);
                const int r = n * 8 + 2 * t + e;
                if (r < what.rows) {
                    float *dst = mo + (warp * room + r) * HD + g * (HD / 8);
#pragma unroll
                    for (int i = 0; i < HD / 16; i += 2) { *reinterpret_cast<float4 *>(dst + 2 * i) = make_float4(o[n][i][e] * f, o[n][i][2 + e] * f, o[n][i + 1][e] * f, o[n][i + 1][2 + e] * f); }
                    if (g == 0) { mm[warp * room + r] = mx[n][e]; ml[warp * room + r] = l; }
                }
            }
        }
        __syncthreads();
        rows_finish<HD, TILE, PK_INT8>(p, cut, what, mo, mm, ml, room, last_one);
        if (!more) { return; }
        __syncthreads();                      // (the findings' place is free again)
        if (!early) { start(); }
    }
}

template <int HD, int NT, bool IN_PAGE>
cudaError_t launch_bytes_as(const PagedAttention &p, int sms, const LaunchCfg &cfg) {
    using Smem = BytesSmem<HD, NT>;
    const cudaError_t err = allow_dynamic_smem(reinterpret_cast<const void *>(paged_bytes_kernel<HD, NT, IN_PAGE>), (size_t)Smem::BYTES);
    if (err != cudaSuccess) { return err; }
    return launch_maybe_pdl(paged_bytes_kernel<HD, NT, IN_PAGE>, dim3(Smem::CTAS * sms), PR_WARPS * 32, (size_t)Smem::BYTES, cfg.stream, cfg.pdl, p);
}
template <int HD, int NT>
cudaError_t launch_bytes(PagedAttention p, int sms, const LaunchCfg &cfg) {
    const int page = p.view.page_size;
    p.page_shift = -1; p.start_units = PA_START;
    for (int s = 0; s < 31; ++s) { if (page == 1 << s) { p.page_shift = s; } }
    if constexpr (HD != 96) {
        if (page % PR_BLOCK == 0) { return launch_bytes_as<HD, NT, true>(p, sms, cfg); }
    }
    return launch_bytes_as<HD, NT, false>(p, sms, cfg);
}
template <int NT>
cudaError_t launch_bytes(const PagedAttention &p, int head_dim, int sms, const LaunchCfg &cfg) {
    switch (head_dim) {
    case 32: return launch_bytes<32, NT>(p, sms, cfg);
    case 64: return launch_bytes<64, NT>(p, sms, cfg);
    case 96: return launch_bytes<96, NT>(p, sms, cfg);
    case 128: return launch_bytes<128, NT>(p, sms, cfg);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_paged_attention_bytes(const PagedAttention &p, int head_dim, int sms, const LaunchCfg &cfg) {
    return p.tile_rows == 8 ? launch_bytes<1>(p, head_dim, sms, cfg) : p.tile_rows == 16 ? launch_bytes<2>(p, head_dim, sms, cfg) : launch_bytes<4>(p, head_dim, sms, cfg);
}

}  // namespace spyb
