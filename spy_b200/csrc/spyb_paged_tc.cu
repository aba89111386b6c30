// Attention of many rows a sequence (chunks of prompts, groups of query heads) over paged caches on the tcgen05 tensor cores.
//
// Rows and positions go in tiles: up to 256 rows - two tiles of as many whole tokens (with all query heads of the K/V head) as 128 rows hold, each with a warpgroup of its
// own - against 128 positions at a time. S = Q K^T and O += P V are
// tcgen05 MMAs, 128 x 128 x 16 and 128 x head_dim x 16; S, P (fp16, in place of S) and O live in tensor memory, a row a lane, so that a row's maximum and sum stay in
// one thread. While one tile's probabilities are made (16 powers of two a clock and SM, as many clocks as its two products take), the other tile's
// products run. K and V come page by page through tensor maps, in pieces of as many positions as divide the page size, into the 128-byte
// swizzle of the operands: K row by row (K-major), V as it lies (its positions are the product's inner dimension: MN-major), no transposition anywhere.
//   warps 0-3, 4-7   probabilities of tile 0 / 1, rescaling, output          warp 8   issues the MMAs
//   warp 9           copies                                                   warps 10, 11  Q; clear and check the V tiles that not all rows see whole
//   warps 12-15      (8-bit caches) make the operands of K and V: bytes land in a ring of their own, as whole numbers in fp16
// Probabilities are taken against a maximum that follows the true one when that is 2^8 above it: O is rescaled in the first steps and hardly ever after.
// Measured (heads of 128): 8192 tokens of a prompt, 32 heads, 570 us, 965 TFLOP/s of the 1640 of a matrix product; 512 tokens at 32 768 positions 281 us, 970;
// 1500 at 9111, 40 heads, 247 us, 1040; 512 at 3968 52 to 55 us, 595; five tokens of 24 sequences of up to 9000, 111 us, 4.2 TB/s. Heads of 64 have half the
// products for as many powers: 8192 tokens 524 us, 524 TFLOP/s. A step of 256 rows and 128 positions takes 2.4 us, in which 16 powers a clock alone take 1.1; the chain of
// a tile - S, reading it, maximum, powers, P, product - is what bounds it, two tiles hide each other's. Beside the steps: 7 us until the first (lengths, the plan, page
// table, Q and K), 5 us from one stretch to the next and 6 for the join of an item on a cut, which is what holds short contexts back (512 tokens at 1024: 28 us).
// Bytes: 1500 tokens at 9111 392 us, 657 TFLOP/s; 512 at 32 768 408; heads of 64, 4096 tokens 222; five tokens of 24 sequences 158. Shared memory has more to do: operands are read as bytes and written as halves, and every row reads every position's two scales;
// the probabilities' warps have 192 registers in place of 208. (Operands that are rounded products byte x scale: 331 us, and three times the error.)
// Tried and left out: powers by polynomials on the FMA units for some of the columns (slower: their instructions are what is short), the two tiles taking turns by
// barriers (no gain), both tiles on one tile's rows by every second step where only one has rows (24 x 5 rows 122 us against 119: memory bounds those steps).

#include <algorithm>
#include <type_traits>

#include <cuda.h>
#include <math_constants.h>

#include "spyb_internal.h"
#include "spyb_paged.cuh"
#include "spyb_paged_maps.h"
#include "spyb_tc.cuh"

namespace spyb {
namespace {

constexpr int PT_ROWS = 128, PT_KEYS = 128;
constexpr float PT_LEAST = -24.f;                        // log2 of the least scale of bytes; one of 0, or that is not finite, counts as it
constexpr uint32_t PT_HALF = PT_KEYS * 128;              // bytes of 128 rows x 64 elements

template <int HD, int KIND> struct TcShape {
    static constexpr uint32_t OPERAND = PT_KEYS * HD * 2;                      // a tile of Q, K or V
    static constexpr bool BYTES = KIND == PK_INT8;
    static constexpr int THREADS = BYTES ? 512 : 384, READERS = BYTES ? 15 : 11;   // (readers of an entry: eight warps for probabilities, one for MMAs, two for Q and V, four for bytes)
    static constexpr int REGS_SOFTMAX = BYTES ? 192 : 208, REGS_OTHERS = BYTES ? 64 : 88;   // 256 x 208 + 128 x 88 = 384 x 168, 256 x 192 + 256 x 64 = 512 x 128: what the block is launched with
    static constexpr float SLACK = BYTES ? 15.f : 8.f;                         // powers of two that weights may be above what they are taken against: up to 2^15 they are as exact in fp16 as below 1
    static constexpr int SLOTS = BYTES ? (HD == 128 ? 3 : 4) : HD == 128 ? 5 : 8;   // K and V tiles in flight; of bytes: made into operands ahead
    static constexpr int BYTE_SLOTS = BYTES ? (HD == 128 ? 3 : 6) : 0;         // tiles of bytes in flight
    static constexpr uint32_t BYTE_TILE = PT_KEYS * HD;
    static constexpr int Q_BUFFERS = HD == 128 ? 1 : 2;                        // (heads of 64: the next stretch's Q comes while this one's is in use; there is room for it)
    static constexpr uint32_t SMEM = (2 * Q_BUFFERS + SLOTS) * OPERAND + BYTE_SLOTS * BYTE_TILE + 1024; // (+ alignment)
    // tensor memory: S of both tiles, then O of both; P over S, or for heads of 64, whose O leaves room, beside it: the next S is made while P is
    static constexpr bool P_APART = HD == 64;
    static constexpr uint32_t P_COLUMN = P_APART ? 256 : 0, P_STEP = P_APART ? 64 : 128, O_COLUMN = P_APART ? 384 : 256;
};
struct Tile {
    int rows, pos_first, pos_last;                   // of up to 128 rows: how many there are, positions of the first and the last
    int from, to;                                    // steps (of the item) in which it sees anything, within the stretch
};
// One stretch of an item: `todo` steps of 128 positions from step `off` of the item on (todo = 0: behind the last one). The copying warp finds them one after the other
// for all roles.
struct Entry {
    int todo, off, lo, hi;                           // positions [lo, hi) of the item
    int seq, head, tile, row0, first;                // first row of the sequence, its position
    int begin, end;                                  // steps in which either tile sees something: one run, for the second one's positions begin at the first one's end at the latest
    int c0, parts;                                   // the CTAs of the item
    Tile half[2];
    // all rows of a tile see all positions of the step (if their pages are there)
    __device__ __forceinline__ bool whole(const PagedAttention &p, const Tile &h, int step) const {
        const int j = lo + step * PT_KEYS;
        return j + PT_KEYS <= hi && (!p.causal || (j + PT_KEYS - 1 <= h.pos_first && (p.window <= 0 || j > h.pos_last - p.window)));
    }
};
// A lane whose wait has run out (its limit is 0 then) frees nothing any more: no slot that a copy may still be on its way to is filled again, no entry that somebody may
// still read is written over. The other roles' waits run out in turn, so that every role ends by itself, and then who issued copies or products waits for their end, whoever
// it was that gave up. (Waiting for it in every case, at the end of each role, cost 5 % of prompts of heads of 64.)
constexpr uint64_t PT_LANDING_NS = 1000000000;       // what is on its way has this long to land (whatever the limit of the waits)
constexpr int PT_ENTRIES = 4;                        // stretches known ahead
// 8-bit caches, of the last four steps: K's scales with what scores are scaled by anyway, V's and the logarithms of their sizes, and the exponents of powers of two that V's are not above, by the warps that read them
template <int KIND> struct ByteScales {};
template <> struct __align__(16) ByteScales<PK_INT8> { float k[4][PT_KEYS], v[4][PT_KEYS], v_log[4][PT_KEYS], v_top[4][4]; };
template <int KIND> struct TcShared {
    uint64_t full[8], empty[8];                          // a slot's copies have landed; its last MMA is done, and both warps that check V have seen its phase
    uint64_t clean[8];                                   // of the last V tiles: what nobody sees is cleared
    ByteScales<KIND> scale;
    uint64_t byte_full[8], byte_empty[8];                // 8-bit caches: a tile of bytes has landed; its operand is made (`full` is that operand's, `empty` its last MMA's)
    uint64_t q_ready[2][2], q_free[2][2];                // of the two tiles and their buffers, in stretches in which they see anything
    uint64_t s_ready[2], s_free[2], p_ready[2][2], p_free[2], o_ready[2];   // (P ready) of the first 96 positions and the rest; (free) where P lies apart
    uint64_t known[PT_ENTRIES], read[PT_ENTRIES];        // an entry is there; all have read it
    uint64_t joined[2];                                  // all threads of a tile have come so far
    uint64_t over;                                       // (something gave up) the last MMA is done
    uint32_t tmem;
    uint32_t there[8];                                   // of the last tiles: which groups of eight positions are there
    int      poison[8];                                  // of the last stretches: a V tile that some rows see in part holds values that are not finite
    int      last[2];
    int      gave_up;                                    // a wait of some warp has run out
    Entry    entry[PT_ENTRIES];
    PagedPlanShared plan;
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int token, int head, int page) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3,%4,%5,%6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(token), "r"(head), "r"(page) : "memory");
}
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int head, int row) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3,%4,%5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(head), "r"(row) : "memory");
}
// operands in the 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart; `far`: from one 64-element half of an MN-major operand to the next
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t addr, uint32_t far) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(far >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
#define SPYB_R32(r) "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), \
    "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), \
    "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define SPYB_I32(r) "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), \
    "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), \
    "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : SPYB_R32(r) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                   "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float log2_fast(float x) { float y; asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) { uint32_t r; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
__device__ __forceinline__ uint32_t not_finite(uint32_t h2) { return ((h2 & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
// A wait by a whole warp. Its lanes may see the phase's end at different times, and what follows - an elected lane, tensor-memory accesses - is the whole warp's:
// two groups of lanes would elect one each, and products and their completions would count twice.
__device__ __forceinline__ void wait_for(uint32_t bar, uint32_t parity, uint64_t &limit) {
    mbar_wait_lean(bar, parity, limit);
    __syncwarp();
}
struct Walker {                                      // the copying warp's place in the work
    PagedSeq  q;
    PagedPlace at;
    int seq, head, tile, off;

    __device__ __forceinline__ Tile half(const PagedAttention &p, const Entry &e, int t) const {
        Tile h;
        const int r0 = tile * p.tile_rows + t * (p.tile_rows / 2);
        h.rows = max(0, min(p.tile_rows / 2, q.rows * p.group - r0));
        h.pos_first = q.first + (int)((unsigned)r0 / (unsigned)p.group);
        h.pos_last = q.first + (int)((unsigned)(r0 + max(h.rows, 1) - 1) / (unsigned)p.group);
        const int hi = p.causal ? min(e.hi, h.pos_last + 1) : e.hi, lo = p.causal && p.window > 0 ? max(e.lo, h.pos_first - p.window + 1) : e.lo;
        h.from = max(off, (lo - e.lo) / PT_KEYS);
        h.to = h.rows == 0 || hi <= e.lo ? off : min(off + e.todo, (hi - e.lo + PT_KEYS - 1) / PT_KEYS);
        if (h.to <= h.from) { h.from = h.to = off; }
        return h;
    }
    __device__ __forceinline__ Entry entry(const PagedAttention &p) const {
        const PagedItem it = paged_item<PT_KEYS, PT_KEYS>(p, q, tile);
        Entry e;
        e.todo = (int)min((int64_t)(it.units - off), at.end - at.unit);
        e.off = off; e.lo = it.lo; e.hi = it.hi; e.seq = seq; e.head = head; e.tile = tile; e.row0 = q.row0; e.first = q.first;
        const Tile a = half(p, e, 0), b = half(p, e, 1);
        e.half[0] = a; e.half[1] = b;
        e.begin = a.to <= a.from ? b.from : b.to <= b.from ? a.from : min(a.from, b.from);
        e.end = a.to <= a.from ? b.to : b.to <= b.from ? a.to : max(a.to, b.to);
        const PagedCut cut = paged_cut(at, at.unit - off, it.units);
        e.c0 = cut.c0; e.parts = cut.parts;
        return e;
    }
    __device__ __forceinline__ bool next(const PagedAttention &p, int todo) {
        at.unit += todo + p.start_units;
        if (at.unit >= at.end) { return false; }
        off = 0;
        return paged_next(p, false, q, seq, head, tile);
    }
};

__device__ __noinline__ void stand_still(uint64_t ns) {
    const uint64_t t0 = global_timer_ns();
    for (int i = 0; i < (1 << 22) && global_timer_ns() - t0 < ns; ++i) { __nanosleep(200); }
}

// LATE: the self-checks' kernels (p.late)
// Bytes of 32 positions (row0 on) of a tile as an operand: whole numbers, without an error (scales are for scores and probabilities, in f32: rounded products of both would cost a score some 2^-12 of
// its terms, three times the error of the whole). A lane has 16 bytes at a time, four lanes 64 bytes of a row: eight lanes, whose reads and writes are one turn of the banks each, have two rows that both
// the bytes' swizzle and the operand's send to different banks (heads of 128: r and r ^ 5). Places do not change from one group of eight rows to the next, so that they are made once a tile.
template <int HD> __device__ __forceinline__ void make_operand(uint32_t bytes, uint32_t operand, int row0) {
    constexpr int STEPS = HD == 128 ? 2 : 1;                           // a warp's turns for eight rows
    const int lane = threadIdx.x & 31, c = lane & 3;
    uint32_t src[STEPS], dst[STEPS];
#pragma unroll
    for (int e = 0; e < STEPS; ++e) {
        const int first = HD == 128 ? 2 * e + (lane >> 4) : lane >> 2, half = HD == 128 ? lane >> 3 & 1 : 0, row = HD == 128 && (lane & 4) ? first ^ 5 : first;
        src[e] = bytes + (row0 + row) * HD + (HD == 128 ? ((4 * half + c) ^ row) << 4 : c << 4);
        dst[e] = operand + half * PT_HALF + (row0 + row) * 128 + (((2 * c) ^ row) << 4);
    }
#pragma unroll
    for (int i0 = 0; i0 < 4; i0 += 2) {                                // groups of eight rows, two at a time
        uint4 w[2][STEPS];                                             // (reads in flight)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < STEPS; ++e) { w[i][e] = lds128(src[e] + (i0 + i) * 8 * HD); }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int e = 0; e < STEPS; ++e) {
                uint32_t h[8];
                halves_of(w[i][e].x, h[0], h[1]); halves_of(w[i][e].y, h[2], h[3]); halves_of(w[i][e].z, h[4], h[5]); halves_of(w[i][e].w, h[6], h[7]);
                sts128(dst[e] + (i0 + i) * 1024, make_uint4(h[0], h[1], h[2], h[3]));
                sts128((dst[e] ^ 16) + (i0 + i) * 1024, make_uint4(h[4], h[5], h[6], h[7]));
            }
        }
    }
}
__device__ __forceinline__ bool infinite_or_nan(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }

template <int HD, bool LATE, int KIND>
__global__ void __launch_bounds__(TcShape<HD, KIND>::THREADS, 1) paged_tc_kernel(const __grid_constant__ PagedAttention p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                  const int box, int *error_flag, const uint64_t wait_limit) {
    using Shape = TcShape<HD, KIND>;
    constexpr bool BYTES = Shape::BYTES;
    constexpr int SLOTS = Shape::SLOTS;
    extern __shared__ uint8_t raw[];
    __shared__ TcShared<KIND> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u, q_addr = base, ring = base + 2 * Shape::Q_BUFFERS * Shape::OPERAND;
    const uint32_t full = smem_u32(sh.full), empty = smem_u32(sh.empty), clean = smem_u32(sh.clean), known = smem_u32(sh.known), read = smem_u32(sh.read), joined = smem_u32(sh.joined);
    const uint32_t q_ready = smem_u32(sh.q_ready), q_free = smem_u32(sh.q_free), s_ready = smem_u32(sh.s_ready), s_free = smem_u32(sh.s_free), p_ready = smem_u32(sh.p_ready),
                   o_ready = smem_u32(sh.o_ready), p_free = smem_u32(sh.p_free);
    const uint32_t byte_full = smem_u32(sh.byte_full), byte_empty = smem_u32(sh.byte_empty), byte_ring = ring + SLOTS * Shape::OPERAND;
    if (tid == 0) {
        for (int i = 0; i < 8; ++i) { mbar_init(full + 8 * i, BYTES ? 4 : 1); mbar_init(empty + 8 * i, BYTES ? 1 : 3); mbar_init(clean + 8 * i, 2); sh.poison[i] = 0; }
        if (BYTES) { for (int i = 0; i < 8; ++i) { mbar_init(byte_full + 8 * i, 1); mbar_init(byte_empty + 8 * i, 4); } }
        for (int i = 0; i < 4; ++i) { mbar_init(q_ready + 8 * i, 1); mbar_init(q_free + 8 * i, 1); mbar_init(p_ready + 8 * i, 4); }
        for (int t = 0; t < 2; ++t) { mbar_init(s_ready + 8 * t, 1); mbar_init(s_free + 8 * t, 4); mbar_init(o_ready + 8 * t, 1); mbar_init(p_free + 8 * t, 1); mbar_init(joined + 8 * t, 4); }
        mbar_init(smem_u32(&sh.over), 1);
        sh.gave_up = 0;
        for (int i = 0; i < PT_ENTRIES; ++i) { mbar_init(known + 8 * i, 1); mbar_init(read + 8 * i, Shape::READERS); }
        mbar_init_fence();
    }
    pdl_launch_dependents();
    pdl_wait();
    Walker walk;
    // (at least four units a CTA, items' beginnings among them: 512 tokens at 512 positions 20.8 us, 23.8 from two on; 4 x 20 rows at 700 positions 24.5 and 22.8)
    walk.at = paged_plan<Shape::THREADS, PT_KEYS, PT_KEYS>(p, false, 4, sh.plan);
    if (walk.at.unit >= walk.at.end) { return; }
    if (warp == 8) { asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory"); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    uint64_t limit = wait_limit;
    uint32_t stretch = 0;
    auto gave_up = [&]() {                                // whether a wait of this warp has run out; all of its lanes' limits are 0 then
        if (__all_sync(0xffffffffu, limit != 0)) { return false; }
        limit = 0;
        return true;
    };
    // the next entry; false behind the last one, or when a wait gave up (the roles then end one after the other: nobody waits without a limit)
    auto next_entry = [&]() {
        wait_for(known + 8 * (stretch & (PT_ENTRIES - 1)), (stretch / PT_ENTRIES) & 1, limit);
        return !gave_up() && sh.entry[stretch & (PT_ENTRIES - 1)].todo != 0;
    };
    auto entry_read = [&](bool by_me) {
        if (by_me) { mbar_arrive(read + 8 * (stretch & (PT_ENTRIES - 1))); }
        ++stretch;
    };

    // K and V tiles take slots in turn: K of step 0, V of step 0, K of step 1, ...
    uint32_t slot = 0, phase = 0, issued = 0;             // (issued: tiles of K and V by the copying warp, of Q by those that check V)
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Shape::REGS_SOFTMAX));
        // ---------------------------------------------------------------------------------- probabilities, output
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                                   // (32 lanes a warp, in the address's upper half)
        const uint32_t s_tmem = tmem + lanes + t * PT_KEYS, p_tmem = tmem + lanes + Shape::P_COLUMN + t * Shape::P_STEP, o_tmem = tmem + lanes + Shape::O_COLUMN + t * HD;
        const float scale = p.scale_log2;
        const int half_tokens = PT_ROWS / p.group, row_token = (int)((unsigned)row / (unsigned)p.group), g = row - row_token * p.group;   // a tile has whole tokens
        uint32_t s_phase = 0, o_phase = 0, joined_phase = 0, p_phase = 1, tiles = 0;
        auto all_of_tile = [&]() {                            // the tile's four warps
            __syncwarp();
            if (lane == 0) { mbar_arrive(joined + 8 * t); }
            wait_for(joined + 8 * t, joined_phase, limit);
            joined_phase ^= 1;
        };
        while (next_entry()) {
            const Entry &en = sh.entry[stretch & (PT_ENTRIES - 1)];
            float m = -CUDART_INF_F, l = 0.f;
            const Tile own = en.half[t];
            const int token = (2 * en.tile + t) * half_tokens + row_token, pos = en.first + token;   // (of rows that are there)
            const bool mine = row < own.rows;                 // others hold what was there before, or another sequence's Q: they decide nothing
            for (int step = own.from; step < own.to; ++step) {
                wait_for(s_ready + 8 * t, s_phase, limit);
                s_phase ^= 1;
                tc_fence_after();
                uint32_t s[128];
                tmem_ld32(s_tmem, s);
                const uint32_t there = *reinterpret_cast<volatile uint32_t *>(&sh.there[(tiles + step - en.begin) & 7]);
                const bool plain = there == 0xffffu && en.whole(p, own, step);
                tmem_ld_wait();
#pragma unroll
                for (int i = 1; i < 4; ++i) { tmem_ld32(s_tmem + 32 * i, s + 32 * i); }
                // bytes: scores by K's scales, so that they are in powers of two already
                const float4 *k_scale = nullptr, *v_scale = nullptr, *v_log = nullptr;
                float v_top = 0.f;
                if constexpr (BYTES) {
                    const int at = (tiles + step - en.begin) & 3;
                    k_scale = reinterpret_cast<const float4 *>(sh.scale.k[at]); v_scale = reinterpret_cast<const float4 *>(sh.scale.v[at]); v_log = reinterpret_cast<const float4 *>(sh.scale.v_log[at]);
                    const float4 e = *reinterpret_cast<const float4 *>(sh.scale.v_top[at]);
                    v_top = fmaxf(fmaxf(e.x, e.y), fmaxf(e.z, e.w));
                }
                auto by_scales = [&](int from, int to) {
                    if constexpr (BYTES) {
#pragma unroll
                        for (int c = 0; c < 128; c += 4) {
                            if (c < from || c >= to) { continue; }
                            const float4 k = k_scale[c / 4];
                            float a, b;
                            f2_unpack(f2_mul(f2_pack_bits(s[c], s[c + 1]), f2_pack(k.x, k.y)), a, b);
                            s[c] = __float_as_uint(a); s[c + 1] = __float_as_uint(b);
                            f2_unpack(f2_mul(f2_pack_bits(s[c + 2], s[c + 3]), f2_pack(k.z, k.w)), a, b);
                            s[c + 2] = __float_as_uint(a); s[c + 3] = __float_as_uint(b);
                        }
                    }
                };
                if (plain) { by_scales(0, 32); }
                if (!plain) {
                    const int j0 = en.lo + step * PT_KEYS;
                    const int c1 = (p.causal ? min(en.hi, pos + 1) : en.hi) - j0, c0 = p.causal && p.window > 0 ? pos - p.window + 1 - j0 : 0;
                    tmem_ld_wait();
                    by_scales(0, 128);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int a = min(max(c0 - 32 * i, 0), 32), b = min(max(c1 - 32 * i, 0), 32);
                        uint32_t seen = ((there >> 4 * i & 15) * 0x00204081u & 0x01010101u) * 0xffu;      // (four groups of eight)
                        seen &= (b == 32 ? 0xffffffffu : (1u << b) - 1) & (a == 32 ? 0u : 0xffffffffu << a);
                        if (__all_sync(0xffffffffu, seen == 0xffffffffu)) { continue; }
#pragma unroll
                        for (int c = 0; c < 32; ++c) { if (!(seen >> c & 1)) { s[32 * i + c] = 0xff800000u; } }
                    }
                }
                const uint64_t scale2 = f2_pack(scale, scale);
                uint64_t neg2 = 0, sum[2] = {0, 0};
                auto powers = [&](int i) {                    // probabilities of these columns against m, into tensor memory
                    uint32_t h[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        float a, b;
                        const uint64_t x = f2_pack_bits(s[32 * i + 2 * c], s[32 * i + 2 * c + 1]);
                        f2_unpack(BYTES ? f2_add(x, neg2) : f2_fma(x, scale2, neg2), a, b);
                        a = exp2_fast(a); b = exp2_fast(b);
                        const uint64_t power = f2_pack(a, b);
                        sum[c & 1] = f2_add(sum[c & 1], power);
                        if constexpr (BYTES) {                // (V's scales beside the probabilities)
                            const float2 v = reinterpret_cast<const float2 *>(v_scale)[16 * i + c];
                            f2_unpack(f2_mul(power, f2_pack(v.x, v.y)), a, b);
                        }
                        h[c] = pack_f16(a, b);
                    }
                    tmem_st16(p_tmem + 16 * i, h);
                };
                auto hand_over = [&](int part) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(p_ready + 16 * t + 8 * part); }
                };
                if (Shape::P_APART) { wait_for(p_free + 8 * t, p_phase, limit); p_phase ^= 1; tc_fence_after(); }   // (P's products of the step before; else S is made behind them)
                // Powers against the maximum of the steps before, which nearly always does; whether it did shows beside them. (Not the stretch's first time round.)
                bool fresh = step == own.from, scaled = false, moved = false;   // (moved: once a step, for the bound of bytes stays where it is)
                for (;;) {
                    const float neg = m == -CUDART_INF_F ? 0.f : -m;
                    neg2 = f2_pack(neg, neg);
                    sum[0] = sum[1] = 0;
                    if (!fresh) { powers(0); }
                    tmem_ld_wait();
                    if (BYTES && plain && !scaled) { by_scales(32, 128); scaled = true; }
                    if (!fresh) { powers(1); }
                    float tops[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { tops[e] = fmaxf(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])); }
#pragma unroll
                    for (int c = 8; c < 128; c += 8) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) { tops[e] = max3(tops[e], __uint_as_float(s[c + 2 * e]), __uint_as_float(s[c + 2 * e + 1])); }
                    }
                    const float most = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
                    float top = BYTES ? most + v_top : most * scale;
                    const bool above = !(BYTES && moved) && __any_sync(0xffffffffu, mine && top > m + Shape::SLACK);
                    if constexpr (BYTES) {
                        // That is a bound: the largest score and the largest scale need not be one position's, nor need the row see both. Where it is far above some row's maximum, rows go on to their own
                        // largest weights: what a row does not see, or has no weight, takes nothing from its other weights. (Only rows that are far above going on: 434 us in place of 392 for 1500 tokens
                        // at 9111, for there are more such turns.)
                        if (above) {
                            float own_top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                            for (int c = 0; c < 128; c += 4) {
                                const float4 v = v_log[c / 4];
                                float a, b;
                                f2_unpack(f2_add(f2_pack_bits(s[c], s[c + 1]), f2_pack(v.x, v.y)), a, b);
                                own_top[0] = max3(own_top[0], a, b);
                                f2_unpack(f2_add(f2_pack_bits(s[c + 2], s[c + 3]), f2_pack(v.z, v.w)), a, b);
                                own_top[1] = max3(own_top[1], a, b);
                            }
                            top = fmaxf(own_top[0], own_top[1]);
                        }
                    }
                    if (above) {
                        const float to = fmaxf(m, top), f = to == m ? 1.f : exp2_fast(m - to);
                        m = to; l *= f;
                        if (step != own.from) {
#pragma unroll 1
                            for (int i = 0; i < HD / 16; ++i) {
                                uint32_t o[16];
                                tmem_ld16(o_tmem + 16 * i, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int c = 0; c < 16; ++c) { o[c] = __float_as_uint(__uint_as_float(o[c]) * f); }
                                tmem_st16(o_tmem + 16 * i, o);
                            }
                        }
                    } else if (!fresh) { break; }
                    fresh = false; moved = true;
                }
                if (Shape::P_APART) {                         // (S is in registers)
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(s_free + 8 * t); }
                }
                powers(2);
                hand_over(0);                                 // (their products run beside the last powers)
                powers(3);
                hand_over(1);
                float a, b;
                f2_unpack(f2_add(sum[0], sum[1]), a, b);
                l += a + b;
            }
            tiles += en.end - en.begin;
            // this stretch's findings
            const bool any = own.to > own.from;
            const int  parts = en.parts, c0 = en.c0;
            if (any) { wait_for(o_ready + 8 * t, o_phase, limit); o_phase ^= 1; tc_fence_after(); }
            float4 *part = reinterpret_cast<float4 *>(p.partial) + (paged_slot(blockIdx.x, c0) * 2 + t) * (PT_ROWS * (HD + 2) / 4);     // [HD / 4][128] x 4, [128], [128]
            const int64_t cell = KIND == PK_PLAIN ? 0 : (int64_t)(en.row0 + token) * (p.n_head_kv * p.group) + en.head * p.group + g;   // (of rows that are there) in what the two passes exchange
            const bool whole_item = parts == 1, with = KIND != PK_PLAIN && p.with_stats != nullptr && en.lo > 0;
            float factor = 1.f, other = 0.f, all = l;         // the row is (o factor + what the first pass found x other) / all
            if (KIND != PK_PLAIN && whole_item && mine) {
                if (p.stats != nullptr) { p.stats[cell] = make_float2(m, l); all = 1.f; }
                else if (with) {
                    const float2 w = p.with_stats[cell];
                    const float top = fmaxf(m, w.x), ref = top == -CUDART_INF_F ? 0.f : top;
                    factor = exp2f(m - ref); other = exp2f(w.x - ref); all = factor * l + other * w.y;
                }
            }
            const float inv = !whole_item ? 1.f : all == 0.f ? 0.f : 1.f / all;
            const bool poisoned = any && *reinterpret_cast<volatile int *>(&sh.poison[stretch & 7]) == (int)stretch + 1;
            const int64_t to_row = (int64_t)(en.row0 + token) * p.out_stride + (en.head * p.group + g) * HD;
#pragma unroll 1
            for (int i = 0; i < HD / 32; ++i) {
                uint32_t o[32];
                __syncwarp();
                if (any) { tmem_ld32(o_tmem + 32 * i, o); tmem_ld_wait(); }
                else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) { o[c] = 0; }
                }
                if (poisoned && mine) {
                    // values that are not finite were taken out of the V tiles that not all rows see whole: back to the rows that see them
                    const Tile other = en.half[1 - t];
                    for (int step = own.from; step < own.to; ++step) {
                        if (en.whole(p, own, step) && en.whole(p, other, step)) { continue; }
                        const int j0 = en.lo + step * PT_KEYS, ja = max(j0, p.causal && p.window > 0 ? pos - p.window + 1 : 0), jb = min(j0 + PT_KEYS, p.causal ? min(en.hi, pos + 1) : en.hi);
                        for (int j = ja; j < jb; ++j) {
                            const int page = p.view.page_table[(int64_t)en.seq * p.view.table_stride + j / p.view.page_size];
                            if (page < 0 || page >= p.view.n_pages) { continue; }
                            const int64_t at = page * p.view.page_stride + (j % p.view.page_size) * p.view.token_stride + en.head * p.view.head_stride + 32 * i;
                            if constexpr (BYTES) {
                                const uint32_t pair = p.scales.pairs[page * p.scales.page_stride + (j % p.view.page_size) * p.scales.token_stride + en.head * p.scales.head_stride];
                                if (!infinite_or_nan(pair >> 16)) { continue; }
                                const float scale = half2_bits(pair).y;
                                const int8_t *v = reinterpret_cast<const int8_t *>(p.v) + at;
#pragma unroll
                                for (int c = 0; c < 32; ++c) { o[c] = __float_as_uint(__uint_as_float(o[c]) + (float)v[c] * scale); }
                            } else {
                                const __half *v = p.v + at;
#pragma unroll
                                for (int c = 0; c < 32; ++c) {
                                    const float y = __half2float(v[c]);
                                    if (!isfinite(y)) { o[c] = __float_as_uint(__uint_as_float(o[c]) + y); }
                                }
                            }
                        }
                    }
                }
                if (KIND != PK_PLAIN && whole_item && mine && with) {
                    const float4 *u = reinterpret_cast<const float4 *>(p.with_out + cell * HD + 32 * i);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float4 x = u[c];
                        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) { o[4 * c + e] = __float_as_uint(__uint_as_float(o[4 * c + e]) * factor + y[e] * other); }
                    }
                }
                if (parts > 1 && mine) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        part[(8 * i + c) * PT_ROWS + row] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]), __uint_as_float(o[4 * c + 2]), __uint_as_float(o[4 * c + 3]));
                    }
                } else if (mine) {
                    if (p.out_f32) {
                        float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to_row + 32 * i);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            dst[c] = make_float4(__uint_as_float(o[4 * c]) * inv, __uint_as_float(o[4 * c + 1]) * inv, __uint_as_float(o[4 * c + 2]) * inv, __uint_as_float(o[4 * c + 3]) * inv);
                        }
                    } else {
                        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<__half *>(p.out) + to_row + 32 * i);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t h[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) { h[e] = pack_f16(__uint_as_float(o[8 * c + 2 * e]) * inv, __uint_as_float(o[8 * c + 2 * e + 1]) * inv); }
                            dst[c] = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                }
            }
            tc_fence_before();
            if (parts > 1 && own.rows > 0) {
                float *stats = reinterpret_cast<float *>(part + PT_ROWS * HD / 4);
                stats[row] = m; stats[PT_ROWS + row] = l;
            }
            if (KIND != PK_PLAIN && p.cuts != nullptr) {      // (joined by the next kernel, by all SMs: an item's rows are few and its CTAs many)
                if (row == 0 && own.rows > 0 && (whole_item || c0 == (int)blockIdx.x)) { p.cuts[(int64_t)en.head * p.view.n_rows + en.row0 + (2 * en.tile + t) * half_tokens] = make_int2(c0, parts); }
            } else if (parts > 1 && own.rows > 0) {
                __threadfence();
                all_of_tile();
                if (row == 0) {
                    __threadfence();
                    unsigned *arrived = p.arrived + 2 * c0 + t;
                    const bool last = atomicAdd(arrived, 1u) == (unsigned)parts - 1;
                    if (last) { *arrived = 0; __threadfence(); }
                    *reinterpret_cast<volatile int *>(&sh.last[t]) = last;
                }
                all_of_tile();
                if (*reinterpret_cast<volatile int *>(&sh.last[t])) {
                    // Few rows have several threads each, so that all of them load: row `row & (rows - 1)`, every share-th four elements. Either way 16 loads of 16
                    // bytes a thread are in flight: of one CTA's piece, or where rows are few, and their CTAs often many, of four (five rows at 100 000 positions, 18 CTAs
                    // an item: 96 us against 113 in the first way; a tile of 128 rows has few CTAs an item: a chunk of 512 rows 55 us in the first way, 58 in the second)
                    int rows = PT_ROWS;
                    while (rows > 4 && rows / 2 >= own.rows) { rows /= 2; }
                    const int r = row & (rows - 1), share = PT_ROWS / rows, token_in = (int)((unsigned)r / (unsigned)p.group);
                    const float4 *const all = reinterpret_cast<const float4 *>(p.partial) + t * (PT_ROWS * (HD + 2) / 4);
                    auto piece = [&](int i) { return all + paged_slot(c0 + i, c0) * (2 * PT_ROWS * (HD + 2) / 4); };
                    const int64_t out_row = (int64_t)(en.row0 + (2 * en.tile + t) * half_tokens + token_in) * p.out_stride + (en.head * p.group + r - token_in * p.group) * HD;
                    auto join = [&](auto fours, auto ahead) {
                        constexpr int FOURS = decltype(fours)::value, AHEAD = decltype(ahead)::value;
                        float top = -CUDART_INF_F;
#pragma unroll 8
                        for (int i = 0; i < parts; ++i) { top = fmaxf(top, __ldcg(reinterpret_cast<const float *>(piece(i) + PT_ROWS * HD / 4) + r)); }
                        const float ref = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll 1
                        for (int q4 = row / rows; q4 < HD / 4; q4 += FOURS * share) {
                            float4 v[FOURS];
#pragma unroll
                            for (int c = 0; c < FOURS; ++c) { v[c] = make_float4(0.f, 0.f, 0.f, 0.f); }
                            float sum = 0.f;
#pragma unroll 1
                            for (int i0 = 0; i0 < parts; i0 += AHEAD) {
                                float4 u[AHEAD][FOURS];
                                float  pm[AHEAD], pl[AHEAD];
#pragma unroll
                                for (int j = 0; j < AHEAD; ++j) {
                                    const bool is = i0 + j < parts;
                                    const float4 *from = piece(is ? i0 + j : 0);
                                    const float *st = reinterpret_cast<const float *>(from + PT_ROWS * HD / 4);
                                    pm[j] = is ? __ldcg(st + r) : -CUDART_INF_F;
                                    pl[j] = is ? __ldcg(st + PT_ROWS + r) : 0.f;
#pragma unroll
                                    for (int c = 0; c < FOURS; ++c) { u[j][c] = is && q4 + c * share < HD / 4 ? __ldcg(from + (q4 + c * share) * PT_ROWS + r) : make_float4(0.f, 0.f, 0.f, 0.f); }
                                }
#pragma unroll
                                for (int j = 0; j < AHEAD; ++j) {
                                    const float f = exp2_fast(pm[j] - ref);
                                    sum += f * pl[j];
#pragma unroll
                                    for (int c = 0; c < FOURS; ++c) { v[c].x += f * u[j][c].x; v[c].y += f * u[j][c].y; v[c].z += f * u[j][c].z; v[c].w += f * u[j][c].w; }
                                }
                            }
                            if constexpr (KIND != PK_PLAIN) {
                                const int64_t its = (int64_t)(en.row0 + (2 * en.tile + t) * half_tokens + token_in) * (p.n_head_kv * p.group) + en.head * p.group + r - token_in * p.group;
                                if (p.stats != nullptr) {
                                    if (q4 == 0) { p.stats[its] = make_float2(top, sum); }
                                    sum = 1.f;
                                } else if (with) {
                                    const float2 w = p.with_stats[its];
                                    const float both = fmaxf(top, w.x), at = both == -CUDART_INF_F ? 0.f : both, f = exp2f(top - at), h = exp2f(w.x - at);
                                    sum = f * sum + h * w.y;
                                    const float4 *from = reinterpret_cast<const float4 *>(p.with_out + its * HD);
#pragma unroll
                                    for (int c = 0; c < FOURS; ++c) {
                                        if (q4 + c * share >= HD / 4) { break; }
                                        const float4 x = from[q4 + c * share];
                                        v[c] = make_float4(f * v[c].x + h * x.x, f * v[c].y + h * x.y, f * v[c].z + h * x.z, f * v[c].w + h * x.w);
                                    }
                                }
                            }
                            const float inv_all = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                            for (int c = 0; c < FOURS; ++c) { v[c] = make_float4(v[c].x * inv_all, v[c].y * inv_all, v[c].z * inv_all, v[c].w * inv_all); }
                            __half *const out16 = static_cast<__half *>(p.out) + out_row;
#pragma unroll
                            for (int c = 0; c < FOURS; ++c) {
                                const int at = q4 + c * share;
                                if (at >= HD / 4) { break; }
                                if (p.out_f32) { *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + out_row + 4 * at) = v[c]; }
                                else if (FOURS < 16) { *reinterpret_cast<uint2 *>(out16 + 4 * at) = make_uint2(pack_f16(v[c].x, v[c].y), pack_f16(v[c].z, v[c].w)); }
                                else if (c % 2 == 0) {
                                    const float4 b = v[(c + 1) % FOURS];
                                    *reinterpret_cast<uint4 *>(out16 + 4 * at) = make_uint4(pack_f16(v[c].x, v[c].y), pack_f16(v[c].z, v[c].w), pack_f16(b.x, b.y), pack_f16(b.z, b.w));
                                }
                            }
                        }
                    };
                    if (r < own.rows) {
                        if (share == 1) { join(std::integral_constant<int, 16>(), std::integral_constant<int, 1>()); }
                        else { join(std::integral_constant<int, 4>(), std::integral_constant<int, 4>()); }
                    }
                }
            }
            __syncwarp();
            entry_read(lane == 0);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Shape::REGS_OTHERS));
        auto advance = [&]() { if (++slot == SLOTS) { slot = 0; phase ^= 1; } };
        if (warp == 9) {
            // ------------------------------------------------------------------------------ the stretches, and their copies
            constexpr int halves = BYTES ? 1 : HD / 64;                                     // a tile's boxes are 64 elements wide, of bytes all of a head
            constexpr int COPY_SLOTS = BYTES ? Shape::BYTE_SLOTS : SLOTS;
            const uint32_t landed = BYTES ? byte_full : full, free_again = BYTES ? byte_empty : empty;
            const int group = lane % 16 * 8, half = lane >> 4;                              // this lane's eight positions of a tile, and half
            const bool issues = (group & (box - 1)) == 0 && half < halves;
            uint32_t &copies = issued;
            walk.seq = walk.at.seq; walk.head = walk.at.head; walk.tile = walk.at.tile; walk.off = walk.at.off;
            walk.q = paged_seq(p.view, walk.seq);
            auto put = [&](const Entry &e) {                                                // false: somebody gave up
                const uint32_t i = stretch & (PT_ENTRIES - 1);
                wait_for(read + 8 * i, ((stretch / PT_ENTRIES) & 1) ^ 1, limit);
                if (gave_up()) { return false; }
                if (lane == 0) { sh.entry[i] = e; mbar_arrive(known + 8 * i); }
                ++stretch;
                return true;
            };
            for (;;) {
                const Entry e = walk.entry(p);
                if (!put(e)) { break; }
                const int32_t *table = p.view.page_table + (int64_t)e.seq * p.view.table_stride;
                auto page_of = [&](int step) {                                              // (one step ahead: the table's latency is hidden)
                    const int j = e.lo + step * PT_KEYS + group;
                    return step < e.end && j < e.hi ? table[j / p.view.page_size] : -1;
                };
                int named = page_of(e.begin);
                for (int step = e.begin; step < e.end; ++step) {
                    const bool ok = named >= 0 && named < p.view.n_pages;
                    const int page = ok ? named : p.view.n_pages, token = ok ? (e.lo + step * PT_KEYS + group) % p.view.page_size : 0;
                    const uint32_t there = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                    named = page_of(step + 1);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        wait_for(free_again + 8 * slot, phase ^ 1, limit);
                        if (LATE && p.late == PA_LATE_KV && copies == 2) { stand_still(3 * wait_limit); }   // (issued all the same, with nobody waiting any more)
                        else if (gave_up()) { break; }
                        const uint32_t bar = landed + 8 * slot, dst = BYTES ? byte_ring + slot * Shape::BYTE_TILE : ring + slot * Shape::OPERAND;
                        if (lane == 0) {
                            if (kv == 0) { *reinterpret_cast<volatile uint32_t *>(&sh.there[copies / 2 & 7]) = there; }
                            mbar_expect_tx(bar, BYTES ? Shape::BYTE_TILE : Shape::OPERAND);
                        }
                        __syncwarp();
                        if (issues) { tma_load(BYTES ? dst + group * HD : dst + half * PT_HALF + group * 128, kv == 0 ? &k_map : &v_map, bar, half * 64, token, e.head, page); }
                        __syncwarp();
                        if (BYTES) { if (++slot == COPY_SLOTS) { slot = 0; phase ^= 1; } }
                        else { advance(); }
                        ++copies;
                    }
                    if (limit == 0) { break; }
                }
                if (limit == 0 || !walk.next(p, e.todo)) { break; }
            }
            if (limit != 0) { Entry over = {}; put(over); }
        } else if (warp == 10 || warp == 11) {
            // ------------------------------------------------------------------------------ Q of a tile each; V tiles that not all rows see whole, half of the rows each
            // (of 8-bit caches Q alone)
            uint32_t tiles = 0, &q_count = issued;
            const int t = warp - 10, v_row0 = t * (PT_KEYS / 2);
            while (next_entry()) {
                const Entry &en = sh.entry[stretch & (PT_ENTRIES - 1)];
                const Tile a = en.half[0], b = en.half[1];
                if (t == 0 ? a.to > a.from : b.to > b.from) {
                    const uint32_t buffer = q_count % Shape::Q_BUFFERS, bar = 16 * t + 8 * buffer;
                    wait_for(q_free + bar, (q_count / Shape::Q_BUFFERS & 1) ^ 1, limit);
                    if (LATE && p.late == PA_LATE_Q && q_count == 0) { stand_still(3 * wait_limit); }
                    else if (gave_up()) { break; }
                    ++q_count;
                    // whole tokens, token by token their heads: what lies behind the sequence's rows is other sequences' or nothing, and goes nowhere
                    if (elect_one()) {
                        const int tokens = PT_ROWS / p.group, row = en.row0 + (2 * en.tile + t) * tokens;
                        mbar_expect_tx(q_ready + bar, tokens * p.group * HD * 2);
#pragma unroll
                        for (int h = 0; h < HD / 64; ++h) { tma_load3(q_addr + (2 * buffer + t) * Shape::OPERAND + h * PT_HALF, &q_map, q_ready + bar, h * 64, en.head * p.group, row); }
                    }
                    __syncwarp();
                }
                if constexpr (!BYTES) {
                    for (int step = en.begin; step < en.end; ++step) {
                        if (LATE && p.late == PA_LATE_CHECKS && tiles < 12) { stand_still(4000); }
                        // K as well, though nothing is done to it: copies land in any order, and a slot's phase that nobody waited for could be taken for the one after the next.
                        // A slot is not filled again before both warps have seen its phase, or they would wait for one that is over
                        wait_for(full + 8 * slot, phase, limit);
                        if (lane == 0 && limit != 0) { mbar_arrive(empty + 8 * slot); }
                        advance();
                        wait_for(full + 8 * slot, phase, limit);
                        if (!(en.whole(p, a, step) && (b.rows == 0 || en.whole(p, b, step)))) {
                            const int j0 = en.lo + step * PT_KEYS;
                            const int first = p.causal && p.window > 0 ? max(0, a.pos_first - p.window + 1) - j0 : 0, end = en.hi - j0;   // rows that some query sees
                            const uint32_t v_addr = ring + slot * Shape::OPERAND;
                            uint32_t bad = 0;
                            auto piece = [&](int i) {                                            // (half, row, piece of the row)
                                const int at = i * 32 + lane;
                                return (at >> 9) * PT_HALF + v_row0 * 128 + (at & 511) * 16;
                            };
    #pragma unroll 8
                            for (int i = 0; i < PT_KEYS / 2 * HD / 8 / 32; ++i) {
                                const int r = v_row0 + (((i * 32 + lane) & 511) >> 3);
                                const uint4 v = lds128(v_addr + piece(i));
                                if (r >= end || r < first) { sts128(v_addr + piece(i), make_uint4(0, 0, 0, 0)); }
                                else { bad |= not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w); }
                            }
                            if (__any_sync(0xffffffffu, bad)) {
    #pragma unroll 1
                                for (int i = 0; i < PT_KEYS / 2 * HD / 8 / 32; ++i) {
                                    const uint4 v = lds128(v_addr + piece(i));
                                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    #pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        if ((w[e] & 0x7c00u) == 0x7c00u) { w[e] &= 0xffff0000u; }
                                        if ((w[e] & 0x7c000000u) == 0x7c000000u) { w[e] &= 0xffffu; }
                                    }
                                    sts128(v_addr + piece(i), make_uint4(w[0], w[1], w[2], w[3]));
                                }
                                if (lane == 0) { *reinterpret_cast<volatile int *>(&sh.poison[stretch & 7]) = (int)stretch + 1; }
                            }
                            fence_async_smem();
                        }
                        __syncwarp();
                        if (lane == 0 && limit != 0) { mbar_arrive(clean + 8 * (tiles & 7)); mbar_arrive(empty + 8 * slot); }
                        advance();
                        ++tiles;
                    }
                }
                __syncwarp();
                entry_read(lane == 0);
            }
        } else if (warp >= 12) {
            // ------------------------------------------------------------------------------ operands of bytes and scales: 32 rows of every K and V tile each
            if constexpr (BYTES) {
                uint32_t tiles = 0, byte_slot = 0, byte_phase = 0;
                const int row0 = (warp - 12) * 32;
                const unsigned page_size = p.view.page_size;
                while (next_entry()) {
                    const Entry &en = sh.entry[stretch & (PT_ENTRIES - 1)];
                    const Tile a = en.half[0], b = en.half[1];
                    // The scales of this lane's position of a step are read a step ahead, its page two. (Loads without branches around them, or each is waited for where it stands: what is not
                    // there reads something that is, and counts as 0.)
                    const int32_t *table = p.view.page_table + (int64_t)en.seq * p.view.table_stride;
                    const uint32_t *pairs = p.scales.pairs + en.head * p.scales.head_stride;
                    const int seen_from = p.causal && p.window > 0 ? max(0, a.pos_first - p.window + 1) : 0, hi = en.hi, lo = en.lo, end = en.end;
                    int page = 0, at = 0;
                    bool ok = false, next_ok = false;
                    uint32_t next_pair = 0;
                    auto find = [&](int step) {
                        const int j = lo + step * PT_KEYS + row0 + lane;
                        ok = step < end && j >= seen_from && j < hi;                                 // (what nobody sees is not there)
                        const unsigned in = ok ? j : 0, which = in / page_size;
                        page = table[which]; at = in - which * page_size;
                    };
                    auto fetch = [&]() {                                                             // of the step that was found last
                        next_ok = ok && page >= 0 && page < p.view.n_pages;
                        next_pair = pairs[(next_ok ? page : 0) * p.scales.page_stride + at * p.scales.token_stride];
                    };
                    if (en.begin < end) { find(en.begin); fetch(); find(en.begin + 1); }
                    for (int step = en.begin; step < end; ++step) {
                        if (LATE && p.late == PA_LATE_CHECKS && tiles < 12) { stand_still(4000); }
                        uint32_t pair = next_ok ? next_pair : 0u;
                        fetch(); find(step + 2);
                        if (!(en.whole(p, a, step) && (b.rows == 0 || en.whole(p, b, step)))) {
                            // 0 x inf: positions that some rows see and others do not. They are taken out, and given back to the rows that see them
                            const bool bad = infinite_or_nan(pair >> 16);
                            if (__any_sync(0xffffffffu, bad)) {
                                if (bad) { pair &= 0xffffu; }
                                if (lane == 0) { *reinterpret_cast<volatile int *>(&sh.poison[stretch & 7]) = (int)stretch + 1; }
                            }
                        }
                        const float2 scale = half2_bits(pair);
                        const unsigned top = __reduce_max_sync(0xffffffffu, infinite_or_nan(pair >> 16) ? 0u : __float_as_uint(fabsf(scale.y)));
#pragma unroll 1
                        for (int kv = 0; kv < 2; ++kv) {
                            wait_for(byte_full + 8 * byte_slot, byte_phase, limit);
                            wait_for(empty + 8 * slot, phase ^ 1, limit);
                            if (gave_up()) { break; }
                            if (kv == 0) {                // (a slot for K is free: what the step four before this one had is read)
                                sh.scale.k[tiles & 3][row0 + lane] = fmaf(scale.x, 0.f, scale.x * p.scale_log2);   // (an infinite one is NaN: its elements' infinities do not add up to one)
                                sh.scale.v[tiles & 3][row0 + lane] = scale.y;
                                sh.scale.v_log[tiles & 3][row0 + lane] = infinite_or_nan(pair >> 16) ? PT_LEAST : fmaxf(log2_fast(fabsf(scale.y)), PT_LEAST);
                                if (lane == 0) { sh.scale.v_top[tiles & 3][warp - 12] = top == 0 ? PT_LEAST : (float)((int)(top >> 23) - 126); }
                            }
                            make_operand<HD>(byte_ring + byte_slot * Shape::BYTE_TILE, ring + slot * Shape::OPERAND, row0);
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) { mbar_arrive(byte_empty + 8 * byte_slot); mbar_arrive(full + 8 * slot); }
                            if (++byte_slot == Shape::BYTE_SLOTS) { byte_slot = 0; byte_phase ^= 1; }
                            advance();
                        }
                        if (limit == 0) { break; }
                        ++tiles;
                    }
                    if (limit == 0) { break; }
                    __syncwarp();
                    entry_read(lane == 0);
                }
            }
        } else if (warp == 8) {
            // ------------------------------------------------------------------------------ MMAs
            constexpr uint32_t idesc_s = idesc_f16(PT_KEYS), idesc_o = idesc_f16(HD) | (1u << 16);   // (bit 16: B is MN-major)
            uint32_t q_count[2] = {0, 0}, s_count[2] = {0, 0}, p_phase[2] = {0, 0}, tiles = 0;
            auto frees = [&]() { return elect_one() && limit != 0; };   // (the lane that issues has seen every wait's end for itself)
            auto scores = [&](int t, uint32_t k_slot, bool last) {
                if (Shape::P_APART) { wait_for(s_free + 8 * t, (s_count[t] & 1) ^ 1, limit); tc_fence_after(); }   // (else P's products, in order, are what frees S)
                ++s_count[t];
                const uint32_t buffer = (q_count[t] - 1) % Shape::Q_BUFFERS;
                if (elect_one()) {
                    const uint64_t a = swizzled_desc(q_addr + (2 * buffer + t) * Shape::OPERAND, 16), b = swizzled_desc(ring + k_slot * Shape::OPERAND, 16);
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint64_t step = ((k >> 2) * PT_HALF + (k & 3) * 32) >> 4;
                        mma_f16_ss(tmem + t * PT_KEYS, a + step, b + step, idesc_s, k != 0);
                    }
                    mma_commit(s_ready + 8 * t);
                    if (last && limit != 0) { mma_commit(q_free + 16 * t + 8 * buffer); }
                }
                __syncwarp();
            };
            while (next_entry()) {
                const Entry &en = sh.entry[stretch & (PT_ENTRIES - 1)];
                const int begin = en.begin, end = en.end, from[2] = {en.half[0].from, en.half[1].from}, to[2] = {en.half[0].to, en.half[1].to};
                __syncwarp();
                entry_read(lane == 0);
                auto active = [&](int t, int step) { return step >= from[t] && step < to[t]; };
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (to[t] > from[t]) { wait_for(q_ready + 16 * t + 8 * (q_count[t] % Shape::Q_BUFFERS), q_count[t] / Shape::Q_BUFFERS & 1, limit); ++q_count[t]; }
                }
                tc_fence_after();
                for (int step = begin; step < end; ++step) {
                    if (step == begin) {
                        wait_for(full + 8 * slot, phase, limit);
                        tc_fence_after();
#pragma unroll
                        for (int t = 0; t < 2; ++t) { if (active(t, step)) { scores(t, slot, step + 1 == to[t]); } }
                        if (frees()) { mma_commit(empty + 8 * slot); }
                        __syncwarp();
                        advance();
                    }
                    const uint32_t v_slot = slot, v_phase = phase;
                    advance();
                    const bool ahead = step + 1 < end;
                    if (ahead) { wait_for(full + 8 * slot, phase, limit); }
                    if (Shape::P_APART && ahead) {
#pragma unroll
                        for (int t = 0; t < 2; ++t) { if (active(t, step + 1)) { scores(t, slot, step + 2 == to[t]); } }
                        if (frees()) { mma_commit(empty + 8 * slot); }
                        __syncwarp();
                    }
                    wait_for(full + 8 * v_slot, v_phase, limit);
                    if (!BYTES) { wait_for(clean + 8 * (tiles & 7), (tiles >> 3) & 1, limit); }   // (an operand is made of what is seen alone)
                    ++tiles;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (active(t, step)) {
#pragma unroll
                            for (int part = 0; part < 2; ++part) {
                                wait_for(p_ready + 16 * t + 8 * part, p_phase[t], limit);
                                tc_fence_after();
                                if (elect_one()) {
                                    const uint64_t b = swizzled_desc(ring + v_slot * Shape::OPERAND, PT_HALF);
#pragma unroll
                                    for (int k = 6 * part; k < 6 + 2 * part; ++k) {
                                        mma_f16_ts(tmem + Shape::O_COLUMN + t * HD, tmem + Shape::P_COLUMN + t * Shape::P_STEP + 8 * k, b + ((k * 2048) >> 4), idesc_o, step != from[t] || k != 0);
                                    }
                                    if (part == 1 && Shape::P_APART) { mma_commit(p_free + 8 * t); }
                                    if (part == 1 && step + 1 == to[t]) { mma_commit(o_ready + 8 * t); }
                                }
                                __syncwarp();
                            }
                            p_phase[t] ^= 1;
                        }
                        if (!Shape::P_APART && ahead && active(t, step + 1)) { scores(t, slot, step + 2 == to[t]); }
                    }
                    if (frees()) {
                        mma_commit(empty + 8 * v_slot);
                        if (!Shape::P_APART && ahead) { mma_commit(empty + 8 * slot); }
                    }
                    __syncwarp();
                    if (ahead) { advance(); }
                }
            }
        }
    }
    if (limit == 0 && lane == 0) { pf_report(error_flag, 7); *reinterpret_cast<volatile int *>(&sh.gave_up) = 1; }
    tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int *>(&sh.gave_up)) {
        uint64_t again = PT_LANDING_NS;
        if (warp == 8) {
            if (elect_one()) { mma_commit(smem_u32(&sh.over)); }
            __syncwarp();
            wait_for(smem_u32(&sh.over), 0, again);
        } else if (warp == 9) {                           // each slot's last copy (the ones before it were waited for by whoever freed the slot)
            constexpr uint32_t COPY_SLOTS = BYTES ? Shape::BYTE_SLOTS : SLOTS;
            for (uint32_t i = 0; i < COPY_SLOTS && i < issued; ++i) {
                if (slot == 0) { slot = COPY_SLOTS; phase ^= 1; }
                --slot;
                wait_for((BYTES ? byte_full : full) + 8 * slot, phase, again);
            }
        } else if (warp == 10 || warp == 11) {
            for (uint32_t i = 1; i <= Shape::Q_BUFFERS && i <= issued; ++i) {
                const uint32_t n = issued - i;
                wait_for(q_ready + 16 * (warp - 10) + 8 * (n % Shape::Q_BUFFERS), n / Shape::Q_BUFFERS & 1, again);
            }
        }
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) { cudaGetLastError(); f = nullptr; }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}
// (Bytes of a position are 128 or fewer: where positions lie apart, more than these would be another head's. Three of 100 000 by token, 8 heads: 121 us with 256, 115 with 128.)
bool tensor_map(CUtensorMap *map, const __half *data, int n, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box, bool bytes = false, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return encoder() != nullptr && encoder()(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, n, const_cast<__half *>(data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                             swizzle, bytes ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// pages of one pool: [page][head][position][element] whatever the order of the strides; boxes of `box` positions x 64 elements, or x all bytes of a head
bool page_map(CUtensorMap *map, const __half *pool, const PagedView &v, int heads, int head_dim, int box, bool bytes, CUtensorMapSwizzle swizzle) {
    const cuuint64_t size = bytes ? 1 : 2;
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)v.page_size, (cuuint64_t)heads, (cuuint64_t)v.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)v.token_stride * size, (cuuint64_t)v.head_stride * size, (cuuint64_t)v.page_stride * size};
    const cuuint32_t boxes[4] = {bytes ? (cuuint32_t)head_dim : 64, (cuuint32_t)box, 1, 1};
    return tensor_map(map, pool, 4, dims, strides, boxes, bytes, swizzle);
}
// Q: [row][head][element], boxes of whole tokens of a group of heads
bool query_map(CUtensorMap *map, const PagedAttention &p, int n_head, int head_dim) {
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)n_head, (cuuint64_t)p.view.n_rows}, strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)p.q_stride * 2};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(PT_ROWS / p.group)};
    return tensor_map(map, p.q, 3, dims, strides, boxes);
}
// the warpgroups' registers after their split are what the block is launched with: fewer, and the split would wait for ever
template <int HD, bool LATE, int KIND> cudaError_t registers_suffice() {
    static const cudaError_t answer = [] {
        cudaFuncAttributes a;
        const cudaError_t err = cudaFuncGetAttributes(&a, paged_tc_kernel<HD, LATE, KIND>);
        return err != cudaSuccess ? err : a.numRegs * TcShape<HD, KIND>::THREADS >= 256 * TcShape<HD, KIND>::REGS_SOFTMAX + (TcShape<HD, KIND>::THREADS - 256) * TcShape<HD, KIND>::REGS_OTHERS ? cudaSuccess : cudaErrorInvalidConfiguration;
    }();
    return answer;
}
template <int HD, bool LATE, int KIND>
cudaError_t launch_tc(const PagedAttention &p, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, int box, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    cudaError_t err = registers_suffice<HD, LATE, KIND>();
    if (err != cudaSuccess) { return err; }
    err = allow_dynamic_smem(reinterpret_cast<const void *>(paged_tc_kernel<HD, LATE, KIND>), TcShape<HD, KIND>::SMEM);
    if (err != cudaSuccess) { return err; }
    return launch_maybe_pdl(paged_tc_kernel<HD, LATE, KIND>, dim3(sms), TcShape<HD, KIND>::THREADS, TcShape<HD, KIND>::SMEM, cfg.stream, cfg.pdl, p, q, k, v, box, cfg.error_flag, wait_limit);
}

template <bool LATE, int KIND>
cudaError_t launch_tc(const PagedAttention &p, int head_dim, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, int box, int sms, const LaunchCfg &cfg, uint64_t wait_limit) {
    return head_dim == 128 ? launch_tc<128, LATE, KIND>(p, q, k, v, box, sms, cfg, wait_limit) : launch_tc<64, LATE, KIND>(p, q, k, v, box, sms, cfg, wait_limit);
}

}  // namespace

bool paged_byte_map(CUtensorMap *map, const void *pool, const PagedView &v, int heads, int head_dim, int box) {
    const int64_t most = std::max({v.token_stride, v.head_stride, v.page_stride}), least = std::min({v.token_stride, v.head_stride, v.page_stride});
    return least > 0 && most < (1ll << 38) && page_map(map, static_cast<const __half *>(pool), v, heads, head_dim, box, true, head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}
static int paged_tc_box(int page_size) {   // positions of a box: the largest power of two up to 128 that divides the page size
    int box = 1;
    while (box < PT_KEYS && page_size % (2 * box) == 0) { box *= 2; }
    return box;
}
bool launch_paged_attention_tc(const PagedAttention &given, int head_dim, int n_head, int sms, const LaunchCfg &cfg, uint64_t wait_limit, cudaError_t *err) {
    const int box = paged_tc_box(given.view.page_size);
    const PagedView &view = given.view;
    const int64_t most = std::max({view.token_stride, view.head_stride, view.page_stride, given.q_stride}), least = std::min({view.token_stride, view.head_stride, view.page_stride, given.q_stride});
    if ((head_dim != 64 && head_dim != 128) || box < 8 || given.group > PT_ROWS || least <= 0 || most >= (1ll << 38)) { return false; }
    PagedAttention p = given;
    p.tile_rows = 2 * (PT_ROWS / p.group) * p.group;
    p.start_units = PA_START;
    CUtensorMap q, k, v;
    const int kind = p.kind();
    const bool bytes = kind == PK_INT8;
    const CUtensorMapSwizzle swizzle = bytes && head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;   // (see make_operand)
    if (!query_map(&q, p, n_head, head_dim) || !page_map(&k, p.k, p.view, p.n_head_kv, head_dim, box, bytes, swizzle) || !page_map(&v, p.v, p.view, p.n_head_kv, head_dim, box, bytes, swizzle)) { return false; }
    const auto launch = kind == PK_SHARED ? launch_tc<false, PK_SHARED> : bytes ? (p.late != PA_ON_TIME ? launch_tc<true, PK_INT8> : launch_tc<false, PK_INT8>)
                                          : p.late != PA_ON_TIME ? launch_tc<true, PK_PLAIN> : launch_tc<false, PK_PLAIN>;
    *err = launch(p, head_dim, q, k, v, box, sms, cfg, wait_limit);
    return true;
}

}  // namespace spyb
