// Attention over a paged cache for more than a few query rows of a KV head (trees of a group's heads, prompts) on tcgen05; formulas and rows as in pi_attn_paged.cu.
//
// A piece of work is 128 query rows (the lanes) of one KV head and a range of its slots, in tiles of 128.  A CTA an SM takes one piece after the other (a counter in
// the workspace: pieces are of unequal lengths), and each of its roles goes on to the next as soon as its own part is done, so that the ends of a piece overlap.
// A tile's keys and values come as tensor copies of one page's rows each into a ring of 128-byte swizzled rows of 64 halves, which is K-major for the scores and MN-major for the
// values; queries lie beside them in the same layout.  Scores S = Q K^T are made into one of three buffers in tensor memory; the probabilities take their place; sums of values O = P V
// of ONE tile go to one or two more, which are drained and added with rounding in registers: the tensor cores cut FP32 sums at every step, so that no sum stays with them for longer
// than a tile.  So every tile has its own maximum (no exchange between tiles; the score buffers are groups of warps' own): the drain joins tiles.
//
// A tile is special where not every row of the piece sees all of its slots: then its group goes over its values before they are used.  Rows of slots that are not there
// become zeros, rows with a value that is not finite too, and whoever sees such a slot has a row of no numbers; scores of slots that a row does not see are replaced by what its
// mask says.
//
// What bounds it, by shape, warm and in a graph (FP32 128, a chunk of 1024 tokens over 4096 slots, 64 heads over 8: 198 us, of which the products, two for one, would take 146; FP16 162): at head_dim 128 FP32 a
// tile takes 2670 clocks, the products 2048, and the sums of a tile, one buffer, wait for the ones before to be drained; FP16 2580, the copies of keys and values 2150 (30 bytes a clock and SM, the rate of the
// memory) and the products 1536; at head_dim 64 FP16 1900, the exponents 1024, the products 768 and the chain from a score to its probability.  One sequence of 32768 slots, 25 FP32 tokens, 64 heads over 8: 63 us; 8 of
// 1000 to 2000, 48 FP16 tokens, 32 heads over 32: 50; 16 of 750 to 1500, 32 FP16 tokens, 128 heads over 8 of 64: 51.  Head_dim 256: 2 x 300 tokens of 3000 slots, 32 heads over 8: FP32 132, FP16 123 (copies: 96 KB a tile and half).
//
// Precision.  Probabilities, and queries of FP32 rows, are the sum of two halves each, 22 bits, i.e. two products in the place of one; queries of FP16 rows are halves as they are.  (One half for
// FP16 rows' probabilities left 1.3 times the error of the result's own rounding, and 9 to 16 rows, which go to the other kernel, had other bits.)  Probabilities are held times 2^14, so their steps end 2^-38 below a tile's largest one.
//
// Warps: 0 issues the products of scores and 2 those of values; 1 asks for keys and 3 for values; 4 takes work and asks for its queries (5..7 make a warpgroup of it, for the registers); 8..19 have the
// probabilities, three groups a tile each in turn, a row a thread; 20..27 drain the sums, a row and half of the columns a thread.
#include "pi_attn_paged.cuh"
#include "pi_tc.cuh"
#include "pi_tc_math.cuh"

#include <algorithm>
#include <cstdlib>

namespace pi {

static constexpr int PT_THREADS = 896, PT_GROUPS = 3;                  // groups of warps with tiles of probabilities
static constexpr int PT_REGS_M = 40, PT_REGS_Q = 40, PT_REGS_S = 72, PT_REGS_D = 104;  // 40 + 40 + 3 x 72 + 2 x 104 of the 7 x 72 of the launch
static constexpr uint32_t PT_SUB = PT_KEYS * 128;                     // bytes of 64 columns of a tile
static constexpr int PT_BOX = 64;                                     // rows of a tensor copy, or a page's if it has fewer
static constexpr int PT_WORK = 4;                                     // pieces of work that a CTA has in hand
static constexpr int PT_INFO = 16;                                    // tiles whose description is kept: more than keys may be ahead of probabilities

struct PtP { AttnPagedP a; int box, units, wide; unsigned int tries; unsigned int * next; CUtensorMap m_q, m_k, m_v; };

// what is in shared memory besides the ring: queries' buffers (upper and, of FP32 rows, lower halves), tiles in the ring
// Of more than 128 columns a piece of work has all scores and half of the values' columns (the sums of all would leave tensor memory for one buffer of scores, FP32 rows' queries no room for a tile's
// keys: the scores are made twice); keys then come 64 columns at a time.
template <int HD, bool TWO> struct PtShape {
    static constexpr bool WIDE = HD > 128;
    static constexpr int HV = WIDE ? HD / 2 : HD, QSUBS = (HD + 63) / 64, SUBS = (HV + 63) / 64;     // columns of the values; pieces of 64 columns of queries and keys, of values
    static constexpr uint32_t TILE = SUBS * PT_SUB, HALF = QSUBS * PT_SUB, QUERIES = HALF * (TWO ? 2 : 1), FILL = WIDE ? PT_SUB : TILE;      // FILL: what a place for keys holds
    static constexpr int QB = HD <= 64 ? 2 : 1, NS = WIDE ? 13 - (int)(QUERIES / PT_SUB) : (int)((196608u - QB * QUERIES) / TILE);
    static constexpr int NW = !WIDE ? NS - NS / 2 : NS >= 7 ? 2 : 1, NK = WIDE ? NS - SUBS * NW : NS - NW;      // places of values, of keys
    static constexpr size_t SMEM = QB * QUERIES + NK * FILL + NW * TILE + 1024;
};

// A piece of work: 128 rows of one KV head and a range of slots
struct PtWork { int tiles, k0, k1, first, n_rows, hk, there, clear, dst, v0; SeqB s; };      // tiles -1: there is no more; dst: number of the part that it makes, -1: results; v0: first column of the values

template <bool WIDE, int HV> __device__ __forceinline__ PtWork pt_piece(const PtP & pp, int unit) {      // (tiles -1: there are no rows, or another part answers for them)
    const AttnPagedP & p = pp.a;
    const AqItem it = ap_item(p, WIDE ? unit >> 1 : unit);
    PtWork w;
    w.tiles = -1;
    w.v0 = WIDE && unit & 1 ? HV : 0;
    w.s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, it.entry);
    const TileP t = ap_tile(p, w.s, p.row_tiles - 1 - it.rt, PT_ROWS);          // (the longest rows first)
    w.k0 = it.split * p.split; w.k1 = it.split == it.n_splits - 1 ? t.seen : min(t.seen, w.k0 + p.split);
    w.first = t.first; w.n_rows = t.n_rows; w.hk = it.hk; w.there = t.there;
    w.dst = it.n_splits > 1 ? (it.item - p.whole) * p.n_splits + it.split : -1;
    w.clear = p.mask ? w.s.pos : w.s.pos + p.by_group.of(t.first) + 1;          // every row sees the slots before it
    if (t.n_rows > 0 && (w.k0 < w.k1 || it.split == 0)) w.tiles = w.k0 < w.k1 ? (w.k1 - w.k0 + PT_KEYS - 1) / PT_KEYS : 0;      // (split 0 answers for rows that see nothing)
    return w;
}

// Barriers by their addresses in shared memory.  Code is kept short: seven roles run at once, and warps that waited for instructions were a third of the time.
// A wait of up to some 20 us at a time (warps that ask again and again take issue slots), `tries` times (PT_TRIES), or until another one of the CTA ran out.
static constexpr unsigned PT_TRIES = 65536;
__device__ __forceinline__ bool pt_wait(uint32_t bar, unsigned parity, uint32_t dead, unsigned tries) {
    unsigned ok;
    asm volatile("{\n .reg .pred p, q;\n .reg .u32 n, d;\n mov.u32 n, 0;\nWAIT:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n @p bra DONE;\n"
                 " ld.volatile.shared.u32 d, [%4];\n add.u32 n, n, 1;\n setp.eq.u32 q, d, 0;\n setp.lt.and.u32 q, n, %5, q;\n @q bra WAIT;\n st.volatile.shared.u32 [%4], 1;\nDONE:\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u), "r"(dead), "r"(tries) : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
// The same without being suspended, for the two warps that issue products: they are told some 100 clocks earlier (chunk 203 -> 198 us); of more warps the asking costs what it gains
__device__ __forceinline__ bool pt_poll(uint32_t bar, unsigned parity, uint32_t dead, unsigned tries) {
    unsigned ok;
    asm volatile("{\n .reg .pred p, q;\n .reg .u32 n, d;\n mov.u32 n, 0;\nWAIT:\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
                 " ld.volatile.shared.u32 d, [%3];\n add.u32 n, n, 1;\n setp.eq.u32 q, d, 0;\n setp.lt.and.u32 q, n, %4, q;\n @q bra WAIT;\n st.volatile.shared.u32 [%3], 1;\nDONE:\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(dead), "r"(tries << 8) : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ void pt_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pt_commit(uint32_t bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" :: "r"(bar) : "memory");
}
// The end of a warp that issues products: none is in flight when tensor memory is given back, whatever ran out before (the wait does not look at that)
__device__ __forceinline__ void pt_end(uint64_t * bar) {
    tc_commit(bar);
    for (unsigned n = 0; n < PT_TRIES && !mbar_try_wait(bar, 0u); n++) {}
    __syncwarp();
}
// N products of 16 steps of K each, both operands in shared memory, 32 bytes on from one to the next (64 columns of a piece are four); the first one adds to D if `add`
template <int N> __device__ __forceinline__ void pt_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    static_assert(N == 2 || N == 4, "");
    if constexpr (N == 4)
        asm volatile("{\n .reg .pred e, p, t;\n .reg .b64 a, b;\n elect.sync _|e, 0xffffffff;\n setp.ne.u32 p, %4, 0;\n setp.eq.u32 t, 0, 0;\n"
                     " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
                     " add.s64 a, %1, 4;\n add.s64 b, %2, 4;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n add.s64 a, %1, 6;\n add.s64 b, %2, 6;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add) : "memory");
    else
        asm volatile("{\n .reg .pred e, p, t;\n .reg .b64 a, b;\n elect.sync _|e, 0xffffffff;\n setp.ne.u32 p, %4, 0;\n setp.eq.u32 t, 0, 0;\n"
                     " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add) : "memory");
}
// Four products of 16 slots each, probabilities in tensor memory, 16 columns on from one to the next, values 2048 bytes on
__device__ __forceinline__ void pt_values(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n .reg .pred e, p, t;\n .reg .b32 a;\n .reg .b64 b;\n elect.sync _|e, 0xffffffff;\n setp.ne.u32 p, %4, 0;\n setp.eq.u32 t, 0, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n add.u32 a, %1, 16;\n add.s64 b, %2, 128;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n"
                 " add.u32 a, %1, 32;\n add.s64 b, %2, 256;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n add.u32 a, %1, 48;\n add.s64 b, %2, 384;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add) : "memory");
}
__device__ __forceinline__ void pt_store8(float * p, const float * v) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
// A place in a ring of barriers, and the parity of its phase
struct PtRing {
    uint32_t bar; unsigned at, parity;
    __device__ __forceinline__ PtRing(uint64_t * bars) : bar(smem_u32(bars)), at(0), parity(0) {}
    template <int N> __device__ __forceinline__ void step() { at++; if (at == N) { at = 0; parity ^= 1; } }
    __device__ __forceinline__ uint32_t here() const { return bar + at * 8u; }
};

// TWO: two halves for queries (FP32 rows)
template <int HD, bool TWO>
__global__ void __launch_bounds__(PT_THREADS, 1) k_attn_paged_tc(const __grid_constant__ PtP pp) {
    using Z = PtShape<HD, TWO>;
    constexpr int KS = HD / 16, SUBS = Z::SUBS, NV = SUBS * 64;       // steps of 16 columns; pieces of 64 columns of the values; columns of the sums (behind HV: unused)
    constexpr bool WIDE = Z::WIDE;
    constexpr uint32_t TILE = Z::TILE, FILL = Z::FILL;
    constexpr int NK = Z::NK, NW = Z::NW, QB = Z::QB;
    constexpr int OB = (512 - PT_GROUPS * PT_KEYS) / NV;              // buffers of sums.  (Two halves of 64 columns, of which one is drained while the other is made: products of 64 columns take as long as those of 128)
    constexpr int DH = Z::HV / 2, DC = DH == 48 ? 16 : 32;               // columns of a thread that drains, and at a time
    constexpr uint32_t T_S = 0, T_O = PT_GROUPS * PT_KEYS;            // tensor memory: three buffers of scores, one or two of sums
    static_assert(NK + PT_GROUPS < PT_INFO && OB >= 1 && PT_REGS_M + PT_REGS_Q + PT_GROUPS * PT_REGS_S + 2 * PT_REGS_D <= 7 * 72, "");
    const AttnPagedP & p = pp.a;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint64_t s_kfull[NK], s_kempty[NK], s_vfull[NW], s_vempty[NW];
    __shared__ uint64_t s_wfull[PT_WORK], s_wempty[PT_WORK], s_qfull[QB], s_qempty[QB];
    __shared__ uint64_t s_qk[PT_GROUPS], s_pv[PT_GROUPS], s_pfull[PT_GROUPS], s_stat[PT_GROUPS], s_scan[PT_GROUPS], s_fin[2], s_asked, s_over;
    __shared__ PtWork s_work[PT_WORK];
    __shared__ uint32_t s_tmem, s_info[PT_INFO];                      // of a tile: which groups of 16 slots are there; bit 8: special
    __shared__ volatile unsigned s_dead;
    __shared__ int s_given;                                           // pieces that this CTA had, there with s_over
    __shared__ uint32_t s_odd[PT_GROUPS][4];                           // slots of a special tile with a value that is not finite
    __shared__ float s_top[PT_GROUPS][PT_ROWS], s_sum[PT_GROUPS][PT_ROWS];         // of a tile: maximum, sum of the probabilities
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t queries = (smem_u32(smem_raw) + 1023u) & ~1023u, keys = queries + QB * Z::QUERIES, values = keys + NK * FILL;

    if (tid < NK) { mbar_init(s_kfull + tid, 1); mbar_init(s_kempty + tid, 1); }
    if (tid < NW) { mbar_init(s_vfull + tid, 1); mbar_init(s_vempty + tid, 1); }
    if (tid < PT_WORK) { mbar_init(s_wfull + tid, 1); mbar_init(s_wempty + tid, PT_THREADS / 32 - 3); }
    if (tid < QB) { mbar_init(s_qfull + tid, 1); mbar_init(s_qempty + tid, 1); }
    if (tid < PT_GROUPS) { mbar_init(s_qk + tid, 2); mbar_init(s_pv + tid, 1); mbar_init(s_pfull + tid, 12); mbar_init(s_stat + tid, 8); mbar_init(s_scan + tid, 4); }
    if (tid < 2) mbar_init(s_fin + tid, 1);
    if (tid == 2) mbar_init(&s_asked, 1);
    if (tid == 3) mbar_init(&s_over, 1);
    if (tid == 0) { s_dead = 0; s_given = 0; }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 0) tc_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    if (tid == 32) { tma_map(&pp.m_q); tma_map(&pp.m_k); tma_map(&pp.m_v); }
    pdl_launch();
    pdl_wait();
    asm volatile("fence.proxy.async;" ::: "memory");                // (what kernels before wrote is read by tensor copies)
    const uint32_t dead = smem_u32((const void *)&s_dead);
    auto wait_at = [&](uint32_t bar, unsigned parity) { return pt_wait(bar, parity, dead, pp.tries); };      // warp-uniform; false: the wait ran out, here or elsewhere in the CTA
    auto poll_at = [&](uint32_t bar, unsigned parity) { return pt_poll(bar, parity, dead, pp.tries); };
    auto wait = [&](uint64_t * bar, unsigned parity) { return wait_at(smem_u32(bar), parity); };
    auto work_of = [&](int n) { return s_work + n % PT_WORK; };
    auto done_with = [&](int n) { __syncwarp(); if (lane == 0) mbar_arrive(s_wempty + n % PT_WORK); };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(PT_REGS_M));
        if (warp == 0) {
            // ============================================================= scores
            bool ok = true;
            PtRing work(s_wfull), qs(s_qfull), buf(s_qk), slot_k(s_kfull);
            const uint32_t pv = smem_u32(s_pv), empty = smem_u32(s_kempty), qempty = smem_u32(s_qempty);
            int g = 0;                                                // tiles in all
            for (int n = 0; ok; n++, work.template step<PT_WORK>()) {
                ok = poll_at(work.here(), work.parity);
                if (!ok) break;
                const int tiles = __shfl_sync(0xffffffffu, s_work[work.at].tiles, 0), span = __shfl_sync(0xffffffffu, s_work[work.at].k1 - s_work[work.at].k0, 0);      // (uniform for the compiler)
                if (tiles < 0) break;
                if (tiles > 0) {
                    ok = poll_at(qs.here(), qs.parity);
                    const uint64_t q = tc_desc_k(queries + qs.at * Z::QUERIES);
                    for (int i = 0, left = span; i < tiles && ok; i++, g++, left -= PT_KEYS) {
                        const uint32_t idesc = tc_idesc(left >= PT_KEYS ? PT_KEYS : (left + 15) / 16 * 16, false), d = tmem + T_S + buf.at * PT_KEYS;
                        if constexpr (!WIDE) ok = poll_at(slot_k.here(), slot_k.parity);
                        if (g >= PT_GROUPS) ok = poll_at(pv + buf.at * 8, buf.parity ^ 1) && ok;       // the buffer's probabilities have been used
                        if (!ok) break;
                        tc_fence_after();
                        // (lower halves of the queries first)
                        if constexpr (WIDE) {
#pragma unroll 1
                            for (int c = 0; c < Z::QSUBS && (ok = poll_at(slot_k.here(), slot_k.parity)); c++) {
                                const uint64_t k = tc_desc_k(keys + slot_k.at * FILL);
                                tc_fence_after();
#pragma unroll 1
                                for (int low = TWO ? 1 : 0; low >= 0; low--) pt_scores<4>(d, q + (uint64_t)low * (Z::HALF >> 4) + c * (PT_SUB >> 4), k, idesc, (TWO && low == 0) || c > 0);
                                pt_commit(empty + slot_k.at * 8);
                                slot_k.template step<NK>();
                            }
                            if (!ok) break;
                        } else {
                            const uint64_t k = tc_desc_k(keys + slot_k.at * FILL);
#pragma unroll 1
                            for (int low = TWO ? 1 : 0; low >= 0; low--) {
#pragma unroll
                                for (int c = 0; c < SUBS; c++) {
                                    const uint64_t at = q + (uint64_t)low * (TILE >> 4) + c * (PT_SUB >> 4);
                                    if (KS - 4 * c >= 4) pt_scores<4>(d, at, k + c * (PT_SUB >> 4), idesc, (TWO && low == 0) || c > 0);
                                    else                 pt_scores<2>(d, at, k + c * (PT_SUB >> 4), idesc, (TWO && low == 0) || c > 0);
                                }
                            }
                        }
                        pt_commit(buf.here());
                        if (lane == 0) pt_arrive(buf.here());         // (what this warp has seen others write is seen by whoever waits)
                        __syncwarp();
                        if constexpr (!WIDE) pt_commit(empty + slot_k.at * 8);
                        if (i + 1 == tiles) pt_commit(qempty + qs.at * 8);
                        buf.template step<PT_GROUPS>();
                        if constexpr (!WIDE) slot_k.template step<NK>();
                    }
                    qs.template step<QB>();
                }
                if (ok) done_with(n);
            }
            pt_end(s_fin);
        } else if (warp == 2) {
            // ============================================================= sums of values
            constexpr uint32_t idesc_v = tc_idesc(NV, true);
            bool ok = true;
            PtRing work(s_wfull), buf(s_pfull), slot_v(s_vfull);
            const uint32_t pv = smem_u32(s_pv), empty = smem_u32(s_vempty);
            unsigned ob = 0;                                          // buffer of sums
            for (int n = 0; ok; n++, work.template step<PT_WORK>()) {
                ok = poll_at(work.here(), work.parity);
                if (!ok) break;
                const int tiles = __shfl_sync(0xffffffffu, s_work[work.at].tiles, 0), span = __shfl_sync(0xffffffffu, s_work[work.at].k1 - s_work[work.at].k0, 0);
                if (tiles < 0) break;
                for (int i = 0, left = span; i < tiles; i++, left -= PT_KEYS) {
                    const uint32_t a = tmem + T_S + buf.at * PT_KEYS, d = tmem + T_O + ob * NV;
                    const uint64_t v = tc_desc_mn(values + slot_v.at * TILE, PT_SUB);
                    const int steps = left >= PT_KEYS ? PT_KEYS / 16 : (left + 15) / 16;
                    ok = poll_at(slot_v.here(), slot_v.parity);
                    ok = poll_at(buf.here(), buf.parity) && ok;       // (the buffer of sums has been drained too)
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int low = 1; low >= 0; low--) {              // (lower halves of the probabilities first)
                        int j = 0;
#pragma unroll 1
                        for (; j + 4 <= steps; j += 4) pt_values(d, a + (uint32_t)(j * 16 + low * 8), v + 128 * j, idesc_v, low == 0 || j > 0);
#pragma unroll 1
                        for (; j < steps; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16 + low * 8), v + 128 * j, idesc_v, low == 0 || j > 0);
                    }
                    pt_commit(pv + buf.at * 8);
                    pt_commit(empty + slot_v.at * 8);
                    buf.template step<PT_GROUPS>();
                    slot_v.template step<NW>();
                    if (++ob == OB) ob = 0;
                }
                if (ok) done_with(n);
            }
            pt_end(s_fin + 1);
        } else {
            // ============================================================= tiles of keys (warp 1) and of values (warp 3): a lane takes a copy of 64 columns of a box's rows
            const bool is_k = warp == 1;
            const CUtensorMap * map = is_k ? &pp.m_k : &pp.m_v;
            const uint32_t full = smem_u32(is_k ? s_kfull : s_vfull), empty = smem_u32(is_k ? s_kempty : s_vempty), lot = is_k ? keys : values;
            const unsigned slots = is_k ? NK : NW;
            const uint32_t fill = is_k ? FILL : TILE;
            const int side = SUBS == 1 || (WIDE && is_k) ? 1 : 2, fills = WIDE && is_k ? Z::QSUBS : 1;       // copies side by side; places that a tile takes
            const int box = side == 2 ? lane >> 1 : lane, x = side == 2 ? (lane & 1) * 64 : 0;
            const bool mine = box * pp.box < PT_KEYS;
            const uint32_t place = (uint32_t)(x >> 6) * PT_SUB + (uint32_t)(box * pp.box) * 128u;
            unsigned slot = 0, parity = 0;
            int at = 0, asked = 0;                                    // tiles in all, places
            bool ok = true;
            for (int n = 0; ok; n++) {
                ok = wait(s_wfull + n % PT_WORK, n / PT_WORK & 1);
                if (!ok) break;
                const PtWork * w = work_of(n);
                const int tiles = w->tiles;
                if (tiles < 0) break;
                auto look = [&](int i) {                              // this lane's row in the pool, -1: not there
                    const int j = w->k0 + i * PT_KEYS + box * pp.box;
                    if (!mine || j >= w->there) return -1;
                    const int page = page_of(p.c, w->s.sq, j >> p.c.shift);
                    return page < 0 ? -1 : ((page * p.c.H + w->hk) << p.c.shift) + (j & (p.c.page - 1));
                };
                int y = tiles > 0 ? look(0) : -1;
                for (int i = 0; i < tiles; i++, at++) {
                    const int row = y;
                    const unsigned copies = __ballot_sync(0xffffffffu, row >= 0);
                    if (is_k) {                                       // which groups of 16 slots are there; whether the tile is special
                        const int j0 = w->k0 + i * PT_KEYS, of = (lane & 7) * 16 / pp.box * side;
                        const uint32_t groups = __ballot_sync(0xffffffffu, lane < 8 && j0 + lane * 16 < w->there && (copies >> of & 1));
                        if (lane == 0) s_info[at % PT_INFO] = groups | (groups != 0xffu || j0 + PT_KEYS > w->clear ? 256u : 0u);
                    }
                    for (int c = 0; c < fills; c++, asked++) {
                        if (asked >= (int)slots && !(ok = wait_at(empty + slot * 8, parity ^ 1))) break;
                        if (lane == 0) mbar_expect_tx((is_k ? s_kfull : s_vfull) + slot, (unsigned)__popc(copies) * pp.box * 128u);
                        __syncwarp();
                        if (row >= 0) tma_tile(lot + slot * fill + place, map, x + (!WIDE ? 0 : is_k ? c * 64 : w->v0), row, (is_k ? s_kfull : s_vfull) + slot);
                        if (c == 0 && i + 1 < tiles) y = look(i + 1);
                        __syncwarp();
                        if (++slot == slots) { slot = 0; parity ^= 1; }
                    }
                    if (!ok) break;
                }
                if (is_k && ok && lane == 0) mbar_arrive(&s_asked);   // (the next piece may be taken)
                if (ok) done_with(n);
            }
            if (lane == 0) ring_land(is_k ? s_kfull : s_vfull, asked, (int)slots);      // (whoever was to wait for them may have given up)
            __syncwarp();
        }
    } else if (warp < 8) {
        // ================================================================= work and its queries (warp 4; 5..7 have nothing to do)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(PT_REGS_Q));
        if (warp == 4) {
            int unit = blockIdx.x;
            auto take = [&]() {
                int then = 0;
                if (lane == 0) then = (int)gridDim.x + (int)atomicAdd(pp.next, 1u);
                unit = __shfl_sync(0xffffffffu, then, 0);
            };
            PtRing qs(s_qfull);
            const uint32_t qempty = smem_u32(s_qempty);
            bool ok = true;
            int u = 0, given = 0;                                     // pieces with tiles, pieces
            for (int n = 0; ok; n++) {
                if (n >= PT_WORK && !(ok = wait(s_wempty + n % PT_WORK, n / PT_WORK & 1 ^ 1))) break;
                // the next piece when the keys of the last one have all been asked for, two or three tiles before it ends: taken as soon as there is room, all pieces of a call of 400
                // were dealt out at its start, and one CTA had 38 tiles where 29 is the mean (trees of many users)
                if (n > 0) {
                    if (!(ok = wait(&s_asked, n & 1 ^ 1) && __all_sync(0xffffffffu, s_dead == 0))) break;       // (nothing is taken behind a wait that ran out)
                    take();
                }
                PtWork w;
                w.tiles = -1;
                while (unit < pp.units) {                             // the next piece that has something to do
                    w = pt_piece<WIDE, Z::HV>(pp, unit);
                    if (w.tiles >= 0) break;
                    take();
                }
                if (lane == 0) { *work_of(n) = w; mbar_arrive(s_wfull + n % PT_WORK); }
                __syncwarp();
                if (w.tiles < 0) break;
                given = n + 1;
                if (w.tiles > 0) {
                    if (u >= QB && !(ok = wait_at(qempty + qs.at * 8, qs.parity ^ 1))) break;
                    u++;
                    if (lane == 0) {
                        mbar_expect_tx(s_qfull + qs.at, Z::QUERIES);
                        const int row = (w.hk * p.b.T + w.s.first) * p.group + w.first;
                        for (int low = 0; low <= (TWO ? 1 : 0); low++)
                            for (int c = 0; c < Z::QSUBS; c++)
                                tma_tile(queries + qs.at * Z::QUERIES + low * Z::HALF + c * PT_SUB, &pp.m_q, c * 64, row + low * p.c.H * p.b.T * p.group, s_qfull + qs.at);
                    }
                    __syncwarp();
                    qs.template step<QB>();
                }
                done_with(n);
            }
            if (lane == 0) { s_given = given; mbar_arrive(&s_over); ring_land(s_qfull, u, QB); }
            __syncwarp();
        }
    } else if (warp < 8 + 4 * PT_GROUPS) {
        // ================================================================= probabilities: a row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(PT_REGS_S));
        const int b = (warp - 8) >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_S + (uint32_t)(b * PT_KEYS);
        const uint32_t qk = smem_u32(s_qk + b), stat = smem_u32(s_stat + b), pfull = smem_u32(s_pfull + b);
        int g = 0, at = b;                                            // tiles in all; the group's next one
        unsigned parity = 0, scans = 0;                               // of the group's barriers; special tiles so far
        bool ok = true;
        for (int n = 0; ok; n++) {
            ok = wait(s_wfull + n % PT_WORK, n / PT_WORK & 1);
            if (!ok) break;
            const PtWork * w = work_of(n);
            const int tiles = w->tiles, span = w->k1 - w->k0;
            if (tiles < 0) break;
            // (-infinity times 0 would be no number)
            const float f = fmaxf(TWO ? (r < w->n_rows ? __ldg(p.factor + (size_t)(w->hk * p.b.T + w->s.first) * p.group + w->first + r) : 0.f) : fabsf(p.scale_log2), 0x1p-126f);
            // the words of its mask (of trees of more than 128 tokens only when they are needed)
            const int tok = r < w->n_rows ? p.by_group.of(w->first + r) : 0x7fffffff;
            uint64_t word[2] = {0, 0};
            if (p.mask && r < w->n_rows) {
                const uint64_t * m = p.mask + (size_t)(w->s.first + tok) * p.words;
                word[0] = __ldg(m);
                if (p.words > 1) word[1] = __ldg(m + 1);
            }
            const bool idle = (warp & 3) * 32 >= w->n_rows;           // no rows: their probabilities may be anything
            for (; at < g + tiles; at += PT_GROUPS, parity ^= 1) {
                const int i = at - g;
                if (!(ok = wait_at(qk, parity))) break;
                tc_fence_after();
                const uint32_t info = s_info[at % PT_INFO];
                const bool masked = info & 256u;
                uint32_t sees[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                if (masked && !idle) {
                    ap_sees128(p, w->s, tok, w->k0 + i * PT_KEYS - w->s.pos, word, sees);
#pragma unroll
                    for (int c = 0; c < 4; c++) sees[c] &= ((info >> (2 * c) & 1 ? 0x0000ffffu : 0u) | (info >> (2 * c + 1) & 1 ? 0xffff0000u : 0u));
                }
                const int chunks = idle ? 0 : min(4, (span - i * PT_KEYS + 31) >> 5);         // of 32 slots
                float m = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < chunks; c++) {
                    float x[32];
                    tc_ld32(x, mine + 32 * c);
                    if (masked) {                                     // the scores of slots that a row does not see are put back as -infinity: their probabilities are 0
                        const uint32_t see = c == 0 ? sees[0] : c == 1 ? sees[1] : c == 2 ? sees[2] : sees[3];
                        if (__any_sync(0xffffffffu, see != 0xffffffffu)) {
#pragma unroll
                            for (int j = 0; j < 32; j++) if (!(see >> j & 1)) x[j] = -INFINITY;
                            tc_st32(mine + 32 * c, x);
                        }
                    }
                    float a[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) a[j] = max3(x[j], x[4 + j], x[8 + j]);
#pragma unroll
                    for (int j = 0; j < 4; j++) a[j] = max3(a[j], x[12 + j], x[16 + j]);
#pragma unroll
                    for (int j = 0; j < 4; j++) a[j] = max3(a[j], x[20 + j], x[24 + j]);
#pragma unroll
                    for (int j = 0; j < 4; j++) a[j] = fmaxf(a[j], x[28 + j]);
                    m = fmaxf(m, max3(a[0], a[1], fmaxf(a[2], a[3])));
                }
                if (masked) tc_wait_st();
                const bool none = m == -INFINITY;
                m *= f;
                const float2 ref = f2(none ? 14.f : 14.f - m), fc = f2(f);
                float2 l[2] = {f2(0.f), f2(0.f)};
#pragma unroll 1
                for (int c = 0; c < chunks; c++) {
                    float x[32];
                    tc_ld32(x, mine + 32 * c);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t hl[16];                              // upper parts of 16 slots, then lower parts
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const float2 y = f2_fma(make_float2(x[h * 16 + j], x[h * 16 + j + 1]), fc, ref), pr = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                            l[j >> 1 & 1] = f2_add(l[j >> 1 & 1], pr);
                            f2_split(pr, hl[j / 2], hl[8 + j / 2]);
                        }
                        tc_st16(mine + 32 * c + 16 * h, hl);
                    }
                }
                float total = (l[0].x + l[0].y) + (l[1].x + l[1].y);
                if (masked) {
                    // the tile's values: a row a thread.  Rows of slots that are not there become zeros; so do those with a value that is not finite, and who sees them has no numbers
                    // (A wait tells phases apart by their parity alone: first the place's former tile has to be used up.  With three places and more it is, as this tile's scores took its buffer.)
                    const int slot = at % NW, former = at - NW;
                    if (NW < PT_GROUPS && former >= 0 && !(ok = wait(s_pv + former % PT_GROUPS, former / PT_GROUPS & 1))) break;
                    if (!(ok = wait(s_vfull + slot, at / NW & 1))) break;
                    const int at_slot = w->k0 + i * PT_KEYS + r;
                    const bool is = info >> (r >> 4) & 1 && at_slot < w->there;
                    const uint32_t row = values + (uint32_t)slot * TILE + (uint32_t)r * 128u;
                    const __half2 null = __floats2half2_rn(0.f, 0.f);
                    __half2 zero[4] = {null, null, null, null};       // no more 0 where a value is not finite
                    if (is && at_slot >= w->clear) {                  // (what every row sees may be anything)
#pragma unroll 4
                        for (int u = 0; u < SUBS * 8; u++) {
                            uint4 x;
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(row + (uint32_t)(u >> 3) * PT_SUB + (uint32_t)((u + lane) & 7) * 16u));
                            const __half2 * v = reinterpret_cast<const __half2 *>(&x);
#pragma unroll
                            for (int c = 0; c < 4; c++) zero[c] = __hfma2(v[c], null, zero[c]);
                        }
                    }
                    const bool odd = !__hbeq2(__hadd2(__hadd2(zero[0], zero[1]), __hadd2(zero[2], zero[3])), null);
                    if (!is || odd) {
#pragma unroll 2
                        for (int u = 0; u < SUBS * 8; u++)
                            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" :: "r"(row + (uint32_t)(u >> 3) * PT_SUB + (uint32_t)((u + lane) & 7) * 16u), "r"(0u) : "memory");
                    }
                    tc_fence_smem();
                    const uint32_t word = __ballot_sync(0xffffffffu, odd);
                    if (lane == 0) { s_odd[b][warp & 3] = word; mbar_arrive(s_scan + b); }
                    if (!(ok = wait(s_scan + b, scans & 1))) break;   // the group's other warps have their words there
                    scans++;
                    uint32_t none_of = 0;
#pragma unroll
                    for (int c = 0; c < 4; c++) none_of |= sees[c] & s_odd[b][c];
                    if (none_of) total = __int_as_float(0x7fc00000);
                }
                if (none && (sees[0] | sees[1] | sees[2] | sees[3])) total = __int_as_float(0x7fc00000);         // (every score that it sees is -infinity)
                if (at >= PT_GROUPS && !(ok = wait_at(stat, parity ^ 1))) break;                // what was there before has been read
                s_sum[b][r] = total;
                s_top[b][r] = m;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) pt_arrive(pfull);
            }
            g += tiles;
            if (ok) done_with(n);
        }
        tc_wait_st();                                                 // (of a tile that was given up)
    } else {
        // ================================================================= sums out
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(PT_REGS_D));
        const int r = (warp & 3) * 32 + lane, d0 = warp >= 24 ? DH : 0;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_O + (uint32_t)d0;
        PtRing buf(s_pfull);
        const uint32_t pfull = smem_u32(s_pfull), pv = smem_u32(s_pv), stat = smem_u32(s_stat);
        unsigned ob = 0;                                              // buffer of sums
        bool ok = true;
        if (lane == 0) for (int i = 0; i < OB; i++) pt_arrive(pfull + i * 8);       // (nothing to drain before the first tiles)
        for (int n = 0; ; n++) {
            if (ok) ok = wait(s_wfull + n % PT_WORK, n / PT_WORK & 1);
            if (!ok) {                                                // after a wait that ran out: the rows of the pieces in hand are no numbers
                for (unsigned k = 0; k < PT_TRIES && !mbar_try_wait(&s_over, 0u); k++) {}
                __syncwarp();
                if (n >= __shfl_sync(0xffffffffu, s_given, 0)) break;
            }
            const PtWork * w = work_of(n);
            const int tiles = w->tiles;
            if (tiles < 0) break;
            float top = -INFINITY, sum = 0.f;
            float acc[DH];
#pragma unroll
            for (int j = 0; j < DH; j++) acc[j] = 0.f;
            for (int i = 0; i < tiles && ok; i++) {
                const int b = buf.at;
                ok = wait_at(buf.here(), buf.parity);
                const float m = s_top[b][r], of = s_sum[b][r], now = fmaxf(top, m);
                __syncwarp();
                if (lane == 0) pt_arrive(stat + b * 8);
                const float was = top == now ? 1.f : exp2_approx(top - now), is = m == -INFINITY ? 0.f : exp2_approx(m - now);
                top = now;
                sum = fmaf(sum, was, of * is);
                ok = wait_at(pv + b * 8, buf.parity) && ok;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < DH; c += DC) {
                    float v[DC];
                    if constexpr (DC == 32) tc_ld32(v, mine + ob * NV + c); else tc_ld16(v, mine + ob * NV + c);
                    if (c + DC == DH) {                           // the buffer goes back
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) pt_arrive(pfull + (buf.at + OB >= PT_GROUPS ? buf.at + OB - PT_GROUPS : buf.at + OB) * 8);
                    }
#pragma unroll
                    for (int j = 0; j < DC; j += 2) {
                        const float2 o = f2_fma(make_float2(v[j], v[j + 1]), f2(is), f2_mul(make_float2(acc[c + j], acc[c + j + 1]), f2(was)));
                        acc[c + j] = o.x; acc[c + j + 1] = o.y;
                    }
                }
                buf.template step<PT_GROUPS>();
                if (++ob == OB) ob = 0;
            }
            if (r < w->n_rows) {
                const int row = w->first + r, of = p.by_group.of(row), h = w->hk * p.group + row - of * p.group;
                if (of >= p.c.n_ctx - w->s.pos) {                     // a token without a slot of its own
                    top = -INFINITY; sum = 0.f;
#pragma unroll
                    for (int j = 0; j < DH; j++) acc[j] = 0.f;
                }
                if (!ok || s_dead) sum = __int_as_float(0x7fc00000);  // a wait ran out, here or in a warp that came to s_pfull all the same: no numbers instead of wrong ones
                // (32 bytes a store where rows lie so: a row a thread meets a line of its own at every store)
                if (w->dst >= 0) {
                    const size_t at = (size_t)w->dst * PT_ROWS + r;
                    if (WIDE && sum != sum) {                         // (the part's sum stands for both halves of the columns, no numbers for the one that has them)
#pragma unroll
                        for (int j = 0; j < DH; j++) acc[j] = sum;
                    }
#pragma unroll
                    for (int j = 0; j < DH; j += 8) pt_store8(p.part + at * HD + w->v0 + d0 + j, acc + j);
                    if (d0 + w->v0 == 0) p.part_ml[at] = make_float2(top, sum);
                } else {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    const size_t at = (size_t)(w->s.first + of) * p.out_stride + (size_t)h * HD + w->v0 + d0;
#pragma unroll
                    for (int j = 0; j < DH; j++) acc[j] *= inv;
                    if constexpr (!TWO) {
#pragma unroll
                        for (int j = 0; j < DH; j += 8) {
                            uint4 u;
                            u.x = h2u(__floats2half2_rn(acc[j], acc[j + 1])); u.y = h2u(__floats2half2_rn(acc[j + 2], acc[j + 3]));
                            u.z = h2u(__floats2half2_rn(acc[j + 4], acc[j + 5])); u.w = h2u(__floats2half2_rn(acc[j + 6], acc[j + 7]));
                            *reinterpret_cast<uint4 *>((__half *)p.out + at + j) = u;
                        }
                    } else if (pp.wide) {
#pragma unroll
                        for (int j = 0; j < DH; j += 8) pt_store8((float *)p.out + at + j, acc + j);
                    } else {
#pragma unroll
                        for (int j = 0; j < DH; j += 4) *reinterpret_cast<float4 *>((float *)p.out + at + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                    }
                }
            }
            if (ok) done_with(n);
        }
        if (!ok) {                                                    // nor are those of pieces that nobody may take any more: a warp of these takes one at a time
            for (;;) {
                int unit = 0;
                if (lane == 0) unit = (int)gridDim.x + (int)atomicAdd(pp.next, 1u);
                unit = __shfl_sync(0xffffffffu, unit, 0);
                if (unit >= pp.units) break;
                const PtWork w = pt_piece<WIDE, Z::HV>(pp, unit);
                const float none = __int_as_float(0x7fc00000);
                for (int row = lane; w.tiles >= 0 && row < w.n_rows; row += 32) {
                    const int of = p.by_group.of(w.first + row), h = w.hk * p.group + w.first + row - of * p.group;
                    const size_t at = (size_t)(w.s.first + of) * p.out_stride + (size_t)h * HD + w.v0, part = (size_t)w.dst * PT_ROWS + row;
                    if (w.dst >= 0 && w.v0 == 0) p.part_ml[part] = make_float2(-INFINITY, none);
#pragma unroll 1
                    for (int j = 0; j < Z::HV; j++) {
                        if (w.dst >= 0)   p.part[part * HD + w.v0 + j] = none;
                        else if (TWO)     ((float *)p.out)[at + j] = none;
                        else              ((__half *)p.out)[at + j] = __float2half_rn(none);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tc_dealloc(s_tmem, 512);
    if (tid == 0 && s_dead) atomicOr(p.status, 16u);
}

// In front of the kernel: its queries as it takes them, halves [low][KV head][row of the group's tokens][HD], and of FP32 rows the factors of their scores; and the status word and the number of the next
// piece cleared (no CTA of the kernel can, as another one may have been at them by then).  A row, over a power of two of its largest value where it is FP32, is one or the sum of two halves; negative
// where the scale is (the factor of the scores is positive: maxima stay maxima).  Eight threads take a row.
template <int HD, bool TWO>
__global__ void __launch_bounds__(256) k_attn_paged_queries(const AttnPagedP p, __half * to, float * factor, unsigned int * next) {
    const int part = threadIdx.x & 7, head = p.n_head, at = blockIdx.x * 32 + (threadIdx.x >> 3);
    pdl_launch();
    pdl_wait();
    if (at == 0 && part == 0) { *p.status = 0u; *next = 0u; }
    if (at >= p.b.T * head) return;                                   // (the same for the eight)
    const int tok = at / head, h = at - tok * head, hk = h / p.group, rows = p.b.T * p.group;
    const size_t row = (size_t)hk * rows + (size_t)tok * p.group + (h - hk * p.group);
    const unsigned mine = 0xffu << (threadIdx.x & 24);
    if constexpr (!TWO) {
        constexpr int N = (HD / 8 + 7) / 8;
        const uint4 * from = reinterpret_cast<const uint4 *>((const __half *)p.q + (size_t)tok * p.q_stride + (size_t)h * HD);
        uint4 x[N];
        const __half2 none = __floats2half2_rn(0.f, 0.f);
        __half2 zero = none;
#pragma unroll
        for (int j = 0; j < N; j++) {
            x[j] = make_uint4(0u, 0u, 0u, 0u);
            if (j * 8 + part < HD / 8) x[j] = __ldg(from + j * 8 + part);
            const __half2 * v = reinterpret_cast<const __half2 *>(x + j);
#pragma unroll
            for (int c = 0; c < 4; c++) zero = __hfma2(v[c], none, zero);
        }
        // a value that is not finite: the row's scores are no numbers (an infinity alone may make them all the lowest value, as if the row saw nothing)
        if (!__hbeq2(zero, none)) x[0].x = 0x7fff7fffu;
        const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j * 8 + part < HD / 8) reinterpret_cast<uint4 *>(to + row * HD)[j * 8 + part] = make_uint4(x[j].x ^ sign, x[j].y ^ sign, x[j].z ^ sign, x[j].w ^ sign);
    } else {
        constexpr int N = HD / 32;
        const float4 * from = reinterpret_cast<const float4 *>((const float *)p.q + (size_t)tok * p.q_stride + (size_t)h * HD);
        float4 v[N];
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = __ldg(from + j * 8 + part);
#pragma unroll
        for (int j = 0; j < N; j++) m = fmaxf(fmaxf(m, fmaxf(fabsf(v[j].x), fabsf(v[j].y))), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(mine, m, o));
        const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127) - 10;     // the largest to 2^10 .. 2^11: lower parts are then exact to 2^-25
        const float up = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), p.scale_log2);
        if (part == 0) factor[row] = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int j = 0; j < N; j++) {
            uint2 hi, lo;
            aq_split(v[j].x * up, v[j].y * up, hi.x, lo.x);
            aq_split(v[j].z * up, v[j].w * up, hi.y, lo.y);
            reinterpret_cast<uint2 *>(to + row * HD)[j * 8 + part] = hi;
            reinterpret_cast<uint2 *>(to + ((size_t)p.c.H * rows + row) * HD)[j * 8 + part] = lo;
        }
    }
}

// With mma.sync every 16 rows of a KV head read its keys and values again, 16 us for 2^25 values of keys (after the first ones); here 128 rows take 5 us more whatever there is, and 7 us more for as many values.
// Both sides measured (us, here and with mma.sync; FP32, 4 query heads a KV head, head_dim 128): 8 sequences of 4096 slots and 8 KV heads 16 rows 39 and 28, 24 rows 38 and 43, 64 rows 39 and 74; one such
// sequence 24 rows 17 and 14, 48 rows 18 and 16, 64 rows 18 and 17; one of 500 slots and 32 KV heads 64 rows 15 and 14.
// The same of head_dim 256 and 192: 8 sequences of 4096 24 rows 86 and 99, 69 and 82; one 24 rows 23 and 21, 21 and 18; 64 rows 23 and 32, 22 and 28; one of 500 and 32 KV heads of 256 64 rows 19 and 19, 128 rows 21 and 36.
// FP16 rows of 128: 8 sequences of 4096 24 rows 35 and 37, 64 rows 36 and 63; one 24 rows 16 and 13, 48 rows 17 and 14, 64 rows 17 and 16.
// (PI_ATTN_TREE_TC=1 takes 17 rows and more whatever there is, 0 none: a diagnostic switch, read once.)
bool attn_paged_tc_takes(int64_t rows, double values) {
    static int forced = -2;
    if (forced == -2) { const char * v = getenv("PI_ATTN_TREE_TC"); forced = v ? v[0] != '0' : -1; }
    if (rows <= 16 || forced == 0) return false;
    return forced == 1 || ((rows + 15) / 16 - 1) * 16 * values > 5.0 * (1 << 25) + 7.0 * values;
}

template <int HD, bool TWO>
static int pt_go(const AttnPagedP & a, cudaStream_t st) {
    constexpr size_t smem = PtShape<HD, TWO>::SMEM;
    static bool done[16] = {false};
    int dev = 0, rc;
    PI_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_attn_paged_tc<HD, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PtP p;
    p.a = a;
    p.box = a.c.page < PT_BOX ? a.c.page : PT_BOX;
    const int64_t rows = (int64_t)a.c.n_pages * a.c.H * a.c.page;
    if ((rc = tensor_map(&p.m_k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.k, HD, rows, HD * 2, 64, p.box, CU_TENSOR_MAP_SWIZZLE_128B)) ||
        (rc = tensor_map(&p.m_v, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.c.v, HD, rows, HD * 2, 64, p.box, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    p.wide = ((uintptr_t)a.out & 31) == 0 && a.out_stride * 4 % 32 == 0;
    p.units = (int)ap_grid(a) * (PtShape<HD, TWO>::WIDE ? 2 : 1);
    p.next = a.status + 8;
    static const char * tries = getenv("PI_ATTN_TREE_TRIES");         // (a diagnostic switch, read once: how often the kernel's waits ask)
    p.tries = tries ? (unsigned)std::min(strtoul(tries, nullptr, 10), (unsigned long)PT_TRIES) : PT_TRIES;
    const int64_t q_rows = (int64_t)a.b.T * a.n_head;
    if ((rc = tensor_map(&p.m_q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.queries, HD, q_rows * (TWO ? 2 : 1), HD * 2, 64, PT_ROWS, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    PI_CUDA(launch_k(k_attn_paged_queries<HD, TWO>, dim3((unsigned)((q_rows + 31) / 32)), dim3(256), 0, st, true, a, a.queries, a.factor, p.next));
    PI_CUDA(launch_k(k_attn_paged_tc<HD, TWO>, dim3((unsigned)(p.units < sm_count() ? p.units : sm_count())), dim3(PT_THREADS), smem, st, true, p));
    return PI_OK;
}

int launch_attn_paged_tc(const AttnPagedP & p, cudaStream_t st) {
    const bool half = p.xtype == PI_TYPE_F16;
    switch (p.c.hd) {
        case 64: return half ? pt_go<64, false>(p, st) : pt_go<64, true>(p, st);
        case 96: return half ? pt_go<96, false>(p, st) : pt_go<96, true>(p, st);
        case 128: return half ? pt_go<128, false>(p, st) : pt_go<128, true>(p, st);
        case 192: return half ? pt_go<192, false>(p, st) : pt_go<192, true>(p, st);
        default: return half ? pt_go<256, false>(p, st) : pt_go<256, true>(p, st);
    }
}

}  // namespace pi
