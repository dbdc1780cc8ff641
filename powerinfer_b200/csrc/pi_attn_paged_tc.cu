// Attention over a paged cache for more than a few query rows of a KV head (trees of a group's heads, prompts) on tcgen05; formulas and rows as in pi_attn_paged.cu.
//
// A CTA takes 128 query rows (the lanes) of one KV head and walks over its slots in tiles of 128.  Queries lie in tensor memory for the whole walk.  A tile's keys and
// values come as tensor copies of one page's rows each into a ring of 128-byte swizzled rows of 64 halves, which is K-major for the scores and MN-major for the
// values.  Scores S = Q K^T are made into one of two buffers in tensor memory; the probabilities take their place; sums of values O = P V of ONE tile go to a third buffer, which is
// drained and added with rounding in registers: the tensor cores cut FP32 sums at every step, so that no sum stays with them for longer than a tile.
// So every tile has its own maximum (no exchange between tiles; the two score buffers are two groups of warps' own): the drain joins tiles.
//
// A tile is special where not every row of the CTA sees all of its slots: then two warps go over its values before they are used.  Rows of slots that are not there
// become zeros, values that are not finite too, and whoever sees such a slot has a row of no numbers; scores of slots that a row does not see are replaced by what its
// mask says.
//
// Precision.  FP32 rows: queries and probabilities are the sum of two halves each, 22 bits, i.e. two products in the place of one.  FP16 rows: queries as they are, probabilities
// one half, 11 bits like the result's own rounding.  Probabilities are held times 2^14, so their steps end 2^-38 below a tile's largest one.
//
// Warps: 0 issues the products; 1 asks for the tiles; 2 and 3 go over special tiles; 4..11 and 12..19 have the even and the odd tiles' probabilities, a row and half of the slots a thread (the
// halves tell each other their maxima); 20..27 drain the sums, a row and half of the columns a thread.
#include "pi_attn_paged.cuh"
#include "pi_tc.cuh"
#include "pi_tc_math.cuh"

#include <cfloat>
#include <type_traits>

namespace pi {

static constexpr int PT_THREADS = 896;
static constexpr int PT_REGS_M = 40, PT_REGS_S = 64, PT_REGS_D = 104;  // 40 + 4 x 64 + 2 x 104 of the 7 x 72 of the launch
static constexpr uint32_t PT_SUB = PT_KEYS * 128;                     // bytes of 64 columns of a tile
static constexpr int PT_BOX = 64;                                     // rows of a tensor copy, or a page's if it has fewer

struct PtP { AttnPagedP a; int box; CUtensorMap m_k, m_v; };

// TWO: two halves for queries and probabilities
template <int HD, bool TWO>
__global__ void __launch_bounds__(PT_THREADS, 1) k_attn_paged_tc(const __grid_constant__ PtP pp) {
    constexpr int KS = HD / 16, SUBS = (HD + 63) / 64, NV = SUBS * 64, NQ = HD / 4;       // steps of 16 columns; pieces of 64 columns; columns of the sums (behind HD: zeros); columns of a thread that loads queries
    constexpr uint32_t TILE = SUBS * PT_SUB;
    constexpr int NS = HD <= 64 ? 12 : 6, NP = NS / 2;                // tiles in the ring, keys and values in turn
    constexpr uint32_t T_Q = 0, T_S = NV, T_O = NV + 2 * PT_KEYS;     // tensor memory: queries (upper, lower), two buffers of scores, sums
    static_assert(T_O + NV <= 512 && PT_REGS_M + 4 * PT_REGS_S + 2 * PT_REGS_D <= 7 * 72, "");
    const AttnPagedP & p = pp.a;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint64_t s_full[NS], s_empty[NS], s_vok[NP];
    __shared__ uint64_t s_qk[2], s_pv[2], s_pfull[2], s_free[2], s_fin;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_dead;
    __shared__ uint32_t s_odd[NP][4];                                 // slots of a special tile with a value that is not finite
    __shared__ float s_f[PT_ROWS];                                    // factor of a row's scores
    __shared__ float s_max[2][2][PT_ROWS], s_sum[2][2][PT_ROWS];       // of a tile's halves: maximum, sum of the probabilities
    __shared__ float s_top[2][PT_ROWS];                               // maximum of a tile
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const AqItem w = ap_item(p, blockIdx.x);
    const int split = w.split, hk = w.hk, rt = p.row_tiles - 1 - w.rt;      // (the longest rows first)
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, w.entry);
    const TileP t = ap_tile(p, s, rt, PT_ROWS);
    if (t.n_rows <= 0) return;
    const int k0 = split * p.split, k1 = split == w.n_splits - 1 ? t.seen : min(t.seen, k0 + p.split);
    if (k0 >= k1 && split > 0) return;                                // (split 0 answers for rows that see nothing)
    const int n_tiles = k0 < k1 ? (k1 - k0 + PT_KEYS - 1) / PT_KEYS : 0;
    const int clear = p.mask ? s.pos : s.pos + p.by_group.of(t.first) + 1;      // every row sees the slots before it

    if (tid < NS) { mbar_init(s_full + tid, 1); mbar_init(s_empty + tid, 1); }
    if (tid < NP) mbar_init(s_vok + tid, 2);
    if (tid < 2) { mbar_init(s_qk + tid, 1); mbar_init(s_pv + tid, 1); mbar_init(s_pfull + tid, 16); mbar_init(s_free + tid, 8); }
    if (tid == 0) { mbar_init(&s_fin, 1); s_dead = 0; }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 0) tc_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    auto wait = [&](uint64_t * bar, unsigned parity) -> bool {        // warp-uniform; false: the wait ran out, here or elsewhere
        bool ok = __all_sync(0xffffffffu, mbar_try_wait(bar, parity));
        if (__builtin_expect(ok, 1)) return true;
        for (int spins = 0; spins < (1 << 20) && !ok && !s_dead; spins++) ok = mbar_try_wait(bar, parity);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok && lane == 0) { s_dead = 1; atomicOr(p.status, 16u); }
        return ok;
    };
    // which of a tile's eight groups of 16 slots are there
    auto present = [&](int i) -> uint32_t {
        const int j = k0 + i * PT_KEYS + (lane & 7) * 16;
        return __ballot_sync(0xffffffffu, lane < 8 && j < t.there && page_of(p.c, s.sq, j >> p.c.shift) >= 0);
    };
    auto special = [&](int i, uint32_t there) { return there != 0xffu || k0 + (i + 1) * PT_KEYS > clear; };

    // ---- tiles: the n-th is keys (even) or values (odd) of tile n / 2
    auto ask = [&](int n) {                                           // a whole warp: a lane takes a copy
        const int slot = n % NS, j = k0 + (n >> 1) * PT_KEYS + lane * pp.box;
        int page = -1;
        if (lane * pp.box < PT_KEYS && j < t.there) page = page_of(p.c, s.sq, j >> p.c.shift);
        const unsigned boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_expect_tx(s_full + slot, boxes * SUBS * pp.box * 128u);
        __syncwarp();
        if (page >= 0) {
            const int y = ((page * p.c.H + hk) << p.c.shift) + (j & (p.c.page - 1));
#pragma unroll
            for (int u = 0; u < SUBS; u++) tma_tile(ring + (uint32_t)slot * TILE + u * PT_SUB + (uint32_t)(lane * pp.box) * 128u, n & 1 ? &pp.m_v : &pp.m_k, u * 64, y, s_full + slot);
        }
        __syncwarp();
    };
    if (warp == 1) for (int n = 0; n < min(NS, 2 * n_tiles); n++) ask(n);

    // ---- queries into tensor memory: a row and a quarter of its columns a thread, straight from global memory
    if (warp >= 4 && warp < 20) {
        const int part = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, row = t.first + r, tok = p.by_group.of(row);
        const size_t from = (size_t)(s.first + tok) * p.q_stride + (size_t)(hk * p.group + row - tok * p.group) * HD + part * NQ;
        const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_Q + (uint32_t)(part * NQ / 2);
        if constexpr (!TWO) {
            uint32_t u[16];
#pragma unroll
            for (int j = 0; j < 16; j++) u[j] = 0u;
            if (r < t.n_rows) {
                const uint4 * at = reinterpret_cast<const uint4 *>((const __half *)p.q + from);
#pragma unroll
                for (int j = 0; j < NQ / 8; j++) { const uint4 v = __ldg(at + j); u[4 * j] = v.x; u[4 * j + 1] = v.y; u[4 * j + 2] = v.z; u[4 * j + 3] = v.w; }
            }
            // a value that is not finite: the row's scores are no numbers (an infinity alone may make them all the lowest value, as if the row saw nothing)
            const __half2 none = __floats2half2_rn(0.f, 0.f);
            __half2 zero[4] = {none, none, none, none};
#pragma unroll
            for (int j = 0; j < NQ / 2; j++) zero[j & 3] = __hfma2(*reinterpret_cast<const __half2 *>(&u[j]), none, zero[j & 3]);
            if (!__hbeq2(__hadd2(__hadd2(zero[0], zero[1]), __hadd2(zero[2], zero[3])), none)) u[0] = 0x7fff7fffu;
            if (p.scale_log2 < 0.f) {                                 // (the factor of the scores is positive: maxima stay maxima)
#pragma unroll
                for (int j = 0; j < 16; j++) u[j] ^= 0x80008000u;
            }
            if (part == 0) s_f[r] = fabsf(p.scale_log2);
            tc_put<NQ / 2>(to, u);
            tc_wait_st();
        } else {
            float4 v[NQ / 4];
            float m = 0.f;
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) {
                v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < t.n_rows) v[j] = __ldg(reinterpret_cast<const float4 *>((const float *)p.q + from) + j);
            }
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) m = fmaxf(fmaxf(m, fmaxf(fabsf(v[j].x), fabsf(v[j].y))), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
            s_max[part >> 1][part & 1][r] = m;
            asm volatile("bar.sync 3, 512;" ::: "memory");
            m = fmaxf(fmaxf(s_max[0][0][r], s_max[0][1][r]), fmaxf(s_max[1][0][r], s_max[1][1][r]));
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127) - 10;     // the largest to 2^10 .. 2^11: lower parts are then exact to 2^-25
            const float up = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), p.scale_log2);
            if (part == 0) s_f[r] = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23);
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int j = 0; j < 16; j++) hi[j] = lo[j] = 0u;
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) {
                aq_split(v[j].x * up, v[j].y * up, hi[2 * j], lo[2 * j]);
                aq_split(v[j].z * up, v[j].w * up, hi[2 * j + 1], lo[2 * j + 1]);
            }
            tc_put<NQ / 2>(to, hi);
            tc_put<NQ / 2>(to + HD / 2, lo);
            tc_wait_st();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    float top = -INFINITY, sum = 0.f;                                 // of a draining thread's row
    float acc[HD / 2];
#pragma unroll
    for (int j = 0; j < HD / 2; j++) acc[j] = 0.f;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(PT_REGS_M));
        if (warp == 0) {
            // ============================================================= products
            constexpr uint32_t idesc_v = tc_idesc(NV, true);
            const int tiles = __shfl_sync(0xffffffffu, n_tiles, 0), span = __shfl_sync(0xffffffffu, k1 - k0, 0);      // (uniform for the compiler)
            bool ok = true;
            auto scores = [&](int i) {
                const int b = i & 1, n = min(PT_KEYS, (span - i * PT_KEYS + 15) / 16 * 16), slot = 2 * i % NS;
                ok = wait(s_full + slot, 2 * i / NS & 1) && ok;
                if (!ok) return;
                tc_fence_after();
                const uint32_t idesc = tc_idesc(n, false), d = tmem + T_S + (uint32_t)(b * PT_KEYS);
                const uint64_t k = tc_desc_k(ring + (uint32_t)slot * TILE);
                if (TWO) {
#pragma unroll
                    for (int j = 0; j < KS; j++) tc_mma_f16_ta(d, tmem + T_Q + HD / 2 + 8 * j, k + (j >> 2) * (PT_SUB >> 4) + 2 * (j & 3), idesc, j > 0);
                }
#pragma unroll
                for (int j = 0; j < KS; j++) tc_mma_f16_ta(d, tmem + T_Q + 8 * j, k + (j >> 2) * (PT_SUB >> 4) + 2 * (j & 3), idesc, TWO || j > 0);
                tc_commit(s_empty + slot);
                tc_commit(s_qk + b);
            };
            if (tiles > 0) scores(0);
            if (tiles > 1) scores(1);
            for (int i = 0; i < tiles && ok; i++) {
                const int b = i & 1, steps = min(PT_KEYS / 16, (span - i * PT_KEYS + 15) / 16), slot = (2 * i + 1) % NS;
                ok = wait(s_vok + (slot >> 1), (2 * i + 1) / NS & 1) && ok;
                ok = wait(s_pfull + b, i >> 1 & 1) && ok;             // (the sums before are drained too)
                if (!ok) break;
                tc_fence_after();
                const uint32_t a = tmem + T_S + (uint32_t)(b * PT_KEYS), d = tmem + T_O;
                const uint64_t v = tc_desc_mn(ring + (uint32_t)slot * TILE, PT_SUB);
                if (steps == PT_KEYS / 16) {
                    if (TWO) {
#pragma unroll
                        for (int j = 0; j < PT_KEYS / 16; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16 + 8), v + 128 * j, idesc_v, j > 0);
                    }
#pragma unroll
                    for (int j = 0; j < PT_KEYS / 16; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16), v + 128 * j, idesc_v, TWO || j > 0);
                } else {
                    if (TWO) for (int j = 0; j < steps; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16 + 8), v + 128 * j, idesc_v, j > 0);
                    for (int j = 0; j < steps; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16), v + 128 * j, idesc_v, TWO || j > 0);
                }
                tc_commit(s_empty + slot);
                tc_commit(s_pv + b);
                if (i + 2 < tiles) scores(i + 2);
            }
            tc_commit(&s_fin);                                        // nothing is in flight when tensor memory is given back
            for (int spins = 0; spins < (1 << 20) && !mbar_try_wait(&s_fin, 0u); spins++) {}
            __syncwarp();
        } else if (warp == 1) {
            // ============================================================= tiles
            int n = min(NS, 2 * n_tiles);
            for (; n < 2 * n_tiles; n++) {
                if (!wait(s_empty + n % NS, n / NS & 1 ^ 1)) break;
                ask(n);
            }
            if (lane == 0) ring_land(s_full, n, NS);
            __syncwarp();
        } else {
            // ============================================================= special tiles' values
            for (int i = 0; i < n_tiles; i++) {
                const int n = 2 * i + 1, slot = n % NS;
                const uint32_t groups = present(i);
                if (!wait(s_full + slot, n / NS & 1)) break;
                if (special(i, groups)) {
                    const int j0 = k0 + i * PT_KEYS;
                    for (int h = 0; h < 2; h++) {                     // rows 0 .. 31 and 64 .. 95, or the others
                        const int r = h * 64 + (warp - 2) * 32 + lane;
                        const bool there = groups >> (r >> 4) & 1 && j0 + r < t.there;
                        bool odd = false;
                        for (int u = 0; u < SUBS * 8; u++) {
                            const uint32_t at = ring + (uint32_t)slot * TILE + (uint32_t)(u >> 3) * PT_SUB + (uint32_t)r * 128u + (uint32_t)((u + lane) & 7) * 16u;
                            uint32_t x[4] = {0u, 0u, 0u, 0u};
                            bool bad = !there;
                            if (there) {
                                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
#pragma unroll
                                for (int c = 0; c < 4; c++) {
                                    if ((x[c] & 0x7c00u) == 0x7c00u) { bad = odd = true; x[c] &= 0xffff0000u; }
                                    if ((x[c] & 0x7c000000u) == 0x7c000000u) { bad = odd = true; x[c] &= 0x0000ffffu; }
                                }
                            }
                            if (bad) asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                        }
                        const uint32_t word = __ballot_sync(0xffffffffu, odd);
                        if (lane == 0) s_odd[slot >> 1][h * 2 + warp - 2] = word;
                    }
                    tc_fence_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(s_vok + (slot >> 1));
            }
        }
    } else if (warp < 20) {
        // ================================================================= probabilities
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(PT_REGS_S));
        const int b = (warp - 4) >> 3, half = (warp - 4) >> 2 & 1, r = (warp & 3) * 32 + lane;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_S + (uint32_t)(b * PT_KEYS + half * 64);
        const bool idle = (warp & 3) * 32 >= t.n_rows;                // no rows: their probabilities may be anything
        const int tok = r < t.n_rows ? p.by_group.of(t.first + r) : 0x7fffffff;
        const float f = s_f[r];
        uint32_t next = b < n_tiles ? present(b) : 0u;
        for (int i = b; i < n_tiles; i += 2) {                        // (to the end whatever waits ran out: the halves meet at a barrier)
            const uint32_t groups = next;
            const bool masked = special(i, groups);
            const int j0 = k0 + i * PT_KEYS + half * 64;
            if (i + 2 < n_tiles) next = present(i + 2);
            uint32_t sees[2] = {0xffffffffu, 0xffffffffu};
            if (masked && !idle) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t g = groups >> (half * 4 + c * 2);
                    sees[c] = ap_sees(p, s, tok, j0 + c * 32 - s.pos) & ((g & 1 ? 0x0000ffffu : 0u) | (g & 2 ? 0xffff0000u : 0u));
                }
            }
            const int parts = idle ? 0 : max(0, min(4, (k1 - j0 + 15) >> 4));      // of 16 slots: the products take no more
            wait(s_qk + b, i >> 1 & 1);
            tc_fence_after();
            float m = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (2 * c >= parts) break;
                float x[32];
                tc_ld32(x, mine + 32 * c);
                if (masked) {
#pragma unroll
                    for (int j = 0; j < 32; j++) if (!(sees[c] >> j & 1)) x[j] = -INFINITY;
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
            s_max[b][half][r] = m;
            asm volatile("bar.sync %0, 256;" :: "r"(1 + b) : "memory");
            m = fmaxf(m, s_max[b][half ^ 1][r]);
            const bool none = m == -INFINITY;
            m = none ? -INFINITY : m * f;                             // (-infinity times a factor of 0 is no number)
            const float2 ref = f2(none ? 14.f : 14.f - m), fc = f2(f);
            float2 l[2] = {f2(0.f), f2(0.f)};
            auto exps = [&](auto with_mask) {
#pragma unroll 1
                for (int c = 0; c < parts; c++) {
                    float x[16];
                    tc_ld16(x, mine + 16 * c);
                    uint32_t hl[16];                                  // upper parts of 16 slots, then lower parts
                    const uint32_t see = (c < 2 ? sees[0] : sees[1]) >> ((c & 1) * 16);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float2 y = f2_fma(make_float2(x[j], x[j + 1]), fc, ref);
                        float2 pr = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        if (decltype(with_mask)::value) {
                            if (!(see >> j & 1)) pr.x = 0.f;
                            if (!(see >> (j + 1) & 1)) pr.y = 0.f;
                        }
                        l[j >> 1 & 1] = f2_add(l[j >> 1 & 1], pr);
                        if constexpr (TWO) f2_split(pr, hl[j / 2], hl[8 + j / 2]);
                        else               hl[j / 2] = h2u(__floats2half2_rn(pr.x, pr.y));
                    }
                    if constexpr (TWO) tc_st16(mine + 16 * c, hl); else tc_put<8>(mine + 16 * c, hl);
                }
            };
            if (masked) exps(std::true_type()); else exps(std::false_type());
            float total = (l[0].x + l[0].y) + (l[1].x + l[1].y);
            if (masked) {
                const int slot = (2 * i + 1) % NS;
                wait(s_vok + (slot >> 1), (2 * i + 1) / NS & 1);
                if ((sees[0] & s_odd[slot >> 1][half * 2]) | (sees[1] & s_odd[slot >> 1][half * 2 + 1])) total = __int_as_float(0x7fc00000);
            }
            if (none && (sees[0] | sees[1])) total = __int_as_float(0x7fc00000);         // (every score that it sees is -infinity)
            if (i >= 2) wait(s_free + b, (i - 2) >> 1 & 1);           // the tile before has been drained: its sums are no more needed
            s_sum[b][half][r] = total;
            if (half == 0) s_top[b][r] = m;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_pfull + b);
        }
    } else {
        // ================================================================= sums out
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(PT_REGS_D));
        const int r = (warp & 3) * 32 + lane, d0 = warp >= 24 ? HD / 2 : 0;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_O + (uint32_t)d0;
        bool ok = true;
        if (lane == 0) mbar_arrive(s_pfull);                          // (no sums before the first tile's)
        for (int i = 0; i < n_tiles && ok; i++) {
            const int b = i & 1;
            ok = wait(s_pfull + b, i >> 1 & 1) && ok;
            const float m = s_top[b][r], now = fmaxf(top, m);
            const float was = top == now ? 1.f : exp2_approx(top - now), is = m == -INFINITY ? 0.f : exp2_approx(m - now);
            top = now;
            sum = fmaf(sum, was, (s_sum[b][0][r] + s_sum[b][1][r]) * is);
            ok = wait(s_pv + b, i >> 1 & 1) && ok;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 2; c += 16) {
                float v[16];
                tc_ld16(v, mine + c);
                if (c + 16 == HD / 2) {                               // the buffer goes back
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(s_free + b); mbar_arrive(s_pfull + (b ^ 1)); }
                }
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 o = f2_fma(make_float2(v[j], v[j + 1]), f2(is), f2_mul(make_float2(acc[c + j], acc[c + j + 1]), f2(was)));
                    acc[c + j] = o.x; acc[c + j + 1] = o.y;
                }
            }
        }
        if (r < t.n_rows) {
            const int row = t.first + r, of = p.by_group.of(row), h = hk * p.group + row - of * p.group;
            if (of >= p.c.n_ctx - s.pos) {                            // a token without a slot of its own
                top = -INFINITY; sum = 0.f;
#pragma unroll
                for (int j = 0; j < HD / 2; j++) acc[j] = 0.f;
            }
            if (!ok || s_dead) sum = __int_as_float(0x7fc00000);      // a wait ran out, here or in a warp that came to s_pfull all the same: no numbers instead of wrong ones
            if (w.n_splits > 1) {
                const size_t at = ((size_t)(w.item - p.whole) * p.n_splits + split) * PT_ROWS + r;
#pragma unroll
                for (int j = 0; j < HD / 2; j += 4) *reinterpret_cast<float4 *>(p.part + at * HD + d0 + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                if (d0 == 0) p.part_ml[at] = make_float2(top, sum);
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const size_t at = (size_t)(s.first + of) * p.out_stride + (size_t)h * HD + d0;
                if (p.xtype == PI_TYPE_F16) {
#pragma unroll
                    for (int j = 0; j < HD / 2; j += 8) {
                        uint4 u;
                        u.x = h2u(__floats2half2_rn(acc[j] * inv, acc[j + 1] * inv)); u.y = h2u(__floats2half2_rn(acc[j + 2] * inv, acc[j + 3] * inv));
                        u.z = h2u(__floats2half2_rn(acc[j + 4] * inv, acc[j + 5] * inv)); u.w = h2u(__floats2half2_rn(acc[j + 6] * inv, acc[j + 7] * inv));
                        *reinterpret_cast<uint4 *>((__half *)p.out + at + j) = u;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < HD / 2; j += 4) *reinterpret_cast<float4 *>((float *)p.out + at + j) = make_float4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tc_dealloc(s_tmem, 512);
}

// Clears the status word in front of the kernel: no CTA of its own can, as another one's wait may have run out by then.
__global__ void k_attn_paged_clear(unsigned int * status) {
    pdl_launch();
    pdl_wait();
    if (threadIdx.x == 0) *status = 0u;
}

bool attn_paged_tc_takes(int hd, int64_t rows) { return hd <= 128 && rows > 16; }

template <int HD, bool TWO>
static int pt_go(const AttnPagedP & a, cudaStream_t st) {
    constexpr int SUBS = (HD + 63) / 64;
    constexpr size_t smem = (size_t)(HD <= 64 ? 12 : 6) * SUBS * PT_SUB + 1024;
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
    PI_CUDA(launch_k(k_attn_paged_clear, dim3(1), dim3(32), 0, st, true, a.status));
    PI_CUDA(launch_k(k_attn_paged_tc<HD, TWO>, dim3(ap_grid(a)), dim3(PT_THREADS), smem, st, true, p));
    return PI_OK;
}

int launch_attn_paged_tc(const AttnPagedP & p, cudaStream_t st) {
    const bool half = p.xtype == PI_TYPE_F16;
    switch (p.c.hd) {
        case 64: return half ? pt_go<64, false>(p, st) : pt_go<64, true>(p, st);
        case 96: return half ? pt_go<96, false>(p, st) : pt_go<96, true>(p, st);
        default: return half ? pt_go<128, false>(p, st) : pt_go<128, true>(p, st);
    }
}

}  // namespace pi
