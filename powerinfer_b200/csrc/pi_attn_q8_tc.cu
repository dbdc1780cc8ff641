// Attention over the KV cache in 8 bits for many query rows of a KV head (prompts and chunks) on tcgen05; formulas and layouts of rows as in
// pi_attn_q8.cu.
//
// A CTA takes 128 query rows (the lanes) of one KV head and walks over its slots in tiles of 128.  Queries lie in tensor memory for the whole walk.
// A tile's codes, contiguous in the cache, come as one bulk copy each of keys and values, and go through registers into shared memory as halves (exact), both in
// the same layout: 128-byte rows of 64 halves, K-major for the scores, MN-major for the values.  Scores S = Q K^T are made into one of two buffers in tensor
// memory; the probabilities take their place, 32 slots a piece; sums of values O = P V of ONE tile go to a third buffer, which is
// drained and added with rounding in registers: the tensor cores cut FP32 sums at every step, so that no sum stays with them for longer than a tile.
// So every tile has its own maximum (no exchange between tiles; the two score buffers are two groups of warps' own): the drain joins tiles.
//
// Precision.  Probabilities, and queries of FP32 rows, as the sum of two halves each, i.e. two products in the place of one: 22 bits.  Queries of FP16 rows
// as they are.  (Probabilities of FP16 rows as one half: 7 % less time for 11 bits.)  Values' scales ride on the probabilities, over the power of two above the
// largest one that the row sees in the tile; probabilities are held times 2^14: 22 bits down to 2^-16 of that scale, an error of 2^-38 of it below.
//
// Measured: 1024 tokens over 4096 slots, 64 FP32 heads of 128 over 8 KV heads 255 us of the call's 270 (tensor pipe 51 % busy, issue slots 64 %); prompts of 701 to 421
// tokens, 128 FP16 heads of 64 329 us (19 %, 60 %).  A tile takes 1.9 us (64 dimensions: 1.4), a CTA 12 us (FP16 of 64: 5.5) besides, the last tile's way and the next CTA's start.
// Bound by the issue slots: 8 exponentials, splits and rounded sums a slot and four rows, halves of the codes, while products of 16 slots take 57 clocks each to issue.
//
// Warps: 0 issues the products; 1 asks for the codes; 4..11 and 12..19 have the even and the odd tiles' probabilities, a row and half of the slots a thread (the halves tell each other
// their maxima); 20..27 make the halves and drain the sums, a row and half of the columns a thread.
#include "pi_attn_q8.cuh"
#include "pi_tc.cuh"
#include "pi_tc_math.cuh"

#include <cfloat>
#include <type_traits>

namespace pi {

static constexpr int AT_THREADS = 896;
static constexpr int AT_REGS_M = 24, AT_REGS_S = 64, AT_REGS_D = 104;  // 24 + 4 x 64 + 2 x 104 of the 7 x 72 of the launch
static constexpr uint32_t AT_SUB = AT_KEYS * 128;                     // bytes of 64 columns of a tile
static constexpr int AT_RAW = 4;                                      // tiles of codes on their way: keys and values in turn

__device__ __forceinline__ void at_ld32(float (&v)[32], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                   "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]) : "r"(addr));
}

__device__ __forceinline__ void at_st8(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// TWO_Q: two halves for each query
template <int HD, bool TWO_Q>
__global__ void __launch_bounds__(AT_THREADS, 1) k_attn_q8_tc(const AttnQ8P p) {
    constexpr int KS = HD / 16, SUBS = HD / 64, U = HD / 32;          // steps of 16 columns; pieces of 64 columns; chunks of 16 codes of a tile a thread
    constexpr uint32_t TILE = SUBS * AT_SUB;
    constexpr uint32_t T_Q = 0, T_S = HD, T_O = HD + 2 * AT_KEYS;     // tensor memory: queries (upper, lower), two buffers of scores, sums
    static_assert(T_O + HD <= 512 && AT_REGS_M + 4 * AT_REGS_S + 2 * AT_REGS_D <= 7 * 72, "");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ uint64_t s_rfull[AT_RAW], s_rempty[AT_RAW];
    __shared__ uint64_t s_kfull[2], s_qk[2], s_pv[2], s_pfull[2], s_free[2], s_fin;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_dead;
    __shared__ float s_f[AT_ROWS];                                    // factor of a row's scores
    __shared__ float s_max[2][2][AT_ROWS], s_sum[2][2][AT_ROWS];       // of a tile's halves: maximum, sum of the probabilities
    __shared__ float s_top[2][AT_ROWS];                               // maximum of a tile
    __shared__ float s_ref[2][AT_ROWS];                               // power of two that its values' scales are held over
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t kbuf = (smem_u32(smem_raw) + 1023u) & ~1023u, vbuf = kbuf + 2 * TILE, raw = vbuf + 2 * TILE;
    const AqItem w = aq_item(p, blockIdx.x);
    const int split = w.split, hk = w.hk, rt = p.row_tiles - 1 - w.rt;      // (the longest rows first)
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, w.entry);
    const TileB t = aq_tile(p, s, rt, AT_ROWS);
    if (t.n_rows <= 0) return;
    const int k0 = split * p.split, k1 = split == w.n_splits - 1 ? t.seen : min(t.seen, k0 + p.split);
    if (k0 >= k1 && split > 0) return;                                // (split 0 answers for rows that see nothing)
    const int n_tiles = k0 < k1 ? (k1 - k0 + AT_KEYS - 1) / AT_KEYS : 0;
    const size_t head = (size_t)max(s.sq, 0) * p.c.H + hk;

    if (tid < 2) {
        mbar_init(s_kfull + tid, 8); mbar_init(s_qk + tid, 1); mbar_init(s_pv + tid, 1);
        mbar_init(s_pfull + tid, 16); mbar_init(s_free + tid, 8);
    }
    if (tid < AT_RAW) { mbar_init(s_rfull + tid, 1); mbar_init(s_rempty + tid, 8); }
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

    // ---- codes: keys and values in turn.  (Slots behind the cache are not read: their halves are of anything, and count nothing.)
    auto ask = [&](int i) {
        const int slot = i % AT_RAW, j0 = k0 + (i >> 1) * AT_KEYS;
        const unsigned bytes = (unsigned)min(AT_KEYS, p.c.n_ctx - j0) * HD;
        mbar_expect_tx(s_rfull + slot, bytes);
        bulk_g2s(smem_raw + (raw - smem_u32(smem_raw)) + (size_t)slot * AT_KEYS * HD, (i & 1 ? p.c.v : p.c.k) + (head * p.c.n_ctx + j0) * HD, bytes, s_rfull + slot);
    };
    if (warp == 1 && lane == 0) for (int i = 0; i < min(AT_RAW, 2 * n_tiles); i++) ask(i);
    // ---- the halves of a tile: a warp takes 8 rows x 64 columns, so that what it stores together meets all banks
    const int ct = tid - 640, cr = (ct >> 2) & 63, cc = ct & 3;       // row (of 64), piece of 16 columns of a thread
    const uint32_t from0 = (uint32_t)(cr * HD + cc * 16), to0 = (uint32_t)cr * 128u + (uint32_t)(((2 * cc) ^ (cr & 7)) * 16);
    auto put = [&](uint32_t from, uint32_t to) {
        uint4 c[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(c[u].x), "=r"(c[u].y), "=r"(c[u].z), "=r"(c[u].w) : "r"(from + from0 + (uint32_t)((u & 1) * 64 * HD + (u >> 1) * 64)) : "memory");
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t at = to + to0 + (uint32_t)(u >> 1) * AT_SUB + (uint32_t)(u & 1) * 8192u;
            const uint32_t w[4] = {c[u].x ^ 0x80808080u, c[u].y ^ 0x80808080u, c[u].z ^ 0x80808080u, c[u].w ^ 0x80808080u};
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at), "r"(q8_lo(w[0])), "r"(q8_hi(w[0])), "r"(q8_lo(w[1])), "r"(q8_hi(w[1])) : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(at ^ 16u), "r"(q8_lo(w[2])), "r"(q8_hi(w[2])), "r"(q8_lo(w[3])), "r"(q8_hi(w[3])) : "memory");
        }
    };

    // ---- queries into tensor memory.  Halves as they are: a row and a quarter of its columns a thread, straight from global memory.
    if constexpr (!TWO_Q) {
        if (warp >= 4 && warp < 20) {
            constexpr int NQ = HD / 4;
            const int part = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, row = t.first + r, tok = p.by_group.of(row);
            uint32_t u[16];
#pragma unroll
            for (int j = 0; j < 16; j++) u[j] = 0u;
            if (r < t.n_rows) {
                const uint4 * from = reinterpret_cast<const uint4 *>((const __half *)p.q + (size_t)(s.first + tok) * p.q_stride + (size_t)(hk * p.group + row - tok * p.group) * HD + part * NQ);
#pragma unroll
                for (int j = 0; j < NQ / 8; j++) { const uint4 v = __ldg(from + j); u[4 * j] = v.x; u[4 * j + 1] = v.y; u[4 * j + 2] = v.z; u[4 * j + 3] = v.w; }
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
            const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_Q + (uint32_t)(part * NQ / 2);
            if (NQ == 32) tc_st16(to, u); else at_st8(to, u);
            tc_wait_st();
        }
    } else {
        // FP32: whole rows to shared memory (the halves' place) as they lie, then a row and a quarter of its columns a thread, scaled and split
        constexpr int NQ = HD / 4, PITCH = HD + 4, LPR = HD / 4;      // lanes that read a row
        const bool mine = warp >= 4 && warp < 20;
        const int part = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
        float * rows = reinterpret_cast<float *>(smem_raw + (kbuf - smem_u32(smem_raw)));
        constexpr int RPW = 8, NL = RPW / (32 / LPR);                 // rows of a warp, all on their way at once
        if (warp < AT_ROWS / RPW) {
            const int r0 = warp * RPW;
            float4 u[NL];
#pragma unroll
            for (int k = 0; k < NL; k++) {
                const int q = r0 + k * (32 / LPR) + lane / LPR, row = t.first + q, tok = p.by_group.of(row);
                u[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (q < t.n_rows) u[k] = aq_query(p.xtype, p.q, (size_t)(s.first + tok) * p.q_stride + (size_t)(hk * p.group + row - tok * p.group) * HD + lane % LPR * 4);
            }
#pragma unroll
            for (int k = 0; k < NL; k++) *reinterpret_cast<float4 *>(rows + (r0 + k * (32 / LPR) + lane / LPR) * PITCH + lane % LPR * 4) = u[k];
        }
        __syncthreads();
        float4 v[NQ / 4];
        if (mine) {
            float m = 0.f;
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) v[j] = *reinterpret_cast<const float4 *>(rows + r * PITCH + part * NQ + j * 4);
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) m = fmaxf(fmaxf(m, fmaxf(fabsf(v[j].x), fabsf(v[j].y))), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
            s_max[part >> 1][part & 1][r] = m;
        }
        __syncthreads();
        if (mine) {
            const float m = fmaxf(fmaxf(s_max[0][0][r], s_max[0][1][r]), fmaxf(s_max[1][0][r], s_max[1][1][r]));
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127) - 10;     // the largest to 2^10 .. 2^11: lower parts are then exact to 2^-25
            const float up = copysignf(__uint_as_float((uint32_t)(127 - e) << 23), p.scale_log2);
            if (part == 0) s_f[r] = fabsf(p.scale_log2) * __uint_as_float((uint32_t)(127 + e) << 23);
            const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_Q + (uint32_t)(part * NQ / 2);
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int j = 0; j < NQ / 4; j++) {
                aq_split(v[j].x * up, v[j].y * up, hi[2 * j], lo[2 * j]);
                aq_split(v[j].z * up, v[j].w * up, hi[2 * j + 1], lo[2 * j + 1]);
            }
            if (NQ == 32) { tc_st16(to, hi); tc_st16(to + HD / 2, lo); }
            else          { at_st8(to, hi);  at_st8(to + HD / 2, lo); }
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
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(AT_REGS_M));
        if (warp == 0) {
            // ============================================================= products
            constexpr uint32_t idesc_v = tc_idesc(HD, true);
            const int tiles = __shfl_sync(0xffffffffu, n_tiles, 0), span = __shfl_sync(0xffffffffu, k1 - k0, 0);      // (uniform for the compiler)
            bool ok = true;
            auto scores = [&](int i) {
                const int b = i & 1, n = min(AT_KEYS, (span - i * AT_KEYS + 15) / 16 * 16);
                ok = wait(s_kfull + b, i >> 1 & 1) && ok;
                if (!ok) return;
                tc_fence_after();
                const uint32_t idesc = tc_idesc(n, false), d = tmem + T_S + (uint32_t)(b * AT_KEYS);
                const uint64_t k = tc_desc_k(kbuf + (uint32_t)b * TILE);
                if (TWO_Q) {
#pragma unroll
                    for (int j = 0; j < KS; j++) tc_mma_f16_ta(d, tmem + T_Q + HD / 2 + 8 * j, k + (j >> 2) * (AT_SUB >> 4) + 2 * (j & 3), idesc, j > 0);
                }
#pragma unroll
                for (int j = 0; j < KS; j++) tc_mma_f16_ta(d, tmem + T_Q + 8 * j, k + (j >> 2) * (AT_SUB >> 4) + 2 * (j & 3), idesc, TWO_Q || j > 0);
                tc_commit(s_qk + b);
            };
            if (tiles > 0) scores(0);
            if (tiles > 1) scores(1);
            for (int i = 0; i < tiles && ok; i++) {
                const int b = i & 1, steps = min(AT_KEYS / 16, (span - i * AT_KEYS + 15) / 16);
                ok = wait(s_pfull + b, i >> 1 & 1) && ok;             // the sums before are drained too, and the values of this tile there (a wait that is over costs 150 clocks)
                if (!ok) break;
                tc_fence_after();
                const uint32_t a = tmem + T_S + (uint32_t)(b * AT_KEYS), d = tmem + T_O;
                const uint64_t v = tc_desc_mn(vbuf + (uint32_t)b * TILE, AT_SUB);
                if (steps == AT_KEYS / 16) {
#pragma unroll
                    for (int j = 0; j < AT_KEYS / 16; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16 + 8), v + 128 * j, idesc_v, j > 0);
#pragma unroll
                    for (int j = 0; j < AT_KEYS / 16; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16), v + 128 * j, idesc_v, true);
                } else {
                    for (int j = 0; j < steps; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16 + 8), v + 128 * j, idesc_v, j > 0);
                    for (int j = 0; j < steps; j++) tc_mma_f16_ta(d, a + (uint32_t)(j * 16), v + 128 * j, idesc_v, true);
                }
                tc_commit(s_pv + b);
                if (i + 2 < tiles) scores(i + 2);
            }
            tc_commit(&s_fin);                                        // nothing is in flight when tensor memory is given back
            for (int spins = 0; spins < (1 << 20) && !mbar_try_wait(&s_fin, 0u); spins++) {}
            __syncwarp();
        } else if (warp == 1) {
            // ============================================================= codes
            int i = min(AT_RAW, 2 * n_tiles);
            for (; i < 2 * n_tiles; i++) {
                const int slot = i % AT_RAW;
                if (!wait(s_rempty + slot, i / AT_RAW & 1 ^ 1)) break;
                if (lane == 0) ask(i);
                __syncwarp();
            }
            if (lane == 0) ring_land(s_rfull, i, AT_RAW);
            __syncwarp();
        }
    } else if (warp < 20) {
        // ================================================================= probabilities
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(AT_REGS_S));
        const int b = (warp - 4) >> 3, half = (warp - 4) >> 2 & 1, r = (warp & 3) * 32 + lane;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_S + (uint32_t)(b * AT_KEYS + half * 64);
        const float * ks = p.c.ks + head * (p.c.n_ctx >> p.c.shift), * vs = p.c.vs + head * (p.c.n_ctx >> p.c.shift);
        const bool there = r < t.n_rows;
        const int sees = there ? aq_sees(s, p.c.n_ctx, p.by_group.of(t.first + r)) : 0;
        const int least = __reduce_min_sync(0xffffffffu, there ? sees : 0x7fffffff);
        const float f = s_f[r];
        auto scales = [&](int i, float & k, float & v) {              // lane j: those of the 16 slots j of the tile (0 behind the range)
            const int j = k0 + i * AT_KEYS + (lane & 7) * 16;
            k = v = 0.f;
            if (j < k1) { k = __ldg(ks + (j >> p.c.shift)); v = __ldg(vs + (j >> p.c.shift)); }
        };
        float sk, sv;
        if (b < n_tiles) scales(b, sk, sv);
        for (int i = b; i < n_tiles; i += 2) {                        // (to the end whatever waits ran out: the halves meet at a barrier)
            const int left = sees - (k0 + i * AT_KEYS + half * 64);   // slots of this half that the row sees
            const float wv = sv, wk = sk, finite = fabsf(sv) <= FLT_MAX ? sv : 0.f;
            float largest = finite;                                   // of the finite ones that the row sees (what others see has no say in it)
            if (k0 + i * AT_KEYS + AT_KEYS > least) {                 // (decided by all eight pieces: the same in both halves)
                largest = 0.f;
#pragma unroll
                for (int c = 0; c < 8; c++) { const float v = __shfl_sync(0xffffffffu, finite, c); if (k0 + i * AT_KEYS + c * 16 < sees) largest = fmaxf(largest, v); }
            } else {
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            }
            // 2^14 over the power of two above it (exact; clamped where that is no normal number)
            const int e = min(max((int)(__float_as_uint(largest) >> 23), 14), 253);
            const float up = __uint_as_float((uint32_t)(267 - e) << 23);
            float fk[4];
#pragma unroll
            for (int c = 0; c < 4; c++) fk[c] = f * __shfl_sync(0xffffffffu, wk, half * 4 + c);
            if (i + 2 < n_tiles) scales(i + 2, sk, sv);
            const bool masked = k0 + i * AT_KEYS + half * 64 + 64 > least;       // (of this warp's rows)
            const int parts = max(0, min(4, (k1 - k0 - i * AT_KEYS - half * 64 + 15) >> 4));      // of 16 slots: the products take no more
            wait(s_qk + b, i >> 1 & 1);
            tc_fence_after();
            float m = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                if (2 * c >= parts) break;
                float x[32];
                at_ld32(x, mine + 32 * c);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float * y = x + h * 16;
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 16; j++) if (c * 32 + h * 16 + j >= left) y[j] = -INFINITY;
                    }
                    float a = max3(y[0], y[1], y[2]), e = max3(y[3], y[4], y[5]);
#pragma unroll
                    for (int j = 6; j < 14; j += 4) { a = max3(a, y[j], y[j + 1]); e = max3(e, y[j + 2], y[j + 3]); }
                    a = fmaxf(max3(a, y[14], y[15]), e);
                    if (a > -INFINITY) m = fmaxf(m, a * fk[2 * c + h]);      // (-infinity times a factor of 0 is no number)
                }
            }
            s_max[b][half][r] = m;
            asm volatile("bar.sync %0, 256;" :: "r"(1 + b) : "memory");
            m = fmaxf(m, s_max[b][half ^ 1][r]);
            const float2 ref = f2(m == -INFINITY ? 0.f : -m);
            float2 l[2] = {f2(0.f), f2(0.f)};
            auto exps = [&](auto with_mask) {
#pragma unroll 1
                for (int c = 0; c < parts; c++) {
                    float x[16];
                    tc_ld16(x, mine + 16 * c);
                    uint32_t hl[16];                                  // upper parts of 16 slots, then lower parts
                    const float2 fc = f2(c == 0 ? fk[0] : c == 1 ? fk[1] : c == 2 ? fk[2] : fk[3]), pv = f2(__shfl_sync(0xffffffffu, wv, half * 4 + c) * up);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float2 y = f2_fma(make_float2(x[j], x[j + 1]), fc, ref);
                        float2 pr = make_float2(exp2_approx(y.x), exp2_approx(y.y)), w = f2_mul(pr, pv);
                        if (decltype(with_mask)::value) {             // (a masked slot counts nothing whatever its scores and its block's scales are)
                            if (c * 16 + j >= left) pr.x = w.x = 0.f;
                            if (c * 16 + j + 1 >= left) pr.y = w.y = 0.f;
                        }
                        l[j >> 1 & 1] = f2_add(l[j >> 1 & 1], pr);
                        f2_split(w, hl[j / 2], hl[8 + j / 2]);
                    }
                    tc_st16(mine + 16 * c, hl);
                }
            };
            if (masked) exps(std::true_type()); else exps(std::false_type());
            if (i >= 2) wait(s_free + b, (i - 2) >> 1 & 1);           // the tile before has been drained: its sums are no more needed
            s_sum[b][half][r] = (l[0].x + l[0].y) + (l[1].x + l[1].y);
            if (half == 0) { s_top[b][r] = m; s_ref[b][r] = __uint_as_float((254u << 23) - __float_as_uint(up)); }      // (1 / up)
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_pfull + b);
        }
    } else {
        // ================================================================= tiles in, sums out
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(AT_REGS_D));
        const int r = (warp & 3) * 32 + lane, d0 = warp >= 24 ? HD / 2 : 0;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + T_O + (uint32_t)d0;
        bool ok = true;
        auto drain = [&](int i) {
            const int b = i & 1;
            ok = wait(s_pfull + b, i >> 1 & 1) && ok;
            const float m = s_top[b][r], now = fmaxf(top, m);
            const float was = top == now ? 1.f : exp2_approx(top - now), is = m == -INFINITY ? 0.f : exp2_approx(m - now);
            top = now;
            sum = fmaf(sum, was, (s_sum[b][0][r] + s_sum[b][1][r]) * is);
            const float k = is * s_ref[b][r];
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
                    const float2 o = f2_fma(make_float2(v[j], v[j + 1]), f2(k), f2_mul(make_float2(acc[c + j], acc[c + j + 1]), f2(was)));
                    acc[c + j] = o.x; acc[c + j + 1] = o.y;
                }
            }
        };
        auto take = [&](int n, uint32_t to) {                         // the n-th tile of codes
            const int slot = n % AT_RAW;
            ok = wait(s_rfull + slot, n / AT_RAW & 1) && ok;
            put(raw + (uint32_t)(slot * AT_KEYS * HD), to);
            tc_fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_rempty + slot);
        };
        for (int i = 0; i < n_tiles && ok; i++) {
            const int b = i & 1;
            if (i >= 2) ok = wait(s_qk + b, (i - 2) >> 1 & 1) && ok;
            take(2 * i, kbuf + (uint32_t)b * TILE);
            if (lane == 0) mbar_arrive(s_kfull + b);
            if (i >= 2) drain(i - 2);                                 // (which waits for the value products of tile i - 2: their buffer is free)
            take(2 * i + 1, vbuf + (uint32_t)b * TILE);
            if (i == 0 && lane == 0) mbar_arrive(s_pfull);            // (whoever drains tile i - 1 later has put the values of tile i there before)
        }
        for (int i = max(0, n_tiles - 2); i < n_tiles && ok; i++) drain(i);

        if (r < t.n_rows) {
            const int row = t.first + r, of = p.by_group.of(row), tok = s.first + of, h = hk * p.group + row - of * p.group;
            if (!ok || s_dead) sum = __int_as_float(0x7fc00000);      // a wait ran out, here or in a warp that came to s_pfull all the same: no numbers instead of wrong ones
            if (w.n_splits > 1) {
                const size_t at = ((size_t)(w.item - p.whole) * p.n_splits + split) * AT_ROWS + r;
#pragma unroll
                for (int j = 0; j < HD / 2; j += 4) *reinterpret_cast<float4 *>(p.part + at * HD + d0 + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                if (d0 == 0) p.part_ml[at] = make_float2(top, sum);
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const size_t at = (size_t)tok * p.out_stride + (size_t)h * HD + d0;
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
                if (d0 == 0 && p.lse) p.lse[(size_t)tok * p.n_head + h] = sum == 0.f ? INFINITY : top + log2f(sum);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tc_dealloc(s_tmem, 512);
}

// Clears the status word in front of the kernel: no CTA of its own can, as another one's wait may have run out by then.  (A copy of zeros instead took 4.5 us a call.)
__global__ void k_attn_q8_clear(unsigned int * status) {
    pdl_launch();
    pdl_wait();
    if (threadIdx.x == 0) *status = 0u;
}

// Both sides measured (us, here and with mma.sync; head_dim 128, F32, 4 query heads a KV head, 4096 slots): 8 sequences of 8 KV heads 24 rows 50 and 48, 64 rows 52 and 82, 128
// rows 58 and 156; one sequence 28 and 18, 128 rows 35 and 28, 256 rows 26 and 48.  (It gains from fewer rows on where there are many items, from more where they are few.)
bool attn_q8_tc_takes(int hd, int64_t rows) { return (hd == 64 || hd == 128) && rows >= 64; }

template <int HD, bool TWO_Q>
static int at_go(const AttnQ8P & p, cudaStream_t st) {
    constexpr size_t smem = (size_t)4 * (HD / 64) * AT_SUB + AT_RAW * AT_KEYS * HD + 1024;
    static bool done[16] = {false};
    int dev = 0;
    PI_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_attn_q8_tc<HD, TWO_Q>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PI_CUDA(launch_k(k_attn_q8_clear, dim3(1), dim3(32), 0, st, true, p.status));
    PI_CUDA(launch_k(k_attn_q8_tc<HD, TWO_Q>, dim3(aq_grid(p)), dim3(AT_THREADS), smem, st, true, p));
    return PI_OK;
}

int launch_attn_q8_tc(const AttnQ8P & p, cudaStream_t st) {
    if (p.c.hd == 64) return p.xtype == PI_TYPE_F16 ? at_go<64, false>(p, st) : at_go<64, true>(p, st);
    return p.xtype == PI_TYPE_F16 ? at_go<128, false>(p, st) : at_go<128, true>(p, st);
}

}  // namespace pi
