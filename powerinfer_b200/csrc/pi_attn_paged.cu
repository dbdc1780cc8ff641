// Attention over a paged cache for a ragged batch of trees of drafted tokens: token t of entry i sees the slots before pos0[i], and of the entry's new ones those
// that its mask names (or those up to its own).
//
//     s_j = scale * (q . k_j)     p_j = exp(s_j - max s)     out = sum_j p_j v_j / sum_j p_j     over the slots j that the token sees
//
// For up to 16 query rows of a KV head (the query heads of a group, of one or more tokens); more go to pi_attn_paged_tc.cu where that is faster.
// Bound by the bytes of keys and values: 32 sequences of 1024 to 2048 slots, 32 KV heads of 128, 814 MB: 122 us, 6.7 TB/s (a copy makes 6.5); a call of 77 slots 3 us, the launch.
// A CTA takes the rows of one KV head and a range of slots; its four warps take 16 slots each in turn, a part of one page, copied ahead into a ring of their own (cp.async; no barrier
// between warps), keep a maximum, a sum and all sums of values of their own, and join them at the end.  Long ranges are split over CTAs, whose sums k_attn_paged_join joins.
//
// Precision.  Queries of FP32 rows, over a power of two of their row's largest value, and probabilities are the sum of two halves each, 22 bits, i.e. two products in the place
// of one (the bytes bound it all the same); queries of FP16 rows are halves as they are.  Probabilities are held times 2^8: their steps end 2^-32 below the largest one.  Maxima, sums and
// the exponents' arguments are FP32; sums of values are added with rounding, as the tensor cores cut theirs (FP16 rows' over 2048 steps were 2^-12 too small).
//
// What a row does not see: scores are set to -infinity by the mask's bits, whatever the keys are; slots behind the entry's last and pages that are not there come as zeros; and where a step that not
// every row sees whole holds a value that is not finite, its slots are added one by one to the rows that see them.
//
// Layouts.  A slot's row has 16-byte pieces permuted by its number, so that ldmatrix meets all banks.  The probabilities of the score tile's layout are the value product's
// operand as they stand.  Where the maximum rises by less than 2^7, sums are not scaled anew.
#include "pi_attn_paged.cuh"

#include <cfloat>

namespace pi {

static constexpr int PA_WARPS = 4, PA_THREADS = PA_WARPS * 32, PA_STEP = PA_WARPS * 16;
static constexpr float PA_RISE = 7.f, PA_P = 256.f;                   // bits a maximum may lag; probabilities are held times this (2^7 * 256 < 65504)

template <int HD> struct PaShape {
    static constexpr int KS = HD / 16, NT = HD / 8, PIECES = HD / 8;  // steps of 16 columns, tiles of 8 columns, 16-byte pieces of a row
    static __device__ __forceinline__ uint32_t at(int row, int piece) {
        return (uint32_t)(row * PIECES + (HD % 64 == 0 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3))) * 16u;
    }
    static constexpr int STAGES = HD <= 96 ? 4 : 3, STAGE = 2 * 16 * HD * 2;
    static constexpr int CTAS = HD == 64 ? 3 : HD <= 128 ? 2 : 1;     // that an SM holds
    static constexpr size_t RING = (size_t)PA_WARPS * STAGES * STAGE, JOIN = (size_t)PA_WARPS * 16 * (HD + 4) * 4, QUERIES = 2 * 16 * (2 * HD + 16);
    static constexpr size_t SMEM = (RING > JOIN ? RING : JOIN) + QUERIES;
};

// R rows in shared memory as halves [upper, lower][row][HD + 8], and the factors of their scores
template <int HD, bool TWO, int R> struct PaQueries {
    static constexpr int TPR = PA_THREADS / R, W = HD / 4, N = (W + TPR - 1) / TPR, PITCH = 2 * HD + 16;
    float4 x[N];
    __device__ __forceinline__ void load(const AttnPagedP & p, const SeqB & s, const TileP & t, int hk) {
        const int r = threadIdx.x / TPR, j = threadIdx.x % TPR, row = t.first + r, tok = p.by_group.of(row);
        const size_t at = r < t.n_rows ? (size_t)(s.first + tok) * p.q_stride + (size_t)(hk * p.group + row - tok * p.group) * HD : 0;
#pragma unroll
        for (int u = 0; u < N; u++) {
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < t.n_rows && j + u * TPR < W) x[u] = aq_query(p.xtype, p.q, at + (j + u * TPR) * 4);
        }
    }
    __device__ __forceinline__ void put(const AttnPagedP & p, unsigned char * to, float * factor) {
        const int r = threadIdx.x / TPR, j = threadIdx.x % TPR;
        float m = 0.f, zero = 0.f;                                    // zero: no more 0 where a value is not finite
#pragma unroll
        for (int u = 0; u < N; u++) {
            m = fmaxf(fmaxf(m, fmaxf(fabsf(x[u].x), fabsf(x[u].y))), fmaxf(fabsf(x[u].z), fabsf(x[u].w)));
            zero = fmaf(x[u].x, 0.f, fmaf(x[u].y, 0.f, fmaf(x[u].z, 0.f, fmaf(x[u].w, 0.f, zero))));
        }
        if (zero != 0.f) m = INFINITY;
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // two halves: the largest to 2^10 .. 2^11, a value is then off by 2^-22 of itself, or by 2^-25 (lower parts have no steps below 2^-24)
        const int e = TWO ? min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127) - 10 : 0;
        const float up = __uint_as_float((uint32_t)(127 - e) << 23), down = m < INFINITY ? __uint_as_float((uint32_t)(127 + e) << 23) : __int_as_float(0x7fc00000);
        if (j == 0) factor[r] = down * p.scale_log2;
#pragma unroll
        for (int u = 0; u < N; u++) {
            uint2 hi, lo;
            aq_split(x[u].x * up, x[u].y * up, hi.x, lo.x);
            aq_split(x[u].z * up, x[u].w * up, hi.y, lo.y);
            if (j + u * TPR >= W) break;
            *reinterpret_cast<uint2 *>(to + r * PITCH + (j + u * TPR) * 8) = hi;
            if (TWO || R == 8) *reinterpret_cast<uint2 *>(to + (R + r) * PITCH + (j + u * TPR) * 8) = lo;      // (of FP16 rows 0)
        }
    }
};

// TWO: two halves for queries (FP32 rows).  R: 16 rows, or 8: then rows 0 .. 7 of the products' operands are the upper and rows 8 .. 15 the lower halves of queries and of probabilities, one product in the
// place of two (FP32, 64 heads over 8 of 128: 8 sequences of 8000 slots 44 us with two products, 37 so; one of 32768 35 and 32).
template <int HD, bool TWO, int R>
__global__ void __launch_bounds__(PA_THREADS, PaShape<HD>::CTAS) k_attn_paged(const AttnPagedP p) {
    using S = PaShape<HD>;
    using Q = PaQueries<HD, TWO, R>;
    constexpr int ST = S::STAGES, NH = R / 8, NO = 2 * NH;            // rows and sums of a lane
    constexpr bool PACK = R == 8, Q_REGS = PACK || HD <= 128;         // queries stay in registers
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_m[PA_WARPS][R], s_l[PA_WARPS][R], s_f[R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const AqItem wk = ap_item(p, blockIdx.x);
    const int split = wk.split, hk = wk.hk;
    pdl_launch();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.status) *p.status = 0u;          // (no wait of this kernel runs out)
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, wk.entry);
    const TileP t = ap_tile(p, s, wk.rt, R);
    if (t.n_rows <= 0) return;
    const int k0 = split * p.split, k1 = split == wk.n_splits - 1 ? t.seen : min(t.seen, k0 + p.split);
    if (k0 >= k1 && split > 0) return;                                // (split 0 answers for rows that see nothing)
    unsigned char * queries = smem + (S::SMEM - S::QUERIES);
    Q qs;
    qs.load(p, s, t, hk);
    const __half * kc = p.c.k + page_at(p.c, 0, hk), * vc = p.c.v + page_at(p.c, 0, hk);
    const size_t of_page = page_at(p.c, 1, 0);                        // halves from page to page
    const int first = k0 + warp * 16, steps = first < k1 ? (k1 - first + PA_STEP - 1) / PA_STEP : 0;
    const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * ST * S::STAGE);
    // pages of the next 32 steps, one a lane, and of the 32 behind them
    auto pages = [&](int it) { const int j = first + (it + lane) * PA_STEP; return j < k1 ? page_of(p.c, s.sq, j >> p.c.shift) : -1; };
    int page_now = steps ? pages(0) : -1, page_then = steps > 32 ? pages(32) : -1;
    uint32_t valid = 0;                                               // bit it & 31: step `it`'s page is there
    int asked = 0;
    auto issue = [&]() {
        if (asked < steps) {
            if (asked > 0 && (asked & 31) == 0) { page_now = page_then; page_then = asked + 32 < steps ? pages(asked + 32) : -1; }
            const int page = __shfl_sync(0xffffffffu, page_now, asked & 31), j0 = first + asked * PA_STEP;
            valid = page >= 0 ? valid | 1u << (asked & 31) : valid & ~(1u << (asked & 31));
            if (page >= 0) {
                const size_t at = (size_t)page * of_page + (size_t)(j0 & (p.c.page - 1)) * HD;
                const uint32_t fill = ring + (uint32_t)(asked % ST) * S::STAGE;
#pragma unroll
                for (int u = 0; u < HD / 16; u++) {
                    const int e = u * 32 + lane, row = e / S::PIECES, piece = e - row * S::PIECES, bytes = j0 + row < t.there ? 16 : 0;      // (behind the entry's slots: zeros)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(fill + S::at(row, piece)), "l"(kc + at + e * 8), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(fill + 16 * HD * 2 + S::at(row, piece)), "l"(vc + at + e * 8), "r"(bytes) : "memory");
                }
            }
            asked++;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int it = 0; it < ST - 1; it++) issue();

    qs.put(p, queries, s_f);
    __syncthreads();
    float f[NH], m[NH], l[NH]; int tok[NH]; bool any[NH];             // of rows g and g + 8
#pragma unroll
    for (int h = 0; h < NH; h++) {
        const int r = g + 8 * h;
        tok[h] = r < t.n_rows ? p.by_group.of(t.first + r) : 0x7fffffff;
        f[h] = s_f[r]; m[h] = -INFINITY; l[h] = 0.f; any[h] = false;
    }
    // ldmatrix: a lane names a row of one of four 8 x 8 pieces
    const uint32_t q_at = smem_u32(queries) + (uint32_t)((lane & 15) * Q::PITCH + (lane >> 4) * 16);
    uint32_t a[Q_REGS ? S::KS : 1][4], a_low[Q_REGS && TWO && !PACK ? S::KS : 1][4];
    if constexpr (Q_REGS) {
#pragma unroll
        for (int k = 0; k < S::KS; k++) {
            ldsm4(a[k], q_at + k * 32);
            if constexpr (TWO && !PACK) ldsm4(a_low[k], q_at + R * Q::PITCH + k * 32);
        }
    }
    float o[S::NT][NO];
#pragma unroll
    for (int n = 0; n < S::NT; n++)
#pragma unroll
        for (int j = 0; j < NO; j++) o[n][j] = 0.f;
    const int k_row = (lane & 7) + (lane >> 4) * 8, k_piece = lane >> 3 & 1, v_row = lane & 15, v_piece = lane >> 4;

    for (int it = 0; it < steps; it++) {
        asm volatile("cp.async.wait_group %0;" :: "n"(ST - 2) : "memory");
        __syncwarp();                                                 // the stage is there for all lanes, and all have read the last one
        const bool there = valid >> (it & 31) & 1;
        issue();                                                      // (into which this goes)
        if (!there) continue;                                         // nobody sees the slots of a page that is not there
        const uint32_t kt = ring + (uint32_t)(it % ST) * S::STAGE, vt = kt + 16 * HD * 2;
        const int j0 = first + it * PA_STEP;
        const bool masked = j0 + 16 > s.pos;                          // not wholly of the context, which every row sees
        // ---- scores of 16 slots
        // (the tensor cores cut sums at every step: lower parts have sums of their own, whose steps are small)
        float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, low[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < S::KS; k++) {
            uint32_t b[4];
            ldsm4(b, kt + S::at(k_row, 2 * k + k_piece));
            if constexpr (Q_REGS) {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    if constexpr (TWO && !PACK) mma16816(low[n], a_low[k][0], a_low[k][1], a_low[k][2], a_low[k][3], b[2 * n], b[2 * n + 1]);
                    mma16816(x[n], a[k][0], a[k][1], a[k][2], a[k][3], b[2 * n], b[2 * n + 1]);
                }
            } else {
                uint32_t w[4];
                if constexpr (TWO) {
                    ldsm4(w, q_at + R * Q::PITCH + k * 32);
#pragma unroll
                    for (int n = 0; n < 2; n++) mma16816(low[n], w[0], w[1], w[2], w[3], b[2 * n], b[2 * n + 1]);
                }
                ldsm4(w, q_at + k * 32);
#pragma unroll
                for (int n = 0; n < 2; n++) mma16816(x[n], w[0], w[1], w[2], w[3], b[2 * n], b[2 * n + 1]);
            }
        }
        // ---- probabilities, as A operands of the value products
        uint32_t sees[NH];
#pragma unroll
        for (int h = 0; h < NH; h++) sees[h] = 0xffffu;
        if (masked) {
#pragma unroll
            for (int h = 0; h < NH; h++) sees[h] = ap_sees(p, s, tok[h], j0 - s.pos) & 0xffffu;
        }
        uint32_t pa[4], pl[4];
        float alpha[NH];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < NH; h++) {
            alpha[h] = 1.f;
            any[h] |= sees[h] != 0;
            float y[2][2];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    y[n][j] = (PACK ? x[n][j] + x[n][2 + j] : TWO ? x[n][2 * h + j] + low[n][2 * h + j] : x[n][2 * h + j]) * f[h];
                    if (masked && !(sees[h] >> (n * 8 + 2 * q + j) & 1)) y[n][j] = -INFINITY;
                }
            float top = fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[1][0], y[1][1]));
            if (__any_sync(0xffffffffu, top > m[h] + PA_RISE)) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float now = fmaxf(m[h], top);
                alpha[h] = now == m[h] ? 1.f : exp2_approx(m[h] - now);
                m[h] = now;
                l[h] *= alpha[h];
                moved = true;
            }
            const float ref = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float p0 = exp2_approx(y[n][0] - ref), p1 = exp2_approx(y[n][1] - ref);
                l[h] += p0 + p1;
                if constexpr (PACK) aq_split(p0 * PA_P, p1 * PA_P, pa[2 * n], pa[2 * n + 1]);
                else                aq_split(p0 * PA_P, p1 * PA_P, pa[2 * n + h], pl[2 * n + h]);
            }
        }
        if (moved && it > 0) {
#pragma unroll
            for (int n = 0; n < S::NT; n++)
#pragma unroll
                for (int j = 0; j < NO; j++) o[n][j] *= alpha[j >> 1];
        }
        // ---- values
        bool odd = false;                                             // a value that is not finite, where not every row sees every slot
        if (masked) {
            __half2 zero = __floats2half2_rn(0.f, 0.f);
            const __half2 none = zero;
#pragma unroll
            for (int u = 0; u < HD / 16; u++) {
                uint4 w;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(vt + (uint32_t)(u * 32 + lane) * 16u) : "memory");
                const __half2 * v = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
                for (int j = 0; j < 4; j++) zero = __hfma2(v[j], none, zero);
            }
            odd = __any_sync(0xffffffffu, !__hbeq2(zero, none));
        }
        if (!odd) {
#pragma unroll
            for (int n = 0; n < S::NT; n += 2) {
                uint32_t b[4];
                ldsm4_t(b, vt + S::at(v_row, n + v_piece));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (PACK) {
                        float w[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816(w, pa[0], pa[1], pa[2], pa[3], b[2 * h], b[2 * h + 1]);
                        o[n + h][0] += w[0] + w[2]; o[n + h][1] += w[1] + w[3];
                    } else {                                          // (the tensor cores cut FP32 sums: they are added with rounding)
                        float w[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816(w, pl[0], pl[1], pl[2], pl[3], b[2 * h], b[2 * h + 1]);
                        mma16816(w, pa[0], pa[1], pa[2], pa[3], b[2 * h], b[2 * h + 1]);
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n + h][e] += w[e];
                    }
                }
            }
        } else {
            // slot by slot: the products of one slot's value and all rows' probabilities, kept by the rows that see it.  (Lower parts of probabilities would make no number of an infinity
            // times 0: they count where the value is finite.)
#pragma unroll 1
            for (int j = 0; j < 16; j++) {
                const bool mine = (j >> 1 & 3) == q;                  // this lane's slots are 2q, 2q + 1, 8 + 2q, 9 + 2q
                const uint32_t keep = mine ? (j & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
                const uint32_t lo8 = j < 8 ? keep : 0u, hi8 = j < 8 ? 0u : keep;
                const bool see0 = sees[0] >> j & 1, see1 = sees[NH - 1] >> j & 1;
#pragma unroll
                for (int n = 0; n < S::NT; n += 2) {
                    uint32_t b[4];
                    ldsm4_t(b, vt + S::at(v_row, n + v_piece));
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t b0 = b[2 * h] & lo8, b1 = b[2 * h + 1] & hi8;
                        float w[4] = {0.f, 0.f, 0.f, 0.f}, wl[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816(w, pa[0], pa[1], pa[2], pa[3], b0, b1);
                        if constexpr (!PACK) mma16816(wl, pl[0], pl[1], pl[2], pl[3], b0, b1);
                        else                 { wl[0] = w[2]; wl[1] = w[3]; }
#pragma unroll
                        for (int e = 0; e < NO; e++)
                            if (e < 2 ? see0 : see1) o[n + h][e] += fabsf(w[e]) <= FLT_MAX ? w[e] + wl[e] : w[e];
                    }
                }
            }
        }
    }

    // ---- the four warps' sums together
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    constexpr int PITCH = HD + 4;
    float * so = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int h = 0; h < NH; h++) {
        float sum = l[h];
        if (any[h] && m[h] == -INFINITY) sum = __int_as_float(0x7fc00000);         // (every score that it sees is -infinity: no number)
        const bool none = tok[h] >= p.c.n_ctx - s.pos;                // a token without a slot of its own
        if (none) { m[h] = -INFINITY; sum = 0.f; }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int r = g + 8 * h;
        if (q == 0) { s_m[warp][r] = m[h]; s_l[warp][r] = sum; }
        float * row = so + (size_t)(warp * R + r) * PITCH + 2 * q;
#pragma unroll
        for (int n = 0; n < S::NT; n++) *reinterpret_cast<float2 *>(row + n * 8) = none ? make_float2(0.f, 0.f) : make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    __syncthreads();
    const size_t part0 = ((size_t)(wk.item - p.whole) * p.n_splits + split) * R;
    for (int e = threadIdx.x; e < t.n_rows * (HD / 4); e += PA_THREADS) {
        const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
        float top = s_m[0][r];
#pragma unroll
        for (int w = 1; w < PA_WARPS; w++) top = fmaxf(top, s_m[w][r]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f; float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < PA_WARPS; w++) {
            const float is = exp2_approx(s_m[w][r] - ref), k = is * (1.f / PA_P);
            const float4 u = *reinterpret_cast<const float4 *>(so + (size_t)(w * R + r) * PITCH + d);
            sum = fmaf(is, s_l[w][r], sum);
            v.x = fmaf(k, u.x, v.x); v.y = fmaf(k, u.y, v.y); v.z = fmaf(k, u.z, v.z); v.w = fmaf(k, u.w, v.w);
        }
        if (wk.n_splits > 1) {
            *reinterpret_cast<float4 *>(p.part + (part0 + r) * HD + d) = v;
            if (d == 0) p.part_ml[part0 + r] = make_float2(top, sum);
        } else {
            const int row = t.first + r, of = p.by_group.of(row), h = hk * p.group + row - of * p.group;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const size_t at = (size_t)(s.first + of) * p.out_stride + (size_t)h * HD + d;
            if (p.xtype == PI_TYPE_F16) *reinterpret_cast<uint2 *>((__half *)p.out + at) = make_uint2(h2u(__floats2half2_rn(v.x * inv, v.y * inv)), h2u(__floats2half2_rn(v.z * inv, v.w * inv)));
            else                        *reinterpret_cast<float4 *>((float *)p.out + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        }
    }
}

// The parts of a tile joined, in their order.  A warp has a row: a lane finds the weight of one part, then all parts' sums come with PJ_AT of them on their way at once.
static constexpr int PJ_WARPS = 8, PJ_AT = 4;

template <int HD>
__global__ void __launch_bounds__(PJ_WARPS * 32) k_attn_paged_join(const AttnPagedP p, int R) {
    constexpr int W = HD % 128 == 0 ? 4 : HD % 64 == 0 ? 2 : 1, N = HD / (32 * W);       // values of a lane side by side, and how often
    const int lane = threadIdx.x & 31, at = blockIdx.x * PJ_WARPS + (threadIdx.x >> 5), k = at / R, r = at - k * R, item = p.whole + k;
    pdl_launch();
    pdl_wait();
    if (item >= p.items) return;
    const size_t first = (size_t)k * p.n_splits * R + r;
    // (before it is known how many parts there are: what lies behind the last one is read, and counts nothing)
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < p.n_splits) ml = __ldcg(&p.part_ml[first + (size_t)lane * R]);
    float u[PJ_AT][N * W];
    auto load = [&](int i0, int last) {
#pragma unroll
        for (int c = 0; c < PJ_AT; c++) {
            const float * from = p.part + (first + (size_t)min(i0 + c, last) * R) * HD + lane * W;
#pragma unroll
            for (int j = 0; j < N; j++) {
                if constexpr (W == 4)      { const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + j * 128)); u[c][4 * j] = x.x; u[c][4 * j + 1] = x.y; u[c][4 * j + 2] = x.z; u[c][4 * j + 3] = x.w; }
                else if constexpr (W == 2) { const float2 x = __ldcg(reinterpret_cast<const float2 *>(from + j * 64)); u[c][2 * j] = x.x; u[c][2 * j + 1] = x.y; }
                else                       u[c][j] = __ldcg(from + j * 32);
            }
        }
    };
    load(0, p.n_splits - 1);
    const int of_head = p.by_tiles.of(item), nt = item - of_head * p.row_tiles, rt = R == PT_ROWS ? p.row_tiles - 1 - nt : nt, entry = p.by_heads.of(of_head), hk = of_head - entry * p.c.H;
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, entry);
    const TileP t = ap_tile(p, s, rt, R);
    if (r >= t.n_rows) return;
    const int n = max(1, min(p.n_splits, (t.seen + p.split - 1) / p.split));       // parts that were written
    float top = lane < n ? ml.x : -INFINITY, sum = 0.f, v[N * W];
    for (int i = lane + 32; i < n; i += 32) top = fmaxf(top, __ldcg(&p.part_ml[first + (size_t)i * R]).x);
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int j = 0; j < N * W; j++) v[j] = 0.f;
    float is = 0.f;
    for (int i = 0; i < n; i += PJ_AT) {
        if ((i & 31) == 0) {                                          // weights of 32 parts
            if (i > 0 && i + lane < n) ml = __ldcg(&p.part_ml[first + (size_t)(i + lane) * R]);
            is = i + lane < n ? exp2_approx(ml.x - ref) : 0.f;
            if (i + lane < n) sum = fmaf(is, ml.y, sum);
        }
        if (i > 0) load(i, n - 1);
#pragma unroll
        for (int c = 0; c < PJ_AT; c++) {
            const float w = __shfl_sync(0xffffffffu, is, (i + c) & 31);
            if (i + c >= n) break;
#pragma unroll
            for (int j = 0; j < N * W; j++) v[j] = fmaf(w, u[c][j], v[j]);
        }
    }
    sum = warp_sum(sum);
    const int row = t.first + r, of = p.by_group.of(row), h = hk * p.group + row - of * p.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const size_t to = (size_t)(s.first + of) * p.out_stride + (size_t)h * HD + lane * W;
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (p.xtype == PI_TYPE_F16) {
            __half * o = (__half *)p.out + to + j * 32 * W;
            if constexpr (W == 4)      *reinterpret_cast<uint2 *>(o) = make_uint2(h2u(__floats2half2_rn(v[4 * j] * inv, v[4 * j + 1] * inv)), h2u(__floats2half2_rn(v[4 * j + 2] * inv, v[4 * j + 3] * inv)));
            else if constexpr (W == 2) *reinterpret_cast<uint32_t *>(o) = h2u(__floats2half2_rn(v[2 * j] * inv, v[2 * j + 1] * inv));
            else                       *o = __float2half_rn(v[j] * inv);
        } else {
            float * o = (float *)p.out + to + j * 32 * W;
            if constexpr (W == 4)      *reinterpret_cast<float4 *>(o) = make_float4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
            else if constexpr (W == 2) *reinterpret_cast<float2 *>(o) = make_float2(v[2 * j] * inv, v[2 * j + 1] * inv);
            else                       *o = v[j] * inv;
        }
    }
}

// ---- how the work is cut
struct PaPlan { bool tc; int R, row_tiles, split, n_splits, items, whole; size_t words, q, factor, ml, part; };

// Items are a CTA (a piece of work) each, or split into ranges of at least PA_LEAST slots: none of them, those beyond as many as fill rounds of all CTAs that the SMs hold, or
// all; into the number of parts that is estimated to take the least.  A piece costs as much as its slots and PA_TURN times 64 more (on tcgen05, where parts are larger too, PA_TURN_TC
// whole and PA_TURN_PART as a part), the kernel that joins as PA_TURN times 64 (PA_JOIN_TC on tcgen05, whose CTAs even out whole pieces by themselves).  Measured on tcgen05 (us): 2 x 1024 FP16 tokens over 3000
// slots in pages of 16, 32 heads over 8 of 128, 512 pieces whole 109, 68 of them in two parts 118; 6 x 300 over 2000 65 and 68; 1024 FP32 tokens over 4096, 64 heads over 8 of 128 196 and 195; 3 x 64 FP32 tokens over 6000, 32 heads of 64,
// 96 pieces whole 61, all in three 51.
// With mma.sync: pieces are as long as max_kv says and run in rounds.  On tcgen05 CTAs take one after the other: the same for one sequence; of several half of that and half of the time of sequences of half
// to all of max_kv's length (work over SMs, and half of a piece at the end).
static constexpr int PA_LEAST = 256, PA_TURN = 4, PA_TURN_TC = 3, PA_TURN_PART = 8, PA_JOIN_TC = 12, PA_ROUNDS = 4;        // (more rounds of parts than that: room for the parts, and nothing gained)
static PaPlan pa_plan(const KvPaged & c, const RaggedB & b, int xtype, int n_head, int max_kv) {
    PaPlan r;
    const int64_t rows = (int64_t)b.max_new * (n_head / c.H);
    const int64_t keys = max_kv < 1 ? 1 : max_kv > c.n_ctx ? c.n_ctx : max_kv;
    r.tc = attn_paged_tc_takes(rows, (double)b.n * c.H * keys * c.hd);
    r.R = r.tc ? PT_ROWS : rows <= 8 ? 8 : 16;
    r.row_tiles = (int)((rows + r.R - 1) / r.R);
    const int step = r.tc ? PT_KEYS : PA_STEP;
    const int64_t items = (int64_t)b.n * c.H * r.row_tiles, pieces = r.tc && c.hd > 128 ? 2 : 1;       // (pieces of work that an item is)
    const int64_t slots = (int64_t)sm_count() * (r.tc ? 1 : c.hd == 64 ? 3 : c.hd <= 128 ? 2 : 1), units = (keys + PA_LEAST / 4 - 1) / (PA_LEAST / 4);
    const int turn = r.tc ? PA_TURN_TC : PA_TURN, turn_part = r.tc ? PA_TURN_PART : PA_TURN;
    int64_t n = 1, rest = 0;
    double least = -1;
    for (int all = 0; all <= (r.tc ? 1 : 0); all++) {
        const int64_t of = all ? items * pieces : items * pieces % slots / pieces * pieces, whole = items * pieces - of;        // pieces that are split, and not
        for (int64_t k = 1; of && k <= 128 && (k == 1 || k * PA_LEAST < keys + PA_LEAST); k++) {
            const int64_t rounds = (of * k + slots - 1) / slots, part = (units + k - 1) / k + (k > 1 ? turn_part : turn);
            if (k > 1 && rounds > PA_ROUNDS * (all ? 2 : 1)) break;
            double cost = (double)(whole / slots * (units + turn) + rounds * part);
            if (r.tc && b.n > 1) {
                const double work = (0.75 * items * pieces * units + whole * turn + of * k * (part - (units + k - 1) / k)) / slots + 0.5 * part, longest = (double)(whole ? units + turn : part);
                cost = 0.5 * (cost + (whole + of * k > slots && work > longest ? work : longest));
            }
            if (k > 1) cost += r.tc ? PA_JOIN_TC : PA_TURN;
            if (least < 0 || cost < least) { least = cost; n = k; rest = of / pieces; }
        }
    }
    const int64_t per = ((keys + n - 1) / n + step - 1) / step * step;
    r.split = (int)per; r.n_splits = (int)((keys + per - 1) / per);
    r.items = (int)items;
    r.whole = (int)(r.n_splits == 1 ? items : items - rest);
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    r.ml = up((size_t)(items - r.whole) * r.n_splits * r.R * 8);
    r.part = up((size_t)(items - r.whole) * r.n_splits * r.R * c.hd * 4);
    r.q = r.tc ? up((size_t)b.T * n_head * c.hd * (xtype == PI_TYPE_F16 ? 2 : 4)) : 0;
    r.factor = r.tc && xtype == PI_TYPE_F32 ? up((size_t)b.T * n_head * 4) : 0;
    r.words = r.tc || r.ml + r.part ? 256 : 0;                                // (the status word where pi_op_status looks for it)
    return r;
}

size_t attn_paged_scratch(const KvPaged & c, const RaggedB & b, int xtype, int n_head, int max_kv) {
    const PaPlan r = pa_plan(c, b, xtype, n_head, max_kv);
    return r.words + r.q + r.factor + r.ml + r.part;
}

template <int HD, bool TWO, int R>
static int pa_go(const AttnPagedP & p, cudaStream_t st) {
    static bool done[16] = {false};
    int dev = 0;
    PI_CUDA(cudaGetDevice(&dev));
    constexpr size_t smem = PaShape<HD>::SMEM;
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_attn_paged<HD, TWO, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PI_CUDA(launch_k(k_attn_paged<HD, TWO, R>, dim3(ap_grid(p)), dim3(PA_THREADS), smem, st, true, p));
    return PI_OK;
}

template <int HD>
static int pa_run(const AttnPagedP & p, const PaPlan & r, cudaStream_t st) {
    const int rc = r.tc ? launch_attn_paged_tc(p, st) : r.R == 8 ? (p.xtype == PI_TYPE_F16 ? pa_go<HD, false, 8>(p, st) : pa_go<HD, true, 8>(p, st)) : p.xtype == PI_TYPE_F16 ? pa_go<HD, false, 16>(p, st) : pa_go<HD, true, 16>(p, st);
    if (rc) return rc;
    if (p.items > p.whole) PI_CUDA(launch_k(k_attn_paged_join<HD>, dim3((unsigned)(((int64_t)(p.items - p.whole) * r.R + PJ_WARPS - 1) / PJ_WARPS)), dim3(PJ_WARPS * 32), 0, st, true, p, r.R));
    return PI_OK;
}

int launch_attention_paged(const AttnPagedArgs & a, cudaStream_t st) {
    const PaPlan r = pa_plan(a.c, a.b, a.xtype, a.n_head, a.max_kv);
    AttnPagedP p;
    p.c = a.c; p.b = a.b; p.xtype = a.xtype; p.q = a.q; p.q_stride = a.q_stride; p.n_head = a.n_head; p.group = a.n_head / a.c.H;
    p.mask = a.mask; p.words = a.words;
    p.scale_log2 = a.scale * 1.44269504088896340736f; p.out = a.out; p.out_stride = a.out_stride;
    p.split = r.split; p.n_splits = r.n_splits; p.row_tiles = r.row_tiles; p.items = r.items; p.whole = r.whole;
    p.by_group = AqDiv::by(p.group); p.by_heads = AqDiv::by(a.c.H); p.by_tiles = AqDiv::by(r.row_tiles); p.by_splits = AqDiv::by(r.n_splits);
    char * s = (char *)a.scratch;
    p.status = s ? (unsigned int *)(s + 8) : nullptr;
    s += r.words;
    p.queries = (__half *)s; p.factor = (float *)(s + r.q);
    s += r.q + r.factor;
    p.part_ml = (float2 *)s; p.part = (float *)(s + r.ml);
    switch (a.c.hd) {
        case 64:  return pa_run<64>(p, r, st);
        case 96:  return pa_run<96>(p, r, st);
        case 128: return pa_run<128>(p, r, st);
        case 192: return pa_run<192>(p, r, st);
        default:  return pa_run<256>(p, r, st);
    }
}

}  // namespace pi
