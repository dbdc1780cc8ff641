// Attention over the KV cache in 8 bits, for a ragged batch: query t of sequence i (slot pos0[i] + t) sees slots 0 .. pos0[i] + t.
//
//     s_j = scale * ks[j / B] * (q . k_j)     p_j = exp(s_j - max s)     out = sum_j p_j vs[j / B] v_j / sum_j p_j
//
// Bound by the bytes of the codes.  A CTA takes 8 or 16 query rows that read one KV head (the query heads of a group, of one or more
// tokens) and a range of slots; its four warps take 16 slots each in turn, copied ahead into a ring of their own (cp.async; no barrier
// between warps), keep a maximum, a sum and all sums of values of their own, and join them at the end.  Long ranges are
// split over CTAs, whose sums k_attn_q8_join joins.
//
// Measured (FP16 or FP32 rows, head_dim 128): 32 sequences of 1056 to 2048 slots, 32 heads 79 us (5.2 TB/s; between two lengths 6.7, the copy rate: the rest is what
// CTAs do before their first slot and behind their last, the tail and the launches), one of 32768 slots, 64 heads over 8 KV heads 17 us and 5 of the join.
// Queries are asked for before the ring's codes: behind them they took 3 us of a CTA's 15.
//
// Precision.  Scores of 8 rows are products of whole numbers: the codes as they lie, and a query row of 31 bits and a sign as four digits of 8 bits, which are four rows
// of the tensor cores' tile; their sums are exact.  16 rows have queries as halves, FP16 as they are and FP32 as the sum of two (22 bits), and the codes become halves
// for them: digits are four products for all of the rows, 160 us where two halves take 149 and one 132 (8 sequences of 7 tokens, 8000 slots, 64 heads over 8).
// A probability, times vs over the largest vs so far (at most 1), is the sum of
// two halves, rows 0 .. 7 the upper and rows 8 .. 15 the lower parts, 22 bits down to 2^-10 of the largest vs (held times 2^8 over the power of two
// above it, steps of 2^-24: an error of 2^-32 of that vs below), and a value's code is exact as a half: out = sums * that scale.  The scale is a row's own, of what it sees.  (Probabilities as
// digits would spare the values' conversions, but their sums fill twice the registers, and whole numbers cannot follow a maximum that rises.)
// Maxima, sums and the exponents' arguments are FP32.
//
// Layouts.  mma sums over 32 columns (scores) or 16 slots (values) in any order that both operands share: a lane's piece of a key row is
// 16 contiguous codes, of a value row hd / 8 of them, and every 4 codes are operands of one product.  The probabilities of the score tile's layout
// are the value product's operand as they stand.  Where the maximum rises by less than 2^7, sums are not scaled anew.
#include "pi_attn_q8.cuh"

#include <cfloat>

namespace pi {

static constexpr int AQ_WARPS = 4, AQ_THREADS = AQ_WARPS * 32, AQ_STEP = AQ_WARPS * 16;
static constexpr float AQ_RISE = 7.f, AQ_P = 256.f;                   // bits a maximum may lag; probabilities are held times this (2^7 * 256 < 65504)
static constexpr float AQ_V_LEAST = 0x1p-118f;                        // values' scales below it count relative to it: AQ_P over a scale, and a scale over AQ_P, are normal numbers

template <int HD> struct AqShape {
    static constexpr int KW = HD % 64 == 0 ? 16 : 8, KG = HD / (4 * KW);                   // codes a lane takes of a key row at once, and how often
    static constexpr int VW = HD % 128 == 0 ? 16 : HD % 64 == 0 ? 8 : 4, VG = HD / (8 * VW);
    static constexpr int KS = HD / 16, NT = HD / 8;
    // 16-byte pieces of a slot's row, permuted so that the lanes that load together meet all banks
    static __device__ __forceinline__ int k_at(int row, int byte) { return row * HD + (HD % 128 == 0 ? byte ^ ((row & 1) << 6) : byte); }
    static __device__ __forceinline__ int v_at(int row, int byte) { return row * HD + (HD % 128 == 0 ? byte ^ (((row >> 1) & 3) << 5) : byte); }
    static constexpr int STAGES = HD <= 128 ? 4 : 3, STAGE = 2 * 16 * HD;
    static constexpr int ctas(int mt) { return HD <= 128 && mt == 1 ? 3 : 2; }           // that an SM holds
    // shared memory: the ring, in the end the warps' sums in its place, and the queries
    static constexpr size_t RING = (size_t)AQ_WARPS * STAGES * STAGE;
    template <int MT> static constexpr size_t DIGITS = RING > (size_t)AQ_WARPS * 8 * MT * (HD + 4) * 4 ? RING : (size_t)AQ_WARPS * 8 * MT * (HD + 4) * 4;
    template <int MT> static constexpr size_t SMEM = DIGITS<MT> + (MT == 1 ? 4 * 8 * (HD + 16) : 2 * 16 * (2 * HD + 16));
};

template <int W> __device__ __forceinline__ void aq_lds(uint32_t (&r)[W / 4], const unsigned char * p) {
    if constexpr (W == 16)     { const uint4 u = *reinterpret_cast<const uint4 *>(p); r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w; }
    else if constexpr (W == 8) { const uint2 u = *reinterpret_cast<const uint2 *>(p); r[0] = u.x; r[1] = u.y; }
    else                       r[0] = *reinterpret_cast<const uint32_t *>(p);
}

// A query row of 8 in whole numbers of 31 bits and a sign, as four digits to the base 256 (-128 .. 127), four columns at a time.  (Three digits, 23 bits, are too few: a value is off by
// half of 1, whatever its size is, and queries with a channel tens of times larger than the others are usual.  With four, FP32 values within 2^-7 of the row's
// largest and FP16 ones within 2^-20 are exact.)
struct AqScaled { float up, down; };                                  // factor of the row; of its scores (not a number where a value of the row is not finite: so are they)
__device__ __forceinline__ void aq_max(const float4 & v, float & m, float & zero) {    // zero: no more 0 where a value is not finite
    m = fmaxf(fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    zero = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, zero))));
}
// the largest to 2^29 x 1.98 .. 2^30 x 1.98: four digits reach 2^30 x 1.992.  A value is off by half of 1, at most 2^-30.9 of the largest
__device__ __forceinline__ AqScaled aq_scaled(float m) {
    const int e = min(max((int)((__float_as_uint(m) + 0x20000u) >> 23) - 127, -92), 128) - 30;
    return {__uint_as_float((uint32_t)(127 - e) << 23), m < INFINITY ? __uint_as_float((uint32_t)(127 + e) << 23) : __int_as_float(0x7fc00000)};
}
// the largest to 2^10 .. 2^11: a value as two halves is off by 2^-22 of itself, or by 2^-25 (lower parts have no steps below 2^-24)
__device__ __forceinline__ AqScaled aq_scaled_halves(float m) {
    const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127) - 10;
    return {__uint_as_float((uint32_t)(127 - e) << 23), m < INFINITY ? __uint_as_float((uint32_t)(127 + e) << 23) : __int_as_float(0x7fc00000)};
}
__device__ __forceinline__ void aq_digits(const float4 & x, float up, uint32_t (&d)[4]) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t t[4];
#pragma unroll
    for (int j = 0; j < 4; j++) t[j] = (uint32_t)__float2int_rn(v[j] * up) + 0x80808080u;          // digits + 128
    const uint32_t a = __byte_perm(t[0], t[1], 0x5140), b = __byte_perm(t[2], t[3], 0x5140), c = __byte_perm(t[0], t[1], 0x7362), e = __byte_perm(t[2], t[3], 0x7362);
    d[0] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
    d[1] = __byte_perm(a, b, 0x7632) ^ 0x80808080u;
    d[2] = __byte_perm(c, e, 0x5410) ^ 0x80808080u;
    d[3] = __byte_perm(c, e, 0x7632) ^ 0x80808080u;
}
__device__ __forceinline__ size_t aq_query_at(const AttnQ8P & p, const SeqB & s, int row, int hk, int hd) {
    const int tok = p.by_group.of(row);
    return (size_t)(s.first + tok) * p.q_stride + (size_t)(hk * p.group + row - tok * p.group) * hd;
}
// A lane's pieces of one row as A operands (which only its warp needs): a[d] the d-th digits of every 4 of its columns.  Returns the factor of the scores.
template <int HD>
__device__ __forceinline__ float aq_load_query(const AttnQ8P & p, const SeqB & s, int row, bool there, int hk, int q, uint32_t (&a)[4][HD / 16]) {
    using S = AqShape<HD>;
    float4 x[S::KS];
    float m = 0.f, zero = 0.f;
    const size_t at = there ? aq_query_at(p, s, row, hk, HD) : 0;
#pragma unroll
    for (int c = 0; c < S::KG; c++)
#pragma unroll
        for (int w = 0; w < S::KW / 4; w++) {
            float4 & v = x[c * (S::KW / 4) + w];
            v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (there) v = aq_query(p.xtype, p.q, at + c * 4 * S::KW + q * S::KW + w * 4);
            aq_max(v, m, zero);
        }
    if (zero != 0.f) m = INFINITY;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const AqScaled f = aq_scaled(m);
#pragma unroll
    for (int i = 0; i < S::KS; i++) {
        uint32_t d[4];
        aq_digits(x[i], f.up, d);
#pragma unroll
        for (int k = 0; k < 4; k++) a[k][i] = d[k];
    }
    return f.down * p.scale_log2;
}
// The R rows of a tile in shared memory, by the whole CTA: 8 as digits [digit][row][HD + 16], 16 as halves [upper, lower][row][HD + 8], and the factors of their scores.  The loads come before what
// else the CTA asks for: behind the ring's first codes they are waited for 3 us.
template <int HD, int R> struct AqQueries {
    static constexpr int TPR = AQ_THREADS / R, W = HD / 4, N = (W + TPR - 1) / TPR, PITCH = R == 8 ? HD + 16 : 2 * HD + 16;
    float4 x[N];
    __device__ __forceinline__ void load(const AttnQ8P & p, const SeqB & s, const TileB & t, int hk) {
        const int row = threadIdx.x / TPR, j = threadIdx.x % TPR;
        const size_t at = row < t.n_rows ? aq_query_at(p, s, t.first + row, hk, HD) : 0;
#pragma unroll
        for (int u = 0; u < N; u++) {
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < t.n_rows && j + u * TPR < W) x[u] = aq_query(p.xtype, p.q, at + (j + u * TPR) * 4);
        }
    }
    template <bool TWO_Q> __device__ __forceinline__ void put(const AttnQ8P & p, unsigned char * to, float * factor) {
        const int row = threadIdx.x / TPR, j = threadIdx.x % TPR;
        float m = 0.f, zero = 0.f;
#pragma unroll
        for (int u = 0; u < N; u++) aq_max(x[u], m, zero);
        if (zero != 0.f) m = INFINITY;
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const AqScaled f = R == 8 ? aq_scaled(m) : TWO_Q ? aq_scaled_halves(m) : AqScaled{1.f, m < INFINITY ? 1.f : __int_as_float(0x7fc00000)};
        if (j == 0) factor[row] = f.down * p.scale_log2;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const bool mine = j + u * TPR < W;
            if constexpr (R == 8) {
                uint32_t d[4];
                aq_digits(x[u], f.up, d);
#pragma unroll
                for (int k = 0; k < 4; k++) if (mine) *reinterpret_cast<uint32_t *>(to + (k * R + row) * PITCH + (j + u * TPR) * 4) = d[k];
            } else {
                uint2 hi, lo;
                aq_split(x[u].x * f.up, x[u].y * f.up, hi.x, lo.x);
                aq_split(x[u].z * f.up, x[u].w * f.up, hi.y, lo.y);
                if (mine) *reinterpret_cast<uint2 *>(to + row * PITCH + (j + u * TPR) * 8) = hi;
                if (TWO_Q && mine) *reinterpret_cast<uint2 *>(to + (R + row) * PITCH + (j + u * TPR) * 8) = lo;
            }
        }
    }
};

// Sums of products of digits and codes are whole numbers up to 2^22 (256 x 128 x 128): begun at 1.5 x 2^23's bits, they are that number plus the sum.
static constexpr int AQ_ZERO = 0x4B400000;
// d += (16 rows of 32 digits) x (32 codes of 8 slots)
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool first) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1),
                   "r"(first ? AQ_ZERO : d[0]), "r"(first ? AQ_ZERO : d[1]), "r"(first ? AQ_ZERO : d[2]), "r"(first ? AQ_ZERO : d[3]));
}
__device__ __forceinline__ float aq_score(int d3, int d2, int d1, int d0) {
    const float f3 = __int_as_float(d3) - 12582912.f, f2 = __int_as_float(d2) - 12582912.f, f1 = __int_as_float(d1) - 12582912.f, f0 = __int_as_float(d0) - 12582912.f;
    return fmaf(fmaf(fmaf(f3, 256.f, f2), 256.f, f1), 256.f, f0);
}
// products of 32 columns of 8 slots (b0, b1) and of 8 rows: x[digits 3 | 2], x[digits 1 | 0]
template <int HD>
__device__ __forceinline__ void aq_products(int (&x)[2][4], const uint32_t (&a)[4][HD / 16], int s, uint32_t b0, uint32_t b1) {
#pragma unroll
    for (int d = 0; d < 2; d++) mma16832(x[d], a[3 - 2 * d][2 * s], a[2 - 2 * d][2 * s], a[3 - 2 * d][2 * s + 1], a[2 - 2 * d][2 * s + 1], b0, b1, s == 0);
}
__device__ __forceinline__ float aq_score_of(const int (&x)[2][4], int j) { return aq_score(x[0][j], x[0][2 + j], x[1][j], x[1][2 + j]); }

// TWO_Q: of 16 rows two halves for each query; 8 rows are digits
template <int HD, int MT, bool TWO_Q>
__global__ void __launch_bounds__(AQ_THREADS, AqShape<HD>::ctas(MT)) k_attn_q8(const AttnQ8P p) {
    using S = AqShape<HD>;
    constexpr int R = 8 * MT, ST = S::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_m[AQ_WARPS][R], s_l[AQ_WARPS][R], s_back[AQ_WARPS][R], s_f[R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const AqItem wk = aq_item(p, blockIdx.x);
    const int split = wk.split, rt = wk.rt, hk = wk.hk;
    pdl_launch();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && p.status) *p.status = 0u;          // (no wait of this kernel runs out)
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, wk.entry);
    const TileB t = aq_tile(p, s, rt, R);
    if (t.n_rows <= 0) return;
    const int k0 = split * p.split, k1 = split == wk.n_splits - 1 ? t.seen : min(t.seen, k0 + p.split);
    if (k0 >= k1 && split > 0) return;                                // (split 0 answers for rows that see nothing)

    unsigned char * digits = smem + S::template DIGITS<MT>;
    AqQueries<HD, R> queries;
    queries.load(p, s, t, hk);
    const size_t head = (size_t)max(s.sq, 0) * p.c.H + hk;
    const int8_t * kc = p.c.k + head * p.c.n_ctx * HD, * vc = p.c.v + head * p.c.n_ctx * HD;
    const float * ks = p.c.ks + head * (p.c.n_ctx >> p.c.shift), * vs = p.c.vs + head * (p.c.n_ctx >> p.c.shift);
    const unsigned char * ring = smem + (size_t)warp * ST * S::STAGE;
    const int first = k0 + warp * 16, steps = first < k1 ? (k1 - first + AQ_STEP - 1) / AQ_STEP : 0;
    const int8_t * k_next = kc + (size_t)first * HD + lane * 16, * v_next = vc + (size_t)first * HD + lane * 16;     // (16 slots from a multiple of 16: inside the cache)
    const uint32_t ring_at = smem_u32(ring);
    int left = steps; uint32_t fill = ring_at;                        // steps to be asked for, and where the next one goes
    auto issue = [&]() {
        if (left > 0) {
#pragma unroll
            for (int u = 0; u < HD / 32; u++) {
                const int b = (u * 32 + lane) * 16, row = b / HD, byte = b % HD;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(fill + S::k_at(row, byte)), "l"(k_next + u * 512) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(fill + 16 * HD + S::v_at(row, byte)), "l"(v_next + u * 512) : "memory");
            }
            k_next += AQ_STEP * HD; v_next += AQ_STEP * HD;
            left--;
            fill = fill == ring_at + (ST - 1) * S::STAGE ? ring_at : fill + S::STAGE;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int it = 0; it < ST - 1; it++) issue();

    queries.template put<TWO_Q>(p, digits, s_f);
    __syncthreads();
    float f[MT], m[MT], l[MT]; int sees[MT], least = 0x7fffffff; bool there[MT];
    int scores[MT];                                                   // place of its scores (-1: not kept)
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = mt * 8 + g, tok = p.by_group.of(t.first + row);
        there[mt] = row < t.n_rows;
        f[mt] = s_f[row];
        sees[mt] = there[mt] ? aq_sees(s, p.c.n_ctx, tok) : 0;
        if (there[mt]) least = min(least, sees[mt]);
        scores[mt] = p.scores && there[mt] ? ((s.first + tok) * p.n_head + hk * p.group + t.first + row - tok * p.group) * p.score_pitch + 2 * q : -1;
        m[mt] = -INFINITY; l[mt] = 0.f;
    }
    uint32_t a[4][S::KS];                                             // 8 rows: [digit]; 16 rows: [2 row / 8 + pair of columns] upper and, with two halves, lower parts
    uint32_t a_low[TWO_Q && MT == 2 ? 4 : 1][S::KS];
#pragma unroll
    for (int c = 0; c < S::KG; c++) {
        const int col = c * 4 * S::KW + q * S::KW;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (MT == 1) {
                uint32_t w[S::KW / 4];
                aq_lds<S::KW>(w, digits + (k * R + g) * (HD + 16) + col);
#pragma unroll
                for (int i = 0; i < S::KW / 4; i++) a[k][c * (S::KW / 4) + i] = w[i];
            } else {
                const unsigned char * from = digits + ((k >> 1) * 8 + g) * (2 * HD + 16) + col * 2 + (k & 1) * 4;
#pragma unroll
                for (int i = 0; i < S::KW / 4; i++) {
                    a[k][c * (S::KW / 4) + i] = *reinterpret_cast<const uint32_t *>(from + i * 8);
                    if constexpr (TWO_Q && HD != 128) a_low[k][c * (S::KW / 4) + i] = *reinterpret_cast<const uint32_t *>(from + R * (2 * HD + 16) + i * 8);
                }
            }
        }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    float o[MT][S::NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int n = 0; n < S::NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[mt][n][j] = 0.f;
    uint32_t v_ref[MT];                                               // scale of a row's value sums, a power of two, as bits (of what the row sees: others' scales have no say in it)
#pragma unroll
    for (int mt = 0; mt < MT; mt++) v_ref[mt] = __float_as_uint(AQ_V_LEAST);

    const unsigned char * kt = ring + (ST - 1) * S::STAGE;
    for (int it = 0; it < steps; it++) {
        asm volatile("cp.async.wait_group %0;" :: "n"(ST - 2) : "memory");
        __syncwarp();                                                 // the stage is there for all lanes, and all have read the last one
        issue();                                                      // (into which this goes)
        kt = kt == ring + (ST - 1) * S::STAGE ? ring : kt + S::STAGE;
        const unsigned char * vt = kt + 16 * HD;
        const int j0 = first + it * AQ_STEP;
        const float sk = __ldg(ks + (j0 >> p.c.shift)), sv = __ldg(vs + (j0 >> p.c.shift));

        // ---- scores of 16 slots
        float raw[MT][2][2];
        if constexpr (MT == 1) {
            int x[2][2][4];
#pragma unroll
            for (int c = 0; c < S::KG; c++) {
                uint32_t w[2][S::KW / 4];
#pragma unroll
                for (int n = 0; n < 2; n++) aq_lds<S::KW>(w[n], kt + S::k_at(n * 8 + g, c * 4 * S::KW + q * S::KW));
#pragma unroll
                for (int i = 0; i < S::KW / 8; i++)
#pragma unroll
                    for (int n = 0; n < 2; n++) aq_products<HD>(x[n], a, c * (S::KW / 8) + i, w[n][2 * i], w[n][2 * i + 1]);
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) raw[0][n][j] = aq_score_of(x[n], j);
        } else {
            float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < S::KG; c++) {
                uint32_t w[2][S::KW / 4];
#pragma unroll
                for (int n = 0; n < 2; n++) aq_lds<S::KW>(w[n], kt + S::k_at(n * 8 + g, c * 4 * S::KW + q * S::KW));
                if constexpr (TWO_Q && HD == 128) {                   // (lower parts anew in every step: in registers they spill, 159 us for 149)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint4 * from = reinterpret_cast<const uint4 *>(digits + (R + h * 8 + g) * (2 * HD + 16) + (c * 4 * S::KW + q * S::KW) * 2);
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint4 v = from[u];
                            a_low[2 * h][c * 4 + 2 * u] = v.x; a_low[2 * h + 1][c * 4 + 2 * u] = v.y; a_low[2 * h][c * 4 + 2 * u + 1] = v.z; a_low[2 * h + 1][c * 4 + 2 * u + 1] = v.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < S::KW / 4; i++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const uint32_t u = w[n][i] ^ 0x80808080u, b0 = q8_lo(u), b1 = q8_hi(u);
                        const int k = c * (S::KW / 4) + i;
                        if constexpr (TWO_Q) mma16816(x[n], a_low[0][k], a_low[2][k], a_low[1][k], a_low[3][k], b0, b1);
                        mma16816(x[n], a[0][k], a[2][k], a[1][k], a[3][k], b0, b1);
                    }
            }
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) raw[j >> 1][n][j & 1] = x[n][j];
        }
        // ---- probabilities, as A operands of the value products
        uint32_t pa[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            // to the power of two above it: one rise where the scales are of one size.  (In bits: a division in a branch that some rows take cost 20 us of 141.)
            const uint32_t now = j0 < sees[mt] && sv >= __uint_as_float(v_ref[mt]) ? min((__float_as_uint(sv) & 0x7f800000u) + 0x00800000u, 0x7f000000u) : v_ref[mt];
            float down = __int_as_float(max(0x3f800000 - (int)(now - v_ref[mt]), 0));
            v_ref[mt] = now;
            const float pv = sv * __uint_as_float((262u << 23) - now);                   // (AQ_P = 2^8 over it)
            float y[2][2];
            const float fk = f[mt] * sk;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) y[n][j] = raw[mt][n][j] * fk;
            const bool masked = j0 + 16 > least;
            if (masked) {
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++) if (j0 + n * 8 + 2 * q + j >= sees[mt]) y[n][j] = -INFINITY;
            }
            if (scores[mt] >= 0) {
                float * to = p.scores + scores[mt] + j0;
                *reinterpret_cast<float2 *>(to) = make_float2(y[0][0], y[0][1]);
                *reinterpret_cast<float2 *>(to + 8) = make_float2(y[1][0], y[1][1]);
            }
            float top = fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[1][0], y[1][1]));
            if (__any_sync(0xffffffffu, top > m[mt] + AQ_RISE)) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float now = fmaxf(m[mt], top), alpha = now == m[mt] ? 1.f : exp2_approx(m[mt] - now);
                m[mt] = now;
                l[mt] *= alpha;
                down *= alpha;
            }
            if (it > 0 && __any_sync(0xffffffffu, down != 1.f)) {
#pragma unroll
                for (int n = 0; n < S::NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[mt][n][j] *= down;
            }
            const float ref = m[mt] == -INFINITY ? 0.f : m[mt];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float p0 = exp2_approx(y[n][0] - ref), p1 = exp2_approx(y[n][1] - ref);
                l[mt] += p0 + p1;
                float w0 = p0 * pv, w1 = p1 * pv;
                if (masked) { if (p0 == 0.f) w0 = 0.f; if (p1 == 0.f) w1 = 0.f; }       // (a masked slot counts nothing whatever its block's scale is)
                aq_split(w0, w1, pa[mt][2 * n], pa[mt][2 * n + 1]);
            }
        }
        // ---- values: the lane's slots are 2q, 2q + 1, 8 + 2q, 9 + 2q
#pragma unroll
        for (int c = 0; c < S::VG; c++) {
            uint32_t w[4][S::VW / 4];
#pragma unroll
            for (int r = 0; r < 4; r++) aq_lds<S::VW>(w[r], vt + S::v_at((r >> 1) * 8 + 2 * q + (r & 1), c * 8 * S::VW + g * S::VW));
#pragma unroll
            for (int i = 0; i < S::VW / 4; i++) {
                const uint32_t lo0 = __byte_perm(w[0][i], w[1][i], 0x5140) ^ 0x80808080u, hi0 = __byte_perm(w[0][i], w[1][i], 0x7362) ^ 0x80808080u;
                const uint32_t lo1 = __byte_perm(w[2][i], w[3][i], 0x5140) ^ 0x80808080u, hi1 = __byte_perm(w[2][i], w[3][i], 0x7362) ^ 0x80808080u;
                const uint32_t b[4][2] = {{q8_lo(lo0), q8_lo(lo1)}, {q8_hi(lo0), q8_hi(lo1)}, {q8_lo(hi0), q8_lo(hi1)}, {q8_hi(hi0), q8_hi(hi1)}};
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) mma16816(o[mt][c * S::VW + i * 4 + j], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], b[j][0], b[j][1]);
            }
        }
    }

    // ---- the four warps' sums together
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    constexpr int PITCH = HD + 4;
    float * so = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        float sum = l[mt];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (q == 0) { s_m[warp][mt * 8 + g] = m[mt]; s_l[warp][mt * 8 + g] = sum; s_back[warp][mt * 8 + g] = __uint_as_float(v_ref[mt]) * (1.f / AQ_P); }
        float * row = so + (size_t)(warp * R + mt * 8 + g) * PITCH;
#pragma unroll
        for (int c = 0; c < S::VG; c++)
#pragma unroll
            for (int h = 0; h < 2; h++)                               // columns 2q and 2q + 1 of the tiles: VW contiguous dimensions each
#pragma unroll
                for (int j = 0; j < S::VW; j += 4) {
                    float4 v;
                    v.x = (o[mt][c * S::VW + j][h] + o[mt][c * S::VW + j][h + 2]);
                    v.y = (o[mt][c * S::VW + j + 1][h] + o[mt][c * S::VW + j + 1][h + 2]);
                    v.z = (o[mt][c * S::VW + j + 2][h] + o[mt][c * S::VW + j + 2][h + 2]);
                    v.w = (o[mt][c * S::VW + j + 3][h] + o[mt][c * S::VW + j + 3][h + 2]);
                    *reinterpret_cast<float4 *>(row + c * 8 * S::VW + (2 * q + h) * S::VW + j) = v;
                }
    }
    __syncthreads();
    const size_t part0 = ((size_t)(wk.item - p.whole) * p.n_splits + split) * R;
    for (int e = threadIdx.x; e < t.n_rows * (HD / 4); e += AQ_THREADS) {
        const int r = e / (HD / 4), d = (e - r * (HD / 4)) * 4;
        float top = s_m[0][r];
#pragma unroll
        for (int w = 1; w < AQ_WARPS; w++) top = fmaxf(top, s_m[w][r]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f; float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < AQ_WARPS; w++) {
            const float is = exp2_approx(s_m[w][r] - ref), k = is * s_back[w][r];
            const float4 u = *reinterpret_cast<const float4 *>(so + (size_t)(w * R + r) * PITCH + d);
            sum = fmaf(is, s_l[w][r], sum);
            v.x = fmaf(k, u.x, v.x); v.y = fmaf(k, u.y, v.y); v.z = fmaf(k, u.z, v.z); v.w = fmaf(k, u.w, v.w);
        }
        if (wk.n_splits > 1) {
            *reinterpret_cast<float4 *>(p.part + (part0 + r) * HD + d) = v;
            if (d == 0) p.part_ml[part0 + r] = make_float2(top, sum);
        } else {
            const int row = t.first + r, of = p.by_group.of(row), tok = s.first + of, h = hk * p.group + row - of * p.group;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const size_t at = (size_t)tok * p.out_stride + (size_t)h * HD + d;
            aq_put(p.xtype, p.out, at, v.x * inv); aq_put(p.xtype, p.out, at + 1, v.y * inv);
            aq_put(p.xtype, p.out, at + 2, v.z * inv); aq_put(p.xtype, p.out, at + 3, v.w * inv);
            if (d == 0 && p.lse) p.lse[(size_t)tok * p.n_head + h] = sum == 0.f ? INFINITY : top + log2f(sum);
        }
    }
}

// The splits of a tile joined, in their order.  WPR warps have a row (its splits dealt to them): one where splits are few, eight where one row's
// many partial sums are all there is to wait for (64 rows of 37 splits: a CTA for each tile of rows took 25 us).
static constexpr int AQ_JOIN_FEW = 8;

template <int WPR>
__global__ void __launch_bounds__(256) k_attn_q8_join(const AttnQ8P p, int R) {
    __shared__ float s_sum[8][257];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR, hd = p.c.hd, nd = hd / 32;
    const int at_row = blockIdx.x * (8 / WPR) + warp / WPR, k_item = at_row / R, r = at_row - k_item * R;
    pdl_launch();
    pdl_wait();
    if (k_item >= p.items - p.whole) return;                          // (with WPR = 8: the whole CTA)
    // (the sums are asked for before it is known which splits there are: the others' are dropped.  One way to memory instead of three.)
    const size_t part0 = (size_t)k_item * p.n_splits * R + r;
    float top = -INFINITY, mk[4];
#pragma unroll
    for (int u = 0; u < 4; u++) mk[u] = lane + 32 * u < p.n_splits ? __ldcg(&p.part_ml[part0 + (size_t)(lane + 32 * u) * R]).x : -INFINITY;      // (128 splits at most)
    constexpr int U = 8;
    float2 ml[U]; float pv[U][8];
    auto ask = [&](int k0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = min(k0 + u * WPR, p.n_splits - 1);
            const size_t at = part0 + (size_t)k * R;
            ml[u] = __ldcg(&p.part_ml[at]);
#pragma unroll
            for (int j = 0; j < 8; j++) if (j < nd) pv[u][j] = __ldcg(p.part + at * hd + lane + 32 * j);
        }
    };
    ask(sub);
    const AqItem wk = aq_item(p, p.whole + k_item * p.n_splits);
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, wk.entry);
    const TileB t = aq_tile(p, s, R == AT_ROWS ? p.row_tiles - 1 - wk.rt : wk.rt, R);
    if (r >= t.n_rows) return;
    const int used = max(1, min(p.n_splits, (t.seen + p.split - 1) / p.split));
#pragma unroll
    for (int u = 0; u < 4; u++) if (lane + 32 * u < used) top = fmaxf(top, mk[u]);
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int k0 = sub; k0 < used; k0 += U * WPR) {
        if (k0 != sub) ask(k0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (k0 + u * WPR >= used) break;
            const float w = exp2_approx(ml[u].x - ref);
            sum = fmaf(w, ml[u].y, sum);
#pragma unroll
            for (int j = 0; j < 8; j++) if (j < nd) v[j] = fmaf(w, pv[u][j], v[j]);
        }
    }
    if (WPR > 1) {
#pragma unroll
        for (int j = 0; j < 8; j++) if (j < nd) s_sum[warp][lane + 32 * j] = v[j];
        if (lane == 0) s_sum[warp][256] = sum;
        __syncthreads();
        if (warp > 0) return;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; w++) sum += s_sum[w][256];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < nd) {
                v[j] = 0.f;
#pragma unroll
                for (int w = 0; w < WPR; w++) v[j] += s_sum[w][lane + 32 * j];
            }
    }
    const int row = t.first + r, of = p.by_group.of(row), tok = s.first + of, h = wk.hk * p.group + row - of * p.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const size_t at = (size_t)tok * p.out_stride + (size_t)h * hd + lane;
#pragma unroll
    for (int j = 0; j < 8; j++) if (j < nd) aq_put(p.xtype, p.out, at + 32 * j, v[j] * inv);
    if (lane == 0 && p.lse) p.lse[(size_t)tok * p.n_head + h] = sum == 0.f ? INFINITY : top + log2f(sum);
}

// The accumulated weights where the scores were kept (AqPlan::scores): four slots a thread.  With w_j = sum over the sequence's new tokens and the heads of the
// group of p_j, weights_out[j] = (j < pos0 ? weights_in[j] : 0) + w_j, rows in their order.
__global__ void __launch_bounds__(128) k_attn_q8_weights_kept(const AttnQ8P p, const float * w_in, float * w_out) {
    const int hk = blockIdx.y, i = blockIdx.z, lane = threadIdx.x & 31, j0 = (blockIdx.x * 128 + threadIdx.x) * 4;
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, i);
    const int end = min(s.pos + s.n_new, p.c.n_ctx);
    if (s.sq < 0 || s.n_new == 0 || blockIdx.x * 512 >= end) return;
    bool later = false;                                               // of entries that name one sequence the last one counts
    if (p.b.seq)
        for (int j = i + 1 + lane; j < p.b.n; j += 32) {
            const SeqB o = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, j);
            later |= o.sq == s.sq && o.n_new > 0;
        }
    if (__any_sync(0xffffffffu, later) || j0 >= end) return;
    const size_t at = ((size_t)s.sq * p.c.H + hk) * p.c.n_ctx + j0;  // (n_ctx is a multiple of 16)
    const bool before = w_in && j0 < s.pos;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 had = before ? make_float4(w_in[at], w_in[at + 1], w_in[at + 2], w_in[at + 3]) : sum;
    const int rows = s.n_new * p.group;
#pragma unroll 8
    for (int r = max(0, j0 - s.pos) * p.group; r < rows; r++) {      // (from the first token that sees one of these slots)
        const int tok = p.by_group.of(r), row = (s.first + tok) * p.n_head + hk * p.group + r - tok * p.group;
        const float lse = __ldcg(p.lse + row);
        const int sees = aq_sees(s, p.c.n_ctx, tok) - j0;             // (scores of what a row does not see were not all made)
        const float4 y = __ldcg(reinterpret_cast<const float4 *>(p.scores + (size_t)row * p.score_pitch + j0));
        if (sees > 0) sum.x += exp2_approx(y.x - lse);
        if (sees > 1) sum.y += exp2_approx(y.y - lse);
        if (sees > 2) sum.z += exp2_approx(y.z - lse);
        if (sees > 3) sum.w += exp2_approx(y.w - lse);
    }
    const float v[4] = {sum.x, sum.y, sum.z, sum.w}, h[4] = {had.x, had.y, had.z, had.w};
#pragma unroll
    for (int j = 0; j < 4; j++) if (j0 + j < end) w_out[at + j] = (j0 + j < s.pos ? h[j] : 0.f) + v[j];
}

// weights_out[j] = (j < pos0 ? weights_in[j] : 0) + sum over the sequence's new tokens and the heads of the group of p_j.  The keys are read a second time
// and the scores made again, instead of every score written and read: a warp has the codes of AQ_WT x 16 slots in registers and goes over the rows, 8 at a
// time.  One warp owns a slot: the sum's order is fixed.  Bound by the way from one load to the next: a CTA takes several tiles of slots, and where there are no more
// than 8 rows their queries are made once (8 sequences of 64 heads, 8000 slots: a tile a CTA 47 us, and its loads one after the other).
static constexpr int AQ_WT = 2, AQ_WSTEP = AQ_WARPS * AQ_WT * 16;

template <int HD>
__global__ void __launch_bounds__(AQ_THREADS, HD <= 64 ? 4 : HD <= 128 ? 3 : 2) k_attn_q8_weights(const AttnQ8P p, const float * w_in, float * w_out) {
    using S = AqShape<HD>;
    constexpr int NK = 2 * AQ_WT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3, hk = blockIdx.y, i = blockIdx.z;
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, i);
    if (s.sq < 0 || s.n_new == 0) return;
    const int end = min(s.pos + s.n_new, p.c.n_ctx), n_rows = s.n_new * p.group;
    int j0 = blockIdx.x * AQ_WSTEP + warp * AQ_WT * 16;
    if (j0 >= end) return;
    const size_t head = (size_t)s.sq * p.c.H + hk;
    const int8_t * kc = p.c.k + head * p.c.n_ctx * HD;
    const float * ks = p.c.ks + head * (p.c.n_ctx >> p.c.shift);
    uint32_t w[NK][S::KG][S::KW / 4];
    float sk[AQ_WT], had[NK][2];
    auto load = [&]() {
#pragma unroll
        for (int n = 0; n < NK; n++) {
            const int8_t * row = kc + (size_t)min(j0 + n * 8 + g, p.c.n_ctx - 1) * HD + q * S::KW;       // (slots behind the cache: its last one; no row sees them)
#pragma unroll
            for (int c = 0; c < S::KG; c++) {
                if constexpr (S::KW == 16) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(row + c * 64));
                    w[n][c][0] = u.x; w[n][c][1] = u.y; w[n][c][2] = u.z; w[n][c][3] = u.w;
                } else {
                    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(row + c * 32));
                    w[n][c][0] = u.x; w[n][c][1] = u.y;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int slot = j0 + n * 8 + 2 * q + j;
                had[n][j] = w_in && g == 0 && slot < min(s.pos, end) ? w_in[head * p.c.n_ctx + slot] : 0.f;
            }
        }
#pragma unroll
        for (int n = 0; n < AQ_WT; n++) sk[n] = __ldg(ks + (min(j0 + n * 16, p.c.n_ctx - 1) >> p.c.shift));
    };
    load();
    bool later = false;                                               // of entries that name one sequence the last one counts
    if (p.b.seq) {
        for (int j = i + 1 + lane; j < p.b.n; j += 32) {
            const SeqB o = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, j);
            later |= o.sq == s.sq && o.n_new > 0;
        }
        later = __any_sync(0xffffffffu, later);
    }
    uint32_t a[4][S::KS];
    float f = 0.f, lse = 0.f;
    int a_row = -1, sees = 0;
    if (later) return;
    while (true) {
        float sum[NK][2];
#pragma unroll
        for (int n = 0; n < NK; n++) sum[n][0] = sum[n][1] = 0.f;
        const int tok0 = max(0, j0 - s.pos);                          // the first token that sees one of these slots
        for (int r0 = tok0 * p.group / 8 * 8; r0 < n_rows; r0 += 8) {
            if (r0 != a_row) {
                const int row = r0 + g, tok = p.by_group.of(row);
                const bool there = row < n_rows;
                lse = there ? __ldcg(p.lse + (size_t)(s.first + tok) * p.n_head + hk * p.group + row - tok * p.group) : 0.f;
                f = aq_load_query<HD>(p, s, row, there, hk, q, a);
                sees = there ? aq_sees(s, p.c.n_ctx, tok) : 0;
                a_row = r0;
            }
#pragma unroll
            for (int n = 0; n < NK; n++) {
                int x[2][4];
#pragma unroll
                for (int k = 0; k < HD / 32; k++) aq_products<HD>(x, a, k, w[n][2 * k / (S::KW / 4)][2 * k % (S::KW / 4)], w[n][2 * k / (S::KW / 4)][2 * k % (S::KW / 4) + 1]);
#pragma unroll
                for (int j = 0; j < 2; j++) if (j0 + n * 8 + 2 * q + j < sees) sum[n][j] += exp2_approx(aq_score_of(x, j) * (f * sk[n >> 1]) - lse);
            }
        }
        const int at = j0;
        float before[NK][2];
#pragma unroll
        for (int n = 0; n < NK; n++) { before[n][0] = had[n][0]; before[n][1] = had[n][1]; }
        j0 += gridDim.x * AQ_WSTEP;
        const bool more = j0 < end;
        if (more) load();                                             // (on its way while these are added up)
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], o);
                const int slot = at + n * 8 + 2 * q + j;
                if (g == 0 && slot < end) w_out[head * p.c.n_ctx + slot] = before[n][j] + sum[n][j];
            }
        if (!more) return;
    }
}

// ---- how the work is cut
struct AqPlan { bool tc; int R, row_tiles, split, n_splits, items, whole, pitch; size_t words, lse, ml, part, scores; };     // rows of a tile; bytes of each piece of scratch

// CTAs run in rounds of as many as the SMs hold.  Items that fill rounds are a CTA each; those of the last round, or all where there are fewer, are split
// into ranges of at least AQ_LEAST slots.  A CTA costs as much as its slots and AQ_TURN times 64 more (on tcgen05 AQ_TURN_TC), the kernel that joins
// as AQ_TURN times 64.  Measured on both sides (us): with 1 and 3 for 4 and 10, 40 sequences of 1000 slots, 64 heads over 8 of 128, 30 for 22, 512 tokens over 4096 slots 168 for
// 132; with 12 and 30 the same, but 3 prompts of 300 tokens over 3000 slots, 32 heads over 8, 99 for 117.  AQ_ROUNDS 2 and 8: the same within 3 %.
static constexpr int AQ_LEAST = 256, AQ_TURN = 4, AQ_TURN_TC = 10, AQ_ROUNDS = 4;        // (more rounds than that: room for the parts, and nothing gained)
// Weights: scores of few rows are kept, if they take no more than this (8 sequences of 64 heads and 8000 slots, 16 MB: 28 us for reading the keys again, 6 so)
static constexpr int64_t AQ_SCORES = int64_t(256) << 20;
// ... and if there are no more than AQ_KEEP_ROWS, or their keys in all sequences are AQ_KEEP_WORK bytes: one thread adds a slot's rows one after the other, 0.4 to 0.8 us a row
// however few slots there are, where reading the keys again takes 0.04 us a row and million of bytes (one sequence of 4096 slots and 1 KV head of 96, 1680 rows: 600 us
// kept, 252 read again, 16 rows: the same; 8 sequences of 8000 slots and 8 heads of 96, 64 rows: 53 us and 125)
static constexpr int AQ_KEEP_ROWS = 16;
static constexpr int64_t AQ_KEEP_WORK = int64_t(16) << 20;
static AqPlan aq_plan(const KvQ8 & c, const RaggedB & b, int n_head, int max_kv, bool weights) {
    AqPlan r;
    const int64_t rows = (int64_t)b.max_new * (n_head / c.H);
    r.tc = attn_q8_tc_takes(c.hd, rows);
    r.R = r.tc ? AT_ROWS : rows <= 8 || c.hd > 128 ? 8 : 16;
    r.row_tiles = (int)((rows + r.R - 1) / r.R);
    const int step = r.tc ? AT_KEYS : AQ_STEP;
    const int64_t items = (int64_t)b.n * c.H * r.row_tiles, keys = max_kv < 1 ? 1 : max_kv > c.n_ctx ? c.n_ctx : max_kv;
    const int64_t slots = (int64_t)sm_count() * (r.tc ? 1 : c.hd <= 128 && r.R == 8 ? 3 : 2), rest = items % slots, units = (keys + AQ_LEAST / 4 - 1) / (AQ_LEAST / 4);
    // parts of an item of the last round: the number for which its CTAs, in rounds of their own, take the least
    const int64_t turn = r.tc ? AQ_TURN_TC : AQ_TURN;
    int64_t n = 1, least = -1;
    for (int64_t k = 1; rest && k <= 128 && (k == 1 || k * AQ_LEAST < keys + AQ_LEAST); k++) {
        const int64_t rounds = (rest * k + slots - 1) / slots, cost = rounds * ((units + k - 1) / k + turn) + (k > 1 ? AQ_TURN : 0);
        if (rounds > AQ_ROUNDS) break;
        if (least < 0 || cost < least) { least = cost; n = k; }
    }
    const int64_t per = ((keys + n - 1) / n + step - 1) / step * step;
    r.split = (int)per; r.n_splits = (int)((keys + per - 1) / per);
    r.items = (int)items;
    r.whole = (int)(r.n_splits == 1 ? items : items - rest);
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    r.lse = weights ? up((size_t)b.T * n_head * 4) : 0;
    r.ml = up((size_t)(items - r.whole) * r.n_splits * r.R * 8);
    r.part = up((size_t)(items - r.whole) * r.n_splits * r.R * c.hd * 4);
    // (a sequence may see more slots than expected: their scores need room too)
    const int64_t bytes = (int64_t)b.T * n_head * c.n_ctx * 4;
    const bool kept = weights && !r.tc && bytes <= AQ_SCORES && (rows <= AQ_KEEP_ROWS || (int64_t)b.n * c.H * keys * c.hd >= AQ_KEEP_WORK);
    r.pitch = kept ? c.n_ctx : 0;
    r.scores = kept ? up((size_t)bytes) : 0;
    r.words = r.tc || r.lse + r.ml + r.part + r.scores ? 256 : 0;     // (the status word where pi_op_status looks for it)
    return r;
}

size_t attn_q8_scratch(const KvQ8 & c, const RaggedB & b, int n_head, int max_kv, bool weights) {
    const AqPlan r = aq_plan(c, b, n_head, max_kv, weights);
    return r.words + r.lse + r.ml + r.part + r.scores;
}

template <int HD, int MT, bool TWO_Q>
static int aq_go(const AttnQ8P & p, cudaStream_t st) {
    static bool done[16] = {false};
    int dev = 0;
    PI_CUDA(cudaGetDevice(&dev));
    constexpr size_t smem = AqShape<HD>::template SMEM<MT>;
    if (dev < 0 || dev >= 16 || !done[dev]) {
        PI_CUDA(cudaFuncSetAttribute(k_attn_q8<HD, MT, TWO_Q>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 16) done[dev] = true;
    }
    PI_CUDA(launch_k(k_attn_q8<HD, MT, TWO_Q>, dim3(aq_grid(p)), dim3(AQ_THREADS), smem, st, true, p));
    return PI_OK;
}

template <int HD>
static int aq_run(const AttnQ8P & p, const AqPlan & r, const float * w_in, float * w_out, int max_kv, cudaStream_t st) {
    int rc;
    if (r.tc)                     rc = launch_attn_q8_tc(p, st);
    else if constexpr (HD <= 128) rc = r.R == 8 ? aq_go<HD, 1, true>(p, st) : p.xtype == PI_TYPE_F16 ? aq_go<HD, 2, false>(p, st) : aq_go<HD, 2, true>(p, st);
    else                          rc = aq_go<HD, 1, true>(p, st);
    if (rc) return rc;
    if (p.items > p.whole) {
        const int64_t rows = (int64_t)(p.items - p.whole) * r.R;
        if (p.n_splits <= AQ_JOIN_FEW) PI_CUDA(launch_k(k_attn_q8_join<1>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, true, p, r.R));
        else                           PI_CUDA(launch_k(k_attn_q8_join<8>, dim3((unsigned)rows), dim3(256), 0, st, true, p, r.R));
    }
    if (w_out && p.scores) {
        PI_CUDA(launch_k(k_attn_q8_weights_kept, dim3((unsigned)((p.c.n_ctx + 511) / 512), p.c.H, p.b.n), dim3(128), 0, st, true, p, w_in, w_out));
    } else if (w_out) {
        const int64_t keys = max_kv < 1 ? 1 : max_kv > p.c.n_ctx ? p.c.n_ctx : max_kv, tiles = (keys + AQ_WSTEP - 1) / AQ_WSTEP, of_sms = (int64_t)sm_count() * 8;
        const int64_t most = (of_sms + (int64_t)p.c.H * p.b.n - 1) / ((int64_t)p.c.H * p.b.n);     // CTAs of a head: two rounds of four an SM
        PI_CUDA(launch_k(k_attn_q8_weights<HD>, dim3((unsigned)(tiles < most ? tiles : most), p.c.H, p.b.n), dim3(AQ_THREADS), 0, st, true, p, w_in, w_out));
    }
    return PI_OK;
}

int launch_attention_q8(const AttnQ8Args & a, cudaStream_t st) {
    const AqPlan r = aq_plan(a.c, a.b, a.n_head, a.max_kv, a.w_out != nullptr);
    AttnQ8P p;
    p.c = a.c; p.b = a.b; p.xtype = a.xtype; p.q = a.q; p.q_stride = a.q_stride; p.n_head = a.n_head; p.group = a.n_head / a.c.H;
    p.scale_log2 = a.scale * 1.44269504088896340736f; p.out = a.out; p.out_stride = a.out_stride;
    p.split = r.split; p.n_splits = r.n_splits; p.row_tiles = r.row_tiles; p.items = r.items; p.whole = r.whole;
    p.by_group = AqDiv::by(p.group); p.by_heads = AqDiv::by(a.c.H); p.by_tiles = AqDiv::by(r.row_tiles); p.by_splits = AqDiv::by(r.n_splits);
    char * s = (char *)a.scratch;
    p.status = s ? (unsigned int *)(s + 8) : nullptr;
    s += r.words;
    p.lse = a.w_out ? (float *)s : nullptr;
    p.part_ml = (float2 *)(s + r.lse); p.part = (float *)(s + r.lse + r.ml);
    p.scores = r.scores ? (float *)(s + r.lse + r.ml + r.part) : nullptr; p.score_pitch = r.pitch;
    switch (a.c.hd) {
        case 64:  return aq_run<64>(p, r, a.w_in, a.w_out, a.max_kv, st);
        case 96:  return aq_run<96>(p, r, a.w_in, a.w_out, a.max_kv, st);
        case 128: return aq_run<128>(p, r, a.w_in, a.w_out, a.max_kv, st);
        case 192: return aq_run<192>(p, r, a.w_in, a.w_out, a.max_kv, st);
        default:  return aq_run<256>(p, r, a.w_in, a.w_out, a.max_kv, st);
    }
}

}  // namespace pi
