// What the two kernels of the attention over the 8-bit cache share: their arguments, which rows a tile has and what they see.
#pragma once
#include "pi_kv_q8.cuh"

namespace pi {

// n / d for n < 2^31 by a product (a division is 20 instructions, and what a CTA does before its first slot is waited for)
struct AqDiv {
    unsigned mul, shift;
    __host__ static AqDiv by(int d) {
        AqDiv r{0, 0};
        while ((1ll << r.shift) < d) r.shift++;
        r.mul = (unsigned)((1ull << 32) * ((1ull << r.shift) - (unsigned)d) / (unsigned)d + 1);
        return r;
    }
    __device__ __forceinline__ int of(int n) const { return (int)((__umulhi((unsigned)n, mul) + (unsigned)n) >> shift); }
};

struct AttnQ8P {
    KvQ8 c; RaggedB b;
    int xtype; const void * q; int64_t q_stride; int n_head, group;
    float scale_log2; void * out; int64_t out_stride;
    // An item is a tile of rows of a KV head of an entry.  The first `whole` items are a CTA each, the others n_splits: ranges of `split` slots.
    int split, n_splits, row_tiles, items, whole;
    AqDiv by_group, by_heads, by_tiles, by_splits;                    // the KV heads' number, row_tiles, n_splits
    float * part; float2 * part_ml; float * lse;                      // [split item][split][R][hd], (max, sum) beside them; log2 of the rows' normalisers [T][n_head]
    float * scores; int score_pitch;                                  // (null: not kept) the rows' scores in bits, [T * n_head][pitch]
    unsigned int * status;                                            // (null: no workspace) tcgen05 alone: bit 4, a wait ran out; others clear it
};

struct AqItem { int item, entry, hk, rt, split, n_splits; };
__device__ __forceinline__ AqItem aq_item(const AttnQ8P & p, int cta) {
    AqItem w;
    const int k = cta - p.whole;
    w.n_splits = k < 0 ? 1 : p.n_splits;
    w.item = k < 0 ? cta : p.whole + p.by_splits.of(k);
    w.split = k < 0 ? 0 : k - (w.item - p.whole) * p.n_splits;
    const int of_head = p.by_tiles.of(w.item);
    w.rt = w.item - of_head * p.row_tiles;
    w.entry = p.by_heads.of(of_head);
    w.hk = of_head - w.entry * p.c.H;
    return w;
}
static inline unsigned aq_grid(const AttnQ8P & p) { return (unsigned)(p.whole + (int64_t)(p.items - p.whole) * p.n_splits); }

// rows of the tile, as (token, head): row r of the group's tokens is token r / group, head r % group
struct TileB { int n_rows, first, seen; };                            // rows there are, first row's number, slots that the last row sees (0: none)

__device__ __forceinline__ int aq_sees(const SeqB & s, int n_ctx, int tok) {          // slots that token tok sees
    const int slot = s.pos + tok;
    return s.sq < 0 || slot >= n_ctx ? 0 : slot + 1;
}
__device__ __forceinline__ TileB aq_tile(const AttnQ8P & p, const SeqB & s, int rt, int R) {
    TileB t;
    t.first = rt * R;
    t.n_rows = min(R, s.n_new * p.group - t.first);
    t.seen = 0;
    if (t.n_rows > 0 && s.sq >= 0) {                                  // the last of its rows whose slot there is
        const int last = min(p.by_group.of(t.first + t.n_rows - 1), p.c.n_ctx - 1 - s.pos);
        if (last >= p.by_group.of(t.first)) t.seen = s.pos + last + 1;
    }
    return t;
}
__device__ __forceinline__ void aq_put(int xtype, void * out, size_t at, float v) {
    if (xtype == PI_TYPE_F16) ((__half *)out)[at] = __float2half_rn(v); else ((float *)out)[at] = v;
}
// four values of a query row from column d
__device__ __forceinline__ float4 aq_query(int xtype, const void * q, size_t at) {
    if (xtype == PI_TYPE_F16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>((const __half *)q + at));
        const float2 a = h2f(u.x), b = h2f(u.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return __ldg(reinterpret_cast<const float4 *>((const float *)q + at));
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
// x, y as the sum of two pairs of halves
__device__ __forceinline__ void aq_split(float x, float y, uint32_t & hi, uint32_t & lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2u(h);
    lo = h2u(__floats2half2_rn(x - f.x, y - f.y));
}

// 64 and more rows a KV head on tcgen05 (pi_attn_q8_tc.cu): tiles of AT_ROWS rows, splits a multiple of AT_KEYS slots
static constexpr int AT_ROWS = 128, AT_KEYS = 128;
bool attn_q8_tc_takes(int hd, int64_t rows);
int launch_attn_q8_tc(const AttnQ8P & p, cudaStream_t st);

}  // namespace pi
