// What the kernels of the attention over a paged cache share: their arguments, which rows a tile has and what they see.
#pragma once
#include "pi_attn_q8.cuh"
#include "pi_kv_paged.cuh"

namespace pi {

struct AttnPagedP {
    KvPaged c; RaggedB b;
    int xtype; const void * q; int64_t q_stride; int n_head, group;
    const uint64_t * mask; int words;
    float scale_log2; void * out; int64_t out_stride;
    // An item is a tile of rows of a KV head of an entry.  The first `whole` items are a CTA each, the others n_splits: ranges of `split` slots.
    int split, n_splits, row_tiles, items, whole;
    AqDiv by_group, by_heads, by_tiles, by_splits;                    // the KV heads' number, row_tiles, n_splits
    __half * queries; float * factor;                                 // tcgen05 alone: the queries as halves, the factors of their scores
    float * part; float2 * part_ml;                                   // [split item][split][R][hd], (max, sum) beside them
    unsigned int * status;                                            // (null: no workspace) tcgen05 alone: bit 4, a wait ran out; others clear it
};

__device__ __forceinline__ AqItem ap_item(const AttnPagedP & p, int cta) {
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
static inline unsigned ap_grid(const AttnPagedP & p) { return (unsigned)(p.whole + (int64_t)(p.items - p.whole) * p.n_splits); }

// Rows of the tile, as (token, head): row r of the group's tokens is token r / group, head r % group.
struct TileP { int n_rows, first, seen, there; };                     // rows there are, first row's number, end of the slots that any row sees, of those that the entry has

__device__ __forceinline__ TileP ap_tile(const AttnPagedP & p, const SeqB & s, int rt, int R) {
    TileP t;
    t.first = rt * R;
    t.n_rows = min(R, s.n_new * p.group - t.first);
    t.seen = t.there = 0;
    if (t.n_rows > 0 && s.sq >= 0) {
        const int n_new = min(s.n_new, p.c.n_ctx - s.pos);            // of the new tokens those that have a slot
        t.there = s.pos + n_new;
        if (p.by_group.of(t.first) < n_new) t.seen = p.mask ? t.there : s.pos + min(p.by_group.of(t.first + t.n_rows - 1) + 1, n_new);
    }
    return t;
}
__device__ __forceinline__ uint32_t ap_ones(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Which of the 32 slots from pos + u0 on token `tok` of the entry sees (u0 may be negative: the context), pages aside
__device__ __forceinline__ uint32_t ap_sees(const AttnPagedP & p, const SeqB & s, int tok, int u0) {
    const int n_new = min(s.n_new, p.c.n_ctx - s.pos);
    if (s.sq < 0 || tok >= n_new) return 0u;
    const uint32_t there = ap_ones((p.mask ? n_new : tok + 1) - u0);
    if (!p.mask || u0 <= -32) return there;
    const uint64_t * row = p.mask + (size_t)(s.first + tok) * p.words;
    const int lo = max(u0, 0), w = lo >> 6, sh = lo & 63;
    uint64_t x = w < p.words ? __ldg(row + w) >> sh : 0;
    if (sh > 32 && w + 1 < p.words) x |= __ldg(row + w + 1) << (64 - sh);
    return there & (u0 < 0 ? (uint32_t)x << -u0 | ap_ones(-u0) : (uint32_t)x);
}

// The same for 128 slots; `word`: the first two words of the token's mask
__device__ __forceinline__ void ap_sees128(const AttnPagedP & p, const SeqB & s, int tok, int u0, const uint64_t (&word)[2], uint32_t (&sees)[4]) {
    const int n_new = min(s.n_new, p.c.n_ctx - s.pos);
    const bool none = s.sq < 0 || tok >= n_new;
    const int end = none ? -0x40000000 : (p.mask ? n_new : tok + 1) - u0;
    const int lo = max(u0, 0), w = lo >> 6, sh = lo & 63;
    uint64_t x[3] = {w == 0 ? word[0] : w == 1 ? word[1] : 0, w == 0 ? word[1] : 0, 0};
    if (p.words > 2 && p.mask && !none) {
        const uint64_t * row = p.mask + (size_t)(s.first + tok) * p.words;
#pragma unroll
        for (int i = 0; i < 3; i++) x[i] = w + i < p.words ? __ldg(row + w + i) : 0;
    }
    // bits from lo on, then ones in front of them for the slots before the new ones
    uint64_t a = x[0] >> sh | (sh ? x[1] << (64 - sh) : 0), b = x[1] >> sh | (sh ? x[2] << (64 - sh) : 0);
    const int before = min(max(-u0, 0), 128);
    if (before >= 128)     { a = b = ~0ull; }
    else if (before >= 64) { b = a << (before - 64) | ((1ull << (before - 64)) - 1); a = ~0ull; }
    else if (before > 0)   { b = b << before | a >> (64 - before); a = a << before | ((1ull << before) - 1); }
    if (!p.mask) a = b = ~0ull;
    sees[0] = (uint32_t)a & ap_ones(end); sees[1] = (uint32_t)(a >> 32) & ap_ones(end - 32); sees[2] = (uint32_t)b & ap_ones(end - 64); sees[3] = (uint32_t)(b >> 32) & ap_ones(end - 96);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Many rows of a KV head on tcgen05 (pi_attn_paged_tc.cu): tiles of PT_ROWS rows, splits a multiple of PT_KEYS slots
static constexpr int PT_ROWS = 128, PT_KEYS = 128;
bool attn_paged_tc_takes(int64_t rows, double values);             // rows of a KV head, values of all keys

int launch_attn_paged_tc(const AttnPagedP & p, cudaStream_t st);

}  // namespace pi
