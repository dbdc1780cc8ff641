// What the kernels of the paged cache share: its addresses, the pages of a sequence, trees of drafted tokens.
#pragma once
#include "pi_kv_q8.cuh"

namespace pi {

struct KvPaged {
    __half * k; __half * v; const int32_t * table;                    // of one layer, or of all where a kernel handles all
    int n_layer, n_pages, n_seq, max_pages, H, page, hd, shift;       // page = 1 << shift slots
    int n_ctx;                                                        // max_pages * page
};

struct AppendArgs {
    KvPaged c; RaggedB b;
    int xtype; const void * x[3]; int64_t x_stride[3]; void * q_out; int64_t q_out_stride; int n_head;      // queries, keys, values
    const int32_t * pos; const double * freqs; int n_rot, halves; float mscale;
};

struct AttnPagedArgs {
    KvPaged c; RaggedB b;
    int xtype; const void * q; int64_t q_stride; int n_head;
    const uint64_t * mask; int words; float scale; void * out; int64_t out_stride; int max_kv;
    void * scratch;                                                   // attn_paged_scratch() bytes
};

struct KeepArgs { KvPaged c; const int32_t * path; int max_path; const int32_t * n_path; const int32_t * pos0; const int32_t * seq; int n; };

static constexpr int TREE_MOST = 4096;                                // tokens of a tree

int launch_tree_mask(const RaggedB & b, const int32_t * parents, uint64_t * mask, int words, int32_t * pos, cudaStream_t st);
int launch_tree_accept(const RaggedB & b, int width, const int32_t * tokens, const int32_t * parents, const int32_t * choice, int32_t * path, int32_t * n_path, int32_t * next, cudaStream_t st);
int launch_kv_append_paged(const AppendArgs & a, cudaStream_t st);
int launch_kv_keep_paged(const KeepArgs & a, cudaStream_t st);
size_t attn_paged_scratch(const KvPaged & c, const RaggedB & b, int xtype, int n_head, int max_kv);
int launch_attention_paged(const AttnPagedArgs & a, cudaStream_t st);

#ifdef __CUDACC__

// rows of entry i: first one and how many (what does not fit the arrays is no token)
__device__ __forceinline__ int2 entry_rows(const RaggedB & b, int i) {
    const int first = b.q_start[i], end = b.q_start[i + 1];
    return make_int2(first, first < 0 || first > b.T || end <= first ? 0 : min(min(end, b.T) - first, b.max_new));
}
// page of block `block` of a sequence, -1: not there
__device__ __forceinline__ int page_of(const KvPaged & c, int sq, int block) {
    const int p = block < c.max_pages ? __ldg(c.table + (size_t)sq * c.max_pages + block) : -1;
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}
// halves from the start of a pool to the first row of a page of KV head h
__device__ __forceinline__ size_t page_at(const KvPaged & c, int page, int h) { return (((size_t)page * c.H + h) << c.shift) * c.hd; }

#endif

}  // namespace pi
