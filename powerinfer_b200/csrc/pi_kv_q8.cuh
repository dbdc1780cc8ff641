// What the kernels of the 8-bit KV cache share: the ragged batch, the cache's addresses, codes as halves.
#pragma once
#include "pi_common.cuh"

namespace pi {

// New tokens of n sequences: rows q_start[i] .. q_start[i + 1] - 1 of [T, ...], in slots pos0[i] and on of sequence seq[i] (null: i)
struct RaggedB {
    const int32_t * q_start; const int32_t * seq; const int32_t * pos0;
    int n, T, max_new;
};

struct KvQ8 {
    int8_t * k; int8_t * v; float * ks; float * vs;
    int n_seq, H, n_ctx, hd, block, shift;                            // block = 1 << shift slots share a scale
};

struct AttnQ8Args {
    KvQ8 c; RaggedB b;
    int xtype = 0; const void * q = nullptr; int64_t q_stride = 0; int n_head = 0;
    float scale = 0.f; void * out = nullptr; int64_t out_stride = 0; int max_kv = 0;
    const float * w_in = nullptr; float * w_out = nullptr;
    float * scratch = nullptr;                                        // attn_q8_scratch() bytes
};

struct EvictArgs {
    KvQ8 c; const int32_t * len; const int32_t * seq; int n, keep, n_sink, n_recent;
    const float * w = nullptr; float * w_out = nullptr; int32_t * kept = nullptr;
};

struct RopeExtArgs {
    int xtype; const void * x[2]; void * y[2]; int64_t x_stride[2], y_stride[2]; int heads[2];     // queries, keys
    int T, hd, n_rot, halves; const int32_t * pos; const double * freqs; float mscale;
};

int launch_rope_ext(const RopeExtArgs & a, cudaStream_t st);
int launch_kv_store_q8(const KvQ8 & c, const RaggedB & b, int xtype, const void * k, int64_t k_stride, const void * v, int64_t v_stride, cudaStream_t st);
int launch_kv_load_q8(const KvQ8 & c, const RaggedB & b, int xtype, void * k, int64_t k_stride, void * v, int64_t v_stride, cudaStream_t st);
size_t attn_q8_scratch(const KvQ8 & c, const RaggedB & b, int n_head, int max_kv, bool weights);
int launch_attention_q8(const AttnQ8Args & a, cudaStream_t st);
int launch_kv_evict_q8(const EvictArgs & a, cudaStream_t st);

#ifdef __CUDACC__

struct SeqB { int first, n_new, pos, sq; };                           // first row, tokens, slot of the first, sequence; n_new 0: nothing to do

// Entry i of the batch.  What does not fit the arrays (a start outside 0 .. T, a sequence or a slot that the cache lacks) is no token.
__device__ __forceinline__ SeqB seq_entry(const RaggedB & b, int n_seq, int n_ctx, int i) {
    SeqB s;
    s.first = b.q_start[i];
    const int end = b.q_start[i + 1];
    s.pos = b.pos0[i];
    s.sq = b.seq ? b.seq[i] : i;
    s.n_new = s.first < 0 || s.first > b.T || end <= s.first ? 0 : min(min(end, b.T) - s.first, b.max_new);      // (no difference that 32 bits do not hold)
    if (s.sq < 0 || s.sq >= n_seq || s.pos < 0 || s.pos >= n_ctx) s.sq = -1;
    return s;
}

// four codes (bytes w of one register) as two pairs of halves: 1024 + (code + 128) is the byte behind 0x64; less 1152 it is the code, exactly
__device__ __forceinline__ uint32_t q8_pair(uint32_t biased, uint32_t sel) {
    const uint32_t h = __byte_perm(biased, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t q8_lo(uint32_t biased) { return q8_pair(biased, 0x4140); }
__device__ __forceinline__ uint32_t q8_hi(uint32_t biased) { return q8_pair(biased, 0x4342); }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

#endif

}  // namespace pi
