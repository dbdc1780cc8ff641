// extern "C" surface of the operators of a long context: rotary positions, the KV cache in 8 bits, its attention and eviction.
#include "pi_kv_q8.cuh"

#include <cmath>

namespace pi {

static bool aligned(const void * p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
static const int64_t KV_BIG = int64_t(1) << 30;

static int check_cache(const pi_kv_q8 * c, KvQ8 & o, const char * who) {
    PI_REQUIRE(c && c->k && c->v && c->k_scale && c->v_scale, "%s: null cache", who);
    PI_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->k_scale, 4) && aligned(c->v_scale, 4), "%s: the caches must be 16-byte aligned", who);
    PI_REQUIRE(c->head_dim == 64 || c->head_dim == 96 || c->head_dim == 128 || c->head_dim == 192 || c->head_dim == 256,
               "%s: head_dim=%d must be 64, 96, 128, 192 or 256", who, c->head_dim);
    PI_REQUIRE(c->block == 16 || c->block == 32 || c->block == 64 || c->block == 128, "%s: block=%d must be 16, 32, 64 or 128", who, c->block);
    PI_REQUIRE(c->n_seq > 0 && c->n_head_kv > 0 && c->n_head_kv <= 65535 && c->n_ctx > 0 && c->n_ctx % c->block == 0 && c->n_ctx <= KV_BIG,
               "%s: n_seq=%d, n_head_kv=%d, n_ctx=%d: positive, n_ctx a multiple of block=%d", who, c->n_seq, c->n_head_kv, c->n_ctx, c->block);
    o.k = (int8_t *)c->k; o.v = (int8_t *)c->v; o.ks = c->k_scale; o.vs = c->v_scale;
    o.n_seq = c->n_seq; o.H = c->n_head_kv; o.n_ctx = c->n_ctx; o.hd = c->head_dim; o.block = c->block;
    o.shift = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
    return PI_OK;
}
static int check_type(int xtype, const char * who) {
    PI_REQUIRE(xtype == PI_TYPE_F32 || xtype == PI_TYPE_F16, "%s: unknown type %d of the rows", who, xtype);
    return PI_OK;
}
static int check_rows(const void * x, int64_t stride, int64_t width, int xtype, const char * who, const char * what) {
    const int64_t size = xtype == PI_TYPE_F16 ? 2 : 4;
    PI_REQUIRE(x && aligned(x, 16) && stride >= width && stride * size % 16 == 0 && stride <= KV_BIG,
               "%s: %s must be 16-byte aligned, rows of %lld values at least, a multiple of 16 bytes apart", who, what, (long long)width);
    return PI_OK;
}
// whether rows of two arrays (T of them, `stride` values apart, `width` wide, `size` bytes a value) share memory; columns of one wider matrix need not
static bool rows_meet(const void * a, int64_t sa, int64_t wa, const void * b, int64_t sb, int64_t wb, int64_t T, int64_t size) {
    if (!a || !b || T <= 0) return false;
    const int64_t a0 = (int64_t)(uintptr_t)a, b0 = (int64_t)(uintptr_t)b, a1 = a0 + ((T - 1) * sa + wa) * size, b1 = b0 + ((T - 1) * sb + wb) * size;
    if (a1 <= b0 || b1 <= a0) return false;
    if (sa != sb || T == 1) return true;
    const int64_t pitch = sa * size, at = ((b0 - a0) % pitch + pitch) % pitch;      // where b's rows begin in a's
    return at < wa * size || at + wb * size > pitch;
}
// whether two arrays of n values of four bytes are one and the same, or apart
static bool same_or_apart(const void * a, const void * b, int64_t n) {
    const int64_t a0 = (int64_t)(uintptr_t)a, b0 = (int64_t)(uintptr_t)b;
    return !a || !b || a == b || a0 + 4 * n <= b0 || b0 + 4 * n <= a0;
}
static int check_batch(const pi_kv_batch * b, RaggedB & o, const char * who) {
    PI_REQUIRE(b && b->T >= 0 && b->T <= KV_BIG && b->n >= 0 && b->n <= 65535 && b->max_new >= 0 && (b->n == 0 || (b->q_start && b->pos0)),
               "%s: bad batch (0 <= T <= 2^30, 0 <= n <= 65535, q_start and pos0 given)", who);
    o.q_start = b->q_start; o.seq = b->seq; o.pos0 = b->pos0; o.n = b->n; o.T = b->T; o.max_new = b->max_new < b->T ? b->max_new : b->T;
    return PI_OK;
}

}  // namespace pi

using namespace pi;

extern "C" {
#pragma GCC visibility push(default)

int pi_rope_freqs_host(double * host_freqs, float * host_mscale, int n_rot, float freq_base, float freq_scale, float ext_factor, float attn_factor,
                       float beta_fast, float beta_slow, int n_orig_ctx, const float * host_freq_factors) {
    PI_REQUIRE(host_freqs && host_mscale && n_rot > 0 && n_rot % 2 == 0 && n_rot <= 256 && freq_base > 1.f && freq_scale > 0.f,
               "rope_freqs: n_rot=%d must be even and at most 256, freq_base > 1, freq_scale > 0", n_rot);
    PI_REQUIRE(ext_factor == 0.f || (n_orig_ctx > 0 && beta_fast > 0.f && beta_slow > 0.f), "rope_freqs: ext_factor needs n_orig_ctx, beta_fast and beta_slow");
    const double two_pi = 6.283185307179586476925, base = freq_base, s = freq_scale;
    double lo = 0, hi = 0;
    if (ext_factor != 0.f) {                                          // pairs that make beta turns within the original context
        auto pair = [&](double turns) { return n_rot * log(n_orig_ctx / (turns * two_pi)) / (2 * log(base)); };
        lo = fmax(0.0, floor(pair(beta_fast)));
        hi = fmin(n_rot - 1.0, ceil(pair(beta_slow)));
    }
    for (int i = 0; i < n_rot / 2; i++) {
        const double f = pow(base, -2.0 * i / n_rot) / (host_freq_factors ? (double)host_freq_factors[i] : 1.0);
        double mix = 0;                                               // share of the unscaled angle
        if (ext_factor != 0.f) mix = (1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(0.001, hi - lo)))) * ext_factor;
        host_freqs[i] = f * s * (1.0 - mix) + f * mix;
    }
    *host_mscale = (float)(attn_factor * (ext_factor != 0.f ? 1.0 + 0.1 * log(1.0 / s) : 1.0));
    return PI_OK;
}

int pi_rope_ext(int xtype, const void * q, int64_t q_stride, int n_head, void * q_out, int64_t q_out_stride,
                const void * k, int64_t k_stride, int n_head_kv, void * k_out, int64_t k_out_stride,
                int T, int head_dim, int n_rot, int neox, const int32_t * pos, const double * freqs, float mscale, void * stream) {
    int rc;
    if ((rc = check_type(xtype, "rope_ext"))) return rc;
    PI_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256 && n_rot > 0 && n_rot % 2 == 0 && n_rot <= head_dim,
               "rope_ext: head_dim=%d must be a multiple of 8 up to 256, n_rot=%d even and within it", head_dim, n_rot);
    PI_REQUIRE(T >= 0 && T <= KV_BIG && n_head > 0 && n_head_kv >= 0 && n_head <= 65535 && n_head_kv <= 65535 && (n_head_kv == 0) == (k == nullptr),
               "rope_ext: bad arguments (keys come with n_head_kv > 0, or neither)");
    if (T == 0) return PI_OK;
    PI_REQUIRE(pos && freqs && aligned(freqs, 8), "rope_ext: positions and frequencies are needed");
    const int64_t size = xtype == PI_TYPE_F16 ? 2 : 4;
    RopeExtArgs a;
    const void * x[2] = {q, k}; void * y[2] = {q_out, k_out};
    const int64_t xs[2] = {q_stride, k_stride}, ys[2] = {q_out_stride, k_out_stride};
    a.heads[0] = n_head; a.heads[1] = n_head_kv;
    for (int i = 0; i < 2; i++) {
        a.x[i] = x[i]; a.y[i] = y[i]; a.x_stride[i] = xs[i]; a.y_stride[i] = ys[i];
        if (a.heads[i] == 0) continue;
        const int64_t width = (int64_t)a.heads[i] * head_dim;
        if ((rc = check_rows(x[i], xs[i], width, xtype, "rope_ext", i ? "k" : "q"))) return rc;
        if ((rc = check_rows(y[i], ys[i], width, xtype, "rope_ext", i ? "k_out" : "q_out"))) return rc;
        // in place, or apart: rows that overlap otherwise would be read after they were written
        const bool in_place = x[i] == y[i] && xs[i] == ys[i];
        PI_REQUIRE(in_place || !rows_meet(x[i], xs[i], width, y[i], ys[i], width, T, size), "rope_ext: %s overlaps its result (in place needs the same address and stride)", i ? "k" : "q");
    }
    const int64_t wq = (int64_t)n_head * head_dim, wk = (int64_t)n_head_kv * head_dim;
    PI_REQUIRE(!k || (!rows_meet(q, q_stride, wq, k_out, k_out_stride, wk, T, size) && !rows_meet(k, k_stride, wk, q_out, q_out_stride, wq, T, size) &&
                      !rows_meet(q_out, q_out_stride, wq, k_out, k_out_stride, wk, T, size)), "rope_ext: queries and keys overlap each other's results");
    a.xtype = xtype; a.T = T; a.hd = head_dim; a.n_rot = n_rot; a.halves = neox != 0; a.pos = pos; a.freqs = freqs; a.mscale = mscale;
    PI_REQUIRE((int64_t)T * ((int64_t)(n_head + n_head_kv) * head_dim / 1024 + 1) < (int64_t(1) << 31), "rope_ext: too many tokens for one call");
    return launch_rope_ext(a, (cudaStream_t)stream);
}

int pi_kv_store_q8(const pi_kv_q8 * cache, const pi_kv_batch * batch, int xtype, const void * k, int64_t k_stride, const void * v, int64_t v_stride, void * stream) {
    KvQ8 c; RaggedB b;
    int rc;
    if ((rc = check_cache(cache, c, "kv_store_q8")) || (rc = check_batch(batch, b, "kv_store_q8")) || (rc = check_type(xtype, "kv_store_q8"))) return rc;
    if (b.n == 0 || b.T == 0 || b.max_new == 0) return PI_OK;
    const int64_t width = (int64_t)c.H * c.hd;
    if ((rc = check_rows(k, k_stride, width, xtype, "kv_store_q8", "k")) || (rc = check_rows(v, v_stride, width, xtype, "kv_store_q8", "v"))) return rc;
    PI_REQUIRE(((int64_t)(b.max_new < c.n_ctx ? b.max_new : c.n_ctx) / c.block + 2) * 2 * c.H < (int64_t(1) << 31), "kv_store_q8: too many slots for one call");
    return launch_kv_store_q8(c, b, xtype, k, k_stride, v, v_stride, (cudaStream_t)stream);
}

int pi_kv_load_q8(const pi_kv_q8 * cache, const pi_kv_batch * batch, int xtype, void * k, int64_t k_stride, void * v, int64_t v_stride, void * stream) {
    KvQ8 c; RaggedB b;
    int rc;
    if ((rc = check_cache(cache, c, "kv_load_q8")) || (rc = check_batch(batch, b, "kv_load_q8")) || (rc = check_type(xtype, "kv_load_q8"))) return rc;
    if (b.n == 0 || b.T == 0 || b.max_new == 0) return PI_OK;
    const int64_t width = (int64_t)c.H * c.hd;
    PI_REQUIRE((int64_t)(b.max_new / 16 + 1) * c.H < (int64_t(1) << 30), "kv_load_q8: too many slots for one call");
    if ((rc = check_rows(k, k_stride, width, xtype, "kv_load_q8", "k")) || (rc = check_rows(v, v_stride, width, xtype, "kv_load_q8", "v"))) return rc;
    PI_REQUIRE(!rows_meet(k, k_stride, width, v, v_stride, width, b.T, xtype == PI_TYPE_F16 ? 2 : 4), "kv_load_q8: k and v overlap");
    return launch_kv_load_q8(c, b, xtype, k, k_stride, v, v_stride, (cudaStream_t)stream);
}

static int check_attention(const pi_kv_q8 * cache, const pi_kv_batch * batch, int n_head, KvQ8 & c, RaggedB & b) {
    int rc;
    if ((rc = check_cache(cache, c, "attention_q8")) || (rc = check_batch(batch, b, "attention_q8"))) return rc;
    PI_REQUIRE(n_head > 0 && n_head % c.H == 0 && n_head <= KV_BIG / c.hd, "attention_q8: n_head=%d must be a multiple of n_head_kv=%d", n_head, c.H);
    PI_REQUIRE((int64_t)b.max_new * n_head < (int64_t(1) << 27) && (int64_t)b.n * ((int64_t)b.max_new * (n_head / c.H) / 8 + 1) * c.H < (int64_t(1) << 28),
               "attention_q8: %d sequences of %d tokens of %d heads are too many for a call", b.n, b.max_new, n_head);
    return PI_OK;
}

size_t pi_attention_q8_workspace_bytes(const pi_kv_q8 * cache, const pi_kv_batch * batch, int n_head, int max_kv, int weights) {
    KvQ8 c; RaggedB b;
    if (check_attention(cache, batch, n_head, c, b) || b.n == 0 || b.T == 0 || b.max_new == 0) return 0;
    return attn_q8_scratch(c, b, n_head, max_kv, weights != 0);
}

int pi_attention_q8(const pi_kv_q8 * cache, const pi_kv_batch * batch, int xtype, const void * q, int64_t q_stride, int n_head, int max_kv, float scale,
                    void * out, int64_t out_stride, const float * weights_in, float * weights_out,
                    void * workspace, size_t workspace_bytes, void * stream) {
    KvQ8 c; RaggedB b;
    int rc;
    if ((rc = check_attention(cache, batch, n_head, c, b)) || (rc = check_type(xtype, "attention_q8"))) return rc;
    if (b.n == 0 || b.T == 0 || b.max_new == 0) return PI_OK;
    const int64_t width = (int64_t)n_head * c.hd;
    if ((rc = check_rows(q, q_stride, width, xtype, "attention_q8", "q")) || (rc = check_rows(out, out_stride, width, xtype, "attention_q8", "out"))) return rc;
    PI_REQUIRE(!rows_meet(q, q_stride, width, out, out_stride, width, b.T, xtype == PI_TYPE_F16 ? 2 : 4), "attention_q8: q and out must be different");
    PI_REQUIRE(!weights_in || weights_out, "attention_q8: weights_in without weights_out");
    PI_REQUIRE(same_or_apart(weights_in, weights_out, (int64_t)c.n_seq * c.H * c.n_ctx), "attention_q8: weights_in and weights_out overlap (the same array, or apart)");
    AttnQ8Args a;
    a.c = c; a.b = b; a.xtype = xtype; a.q = q; a.q_stride = q_stride; a.n_head = n_head; a.max_kv = max_kv;
    a.scale = scale; a.out = out; a.out_stride = out_stride; a.w_in = weights_in; a.w_out = weights_out;
    const size_t need = attn_q8_scratch(c, b, n_head, max_kv, weights_out != nullptr);
    if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) { set_error("attention_q8: workspace too small or misaligned"); return PI_ERR_WORKSPACE; }
    a.scratch = need || (workspace && aligned(workspace, 256) && workspace_bytes >= 256) ? (float *)workspace : nullptr;       // (for the status word, where nothing else is needed)
    return launch_attention_q8(a, (cudaStream_t)stream);
}

int pi_kv_evict_q8(const pi_kv_q8 * cache, const int32_t * len, const int32_t * seq, int n, int keep, int n_sink, int n_recent,
                   const float * weights, float * weights_out, int32_t * kept, void * stream) {
    EvictArgs a;
    int rc;
    if ((rc = check_cache(cache, a.c, "kv_evict_q8"))) return rc;
    PI_REQUIRE(n >= 0 && n <= 65535 && n_sink >= 0 && n_recent >= 0, "kv_evict_q8: bad arguments");
    PI_REQUIRE(keep > 0 && keep % a.c.block == 0 && keep <= a.c.n_ctx, "kv_evict_q8: keep=%d must be a multiple of block=%d, at most n_ctx", keep, a.c.block);
    PI_REQUIRE((int64_t)n_sink + n_recent <= keep, "kv_evict_q8: n_sink=%d and n_recent=%d are more than keep=%d", n_sink, n_recent, keep);
    PI_REQUIRE(a.c.n_ctx <= 1 << 18, "kv_evict_q8: n_ctx=%d is more than 262144", a.c.n_ctx);
    if (n == 0) return PI_OK;
    PI_REQUIRE(len && weights && kept, "kv_evict_q8: len, weights and kept are needed");
    PI_REQUIRE(same_or_apart(weights, weights_out, (int64_t)a.c.n_seq * a.c.H * a.c.n_ctx), "kv_evict_q8: weights and weights_out overlap (the same array, or apart)");
    a.len = len; a.seq = seq; a.n = n; a.keep = keep; a.n_sink = n_sink; a.n_recent = n_recent; a.w = weights; a.w_out = weights_out; a.kept = kept;
    return launch_kv_evict_q8(a, (cudaStream_t)stream);
}

#pragma GCC visibility pop
}  // extern "C"
