// extern "C" surface of the operators of drafted tokens over a paged cache: trees, keys and values into pages, their attention, the path that stays.
#include "pi_capi_check.cuh"
#include "pi_kv_paged.cuh"

namespace pi {

static int check_paged(const pi_kv_paged * c, KvPaged & o, const char * who) {
    PI_REQUIRE(c && c->k && c->v && c->table, "%s: null cache", who);
    PI_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->table, 4), "%s: the pools must be 16-byte aligned", who);
    PI_REQUIRE(c->head_dim == 64 || c->head_dim == 96 || c->head_dim == 128 || c->head_dim == 192 || c->head_dim == 256,
               "%s: head_dim=%d must be 64, 96, 128, 192 or 256", who, c->head_dim);
    PI_REQUIRE(c->page == 16 || c->page == 32 || c->page == 64 || c->page == 128, "%s: page=%d must be 16, 32, 64 or 128", who, c->page);
    PI_REQUIRE(c->n_layer > 0 && c->n_pages > 0 && c->n_seq > 0 && c->max_pages > 0 && c->n_head_kv > 0 && c->n_head_kv <= 65535,
               "%s: n_layer=%d, n_pages=%d, n_seq=%d, max_pages=%d, n_head_kv=%d must be positive", who, c->n_layer, c->n_pages, c->n_seq, c->max_pages, c->n_head_kv);
    PI_REQUIRE((int64_t)c->max_pages * c->page <= KV_BIG, "%s: max_pages=%d of %d slots are more than 2^30", who, c->max_pages, c->page);
    PI_REQUIRE((int64_t)c->n_pages * c->n_head_kv * c->page < (int64_t(1) << 31), "%s: a layer of %d pages is more than 2^31 rows", who, c->n_pages);
    o.k = (__half *)c->k; o.v = (__half *)c->v; o.table = c->table;
    o.n_layer = c->n_layer; o.n_pages = c->n_pages; o.n_seq = c->n_seq; o.max_pages = c->max_pages; o.H = c->n_head_kv; o.page = c->page; o.hd = c->head_dim;
    o.shift = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    o.n_ctx = c->max_pages * c->page;
    return PI_OK;
}
static int check_layer(KvPaged & c, int layer, const char * who) {
    PI_REQUIRE(layer >= 0 && layer < c.n_layer, "%s: layer=%d, the cache has %d", who, layer, c.n_layer);
    const size_t at = (size_t)layer * c.n_pages * c.H * c.page * c.hd;
    c.k += at; c.v += at;
    return PI_OK;
}
// an entry's rows alone: pos0 may be missing
static int check_rows_of(const pi_kv_batch * b, RaggedB & o, const char * who) {
    PI_REQUIRE(b, "%s: bad batch", who);
    pi_kv_batch with = *b;
    if (!with.pos0) with.pos0 = with.q_start;
    const int rc = check_batch(&with, o, who);
    if (rc) return rc;
    o.pos0 = b->pos0; o.seq = nullptr;
    PI_REQUIRE(o.max_new <= TREE_MOST, "%s: trees of up to %d tokens: at most %d are handled (max_new)", who, o.max_new, TREE_MOST);
    return PI_OK;
}

}  // namespace pi

using namespace pi;

extern "C" {
#pragma GCC visibility push(default)

int pi_tree_mask(const pi_kv_batch * batch, const int32_t * parents, uint64_t * mask, int words, int32_t * pos, void * stream) {
    RaggedB b;
    int rc;
    if ((rc = check_rows_of(batch, b, "tree_mask"))) return rc;
    PI_REQUIRE(words > 0 && words <= TREE_MOST / 64, "tree_mask: words=%d must be 1 to %d", words, TREE_MOST / 64);
    if (b.n == 0 || b.T == 0 || b.max_new == 0) return PI_OK;
    PI_REQUIRE(parents && mask && aligned(mask, 8) && (!pos || b.pos0), "tree_mask: parents and an 8-byte aligned mask are needed, and pos0 for positions");
    return launch_tree_mask(b, parents, mask, words, pos, (cudaStream_t)stream);
}

int pi_tree_accept(const pi_kv_batch * batch, const int32_t * tokens, const int32_t * parents, const int32_t * choice, int32_t * path, int32_t * n_path, int32_t * next, void * stream) {
    RaggedB b;
    int rc;
    if ((rc = check_rows_of(batch, b, "tree_accept"))) return rc;
    if (b.n == 0) return PI_OK;
    PI_REQUIRE(n_path && next && (b.max_new == 0 || (tokens && parents && choice)) && (batch->max_new == 0 || path), "tree_accept: tokens, parents, choice, path, n_path and next are needed");
    return launch_tree_accept(b, batch->max_new, tokens, parents, choice, path, n_path, next, (cudaStream_t)stream);
}

int pi_kv_append_paged(const pi_kv_paged * cache, const pi_kv_batch * batch, int layer, int xtype, const void * k, int64_t k_stride, const void * v, int64_t v_stride,
                       const void * q, int64_t q_stride, int n_head, void * q_out, int64_t q_out_stride,
                       const int32_t * pos, const double * freqs, int n_rot, int neox, float mscale, void * stream) {
    static const char * who = "kv_append_paged";
    AppendArgs a;
    int rc;
    if ((rc = check_paged(cache, a.c, who)) || (rc = check_layer(a.c, layer, who)) || (rc = check_batch(batch, a.b, who)) || (rc = check_type(xtype, who))) return rc;
    if (freqs) PI_REQUIRE(aligned(freqs, 8) && n_rot > 0 && n_rot % 2 == 0 && n_rot <= a.c.hd, "kv_append_paged: n_rot=%d must be even and within head_dim=%d", n_rot, a.c.hd);
    PI_REQUIRE(!q || (freqs && n_head > 0 && n_head <= 65535), "kv_append_paged: queries come with frequencies and n_head > 0");
    if (a.b.n == 0 || a.b.T == 0 || a.b.max_new == 0) return PI_OK;
    const int64_t width = (int64_t)a.c.H * a.c.hd, wq = (int64_t)n_head * a.c.hd, size = xtype == PI_TYPE_F16 ? 2 : 4;
    if ((rc = check_rows(k, k_stride, width, xtype, who, "k")) || (rc = check_rows(v, v_stride, width, xtype, who, "v"))) return rc;
    if (q) {
        if ((rc = check_rows(q, q_stride, wq, xtype, who, "q")) || (rc = check_rows(q_out, q_out_stride, wq, xtype, who, "q_out"))) return rc;
        PI_REQUIRE((q == q_out && q_stride == q_out_stride) || !rows_meet(q, q_stride, wq, q_out, q_out_stride, wq, a.b.T, size),
                   "kv_append_paged: q overlaps its result (in place needs the same address and stride)");
        PI_REQUIRE(!rows_meet(k, k_stride, width, q_out, q_out_stride, wq, a.b.T, size) && !rows_meet(v, v_stride, width, q_out, q_out_stride, wq, a.b.T, size),
                   "kv_append_paged: keys or values overlap q_out");
    }
    const int64_t heads = (q ? n_head : 0) + 2 * (int64_t)a.c.H;
    PI_REQUIRE((int64_t)a.b.max_new * (heads * a.c.hd / 512 + 2) < (int64_t(1) << 31) && heads * a.c.hd <= KV_BIG, "kv_append_paged: too many tokens for one call");
    a.xtype = xtype; a.x[0] = q; a.x[1] = k; a.x[2] = v; a.x_stride[0] = q_stride; a.x_stride[1] = k_stride; a.x_stride[2] = v_stride;
    a.q_out = q_out; a.q_out_stride = q_out_stride; a.n_head = n_head; a.pos = pos; a.freqs = freqs; a.n_rot = freqs ? n_rot : 0; a.halves = neox != 0; a.mscale = mscale;
    return launch_kv_append_paged(a, (cudaStream_t)stream);
}

static int check_attention_tree(const pi_kv_paged * cache, const pi_kv_batch * batch, int xtype, int n_head, KvPaged & c, RaggedB & b) {
    static const char * who = "attention_tree";
    int rc;
    if ((rc = check_paged(cache, c, who)) || (rc = check_batch(batch, b, who)) || (rc = check_type(xtype, who))) return rc;
    PI_REQUIRE(n_head > 0 && n_head % c.H == 0 && n_head <= KV_BIG / c.hd, "attention_tree: n_head=%d must be a multiple of n_head_kv=%d", n_head, c.H);
    PI_REQUIRE((int64_t)b.T * n_head < (int64_t(1) << 30) && (int64_t)b.max_new * n_head < (int64_t(1) << 27) && (int64_t)b.n * ((int64_t)b.max_new * (n_head / c.H) / 16 + 1) * c.H < (int64_t(1) << 28),
               "attention_tree: %d sequences of %d tokens of %d heads are too many for a call", b.n, b.max_new, n_head);
    return PI_OK;
}

size_t pi_attention_tree_workspace_bytes(const pi_kv_paged * cache, const pi_kv_batch * batch, int xtype, int n_head, int max_kv) {
    KvPaged c; RaggedB b;
    if (check_attention_tree(cache, batch, xtype, n_head, c, b) || b.n == 0 || b.T == 0 || b.max_new == 0) return 0;
    return attn_paged_scratch(c, b, xtype, n_head, max_kv);
}

int pi_attention_tree(const pi_kv_paged * cache, const pi_kv_batch * batch, int layer, int xtype, const void * q, int64_t q_stride, int n_head, const uint64_t * mask, int mask_words,
                      int max_kv, float scale, void * out, int64_t out_stride, void * workspace, size_t workspace_bytes, void * stream) {
    static const char * who = "attention_tree";
    AttnPagedArgs a;
    int rc;
    if ((rc = check_attention_tree(cache, batch, xtype, n_head, a.c, a.b)) || (rc = check_layer(a.c, layer, who))) return rc;
    PI_REQUIRE(!mask || (aligned(mask, 8) && mask_words > 0 && mask_words <= TREE_MOST / 64), "attention_tree: a mask is 8-byte aligned and has 1 to %d words a row", TREE_MOST / 64);
    if (a.b.n == 0 || a.b.T == 0 || a.b.max_new == 0) return PI_OK;
    const int64_t width = (int64_t)n_head * a.c.hd;
    if ((rc = check_rows(q, q_stride, width, xtype, who, "q")) || (rc = check_rows(out, out_stride, width, xtype, who, "out"))) return rc;
    PI_REQUIRE(!rows_meet(q, q_stride, width, out, out_stride, width, a.b.T, xtype == PI_TYPE_F16 ? 2 : 4), "attention_tree: q and out must be different");
    a.xtype = xtype; a.q = q; a.q_stride = q_stride; a.n_head = n_head; a.mask = mask; a.words = mask_words; a.scale = scale; a.out = out; a.out_stride = out_stride; a.max_kv = max_kv;
    const size_t need = attn_paged_scratch(a.c, a.b, xtype, n_head, max_kv);
    if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) { set_error("attention_tree: workspace too small or misaligned"); return PI_ERR_WORKSPACE; }
    a.scratch = need || (workspace && aligned(workspace, 256) && workspace_bytes >= 256) ? workspace : nullptr;       // (for the status word, where nothing else is needed)
    return launch_attention_paged(a, (cudaStream_t)stream);
}

int pi_kv_keep_paged(const pi_kv_paged * cache, const int32_t * path, int max_path, const int32_t * n_path, const int32_t * pos0, const int32_t * seq, int n, void * stream) {
    KeepArgs a;
    int rc;
    if ((rc = check_paged(cache, a.c, "kv_keep_paged"))) return rc;
    PI_REQUIRE(n >= 0 && n <= 65535 && max_path >= 0 && max_path <= KV_BIG, "kv_keep_paged: bad arguments (0 <= n <= 65535, max_path not negative)");
    PI_REQUIRE((int64_t)a.c.n_layer * 2 * a.c.H < (int64_t(1) << 31), "kv_keep_paged: too many layers");
    if (n == 0 || max_path == 0) return PI_OK;
    PI_REQUIRE(path && n_path && pos0, "kv_keep_paged: path, n_path and pos0 are needed");
    a.path = path; a.max_path = max_path; a.n_path = n_path; a.pos0 = pos0; a.seq = seq; a.n = n;
    return launch_kv_keep_paged(a, (cudaStream_t)stream);
}

#pragma GCC visibility pop
}  // extern "C"
