// Checks of arguments that the C entry points of the 8-bit and of the paged cache share.
#pragma once
#include "pi_kv_q8.cuh"

namespace pi {

static inline bool aligned(const void * p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
static const int64_t KV_BIG = int64_t(1) << 30;

static inline int check_type(int xtype, const char * who) {
    PI_REQUIRE(xtype == PI_TYPE_F32 || xtype == PI_TYPE_F16, "%s: unknown type %d of the rows", who, xtype);
    return PI_OK;
}
static inline int check_rows(const void * x, int64_t stride, int64_t width, int xtype, const char * who, const char * what) {
    const int64_t size = xtype == PI_TYPE_F16 ? 2 : 4;
    PI_REQUIRE(x && aligned(x, 16) && stride >= width && stride * size % 16 == 0 && stride <= KV_BIG,
               "%s: %s must be 16-byte aligned, rows of %lld values at least, a multiple of 16 bytes apart", who, what, (long long)width);
    return PI_OK;
}
// whether rows of two arrays (T of them, `stride` values apart, `width` wide, `size` bytes a value) share memory; columns of one wider matrix need not
static inline bool rows_meet(const void * a, int64_t sa, int64_t wa, const void * b, int64_t sb, int64_t wb, int64_t T, int64_t size) {
    if (!a || !b || T <= 0) return false;
    const int64_t a0 = (int64_t)(uintptr_t)a, b0 = (int64_t)(uintptr_t)b, a1 = a0 + ((T - 1) * sa + wa) * size, b1 = b0 + ((T - 1) * sb + wb) * size;
    if (a1 <= b0 || b1 <= a0) return false;
    if (sa != sb || T == 1) return true;
    const int64_t pitch = sa * size, at = ((b0 - a0) % pitch + pitch) % pitch;      // where b's rows begin in a's
    return at < wa * size || at + wb * size > pitch;
}
static inline int check_batch(const pi_kv_batch * b, RaggedB & o, const char * who) {
    PI_REQUIRE(b && b->T >= 0 && b->T <= KV_BIG && b->n >= 0 && b->n <= 65535 && b->max_new >= 0 && (b->n == 0 || (b->q_start && b->pos0)),
               "%s: bad batch (0 <= T <= 2^30, 0 <= n <= 65535, q_start and pos0 given)", who);
    o.q_start = b->q_start; o.seq = b->seq; o.pos0 = b->pos0; o.n = b->n; o.T = b->T; o.max_new = b->max_new < b->T ? b->max_new : b->T;
    return PI_OK;
}

}  // namespace pi
