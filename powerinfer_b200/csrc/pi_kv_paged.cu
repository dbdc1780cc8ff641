// Keys and values into the pages of a cache, keys and queries rotated on the way; and the rows of an accepted path moved up.
//
//     k_cache[slot] = fp16(R(pos) k)     v_cache[slot] = fp16(v)     q_out = R(pos) q     R as in pi_rope.cu
//
// A CTA takes up to 8 tokens, one after the other, and a share of their heads (queries, keys, values).  A thread has 16 values of one head, which it finds once; it requests those of the first token,
// and the angles of all tokens (n_rot / 2 each, once for all heads, in 64 bits) are made while they travel; then every token's are asked for before the last one's are turned and stored.  Bound by the bytes
// for many tokens (3329 of 128 FP16 heads over 8 of 64: 24 us, 5.1 TB/s; FP32 40 us), by the launch and the angles for few (150 tokens of 64 FP32 heads over 8 of 128: 6.2 us).
#include "pi_attn_q8.cuh"
#include "pi_kv_paged.cuh"
#include "pi_rope.cuh"

namespace pi {

static constexpr int AP_THREADS = 256, AP_TOKENS = 8, AP_LEAST = 896;

struct AppendP {
    AppendArgs a;
    int heads[3];                                                     // queries (0: none), keys, values
    int parts, per_head, tokens;                                      // CTAs that share a token; units of a head (of queries and keys); tokens of a CTA
    AqDiv by_unit, by_value, by_half;                                 // units of a head of queries and keys, of values; n_rot / 2
};

// 8 values of a row, as they are stored
template <typename T> struct Eight { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ void load8(const T * p, Eight<T> & e) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) e.w[i] = reinterpret_cast<const uint4 *>(p)[i];
}
__device__ __forceinline__ void open8(const Eight<float> & e, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; i++) { v[4 * i] = __uint_as_float(e.w[i].x); v[4 * i + 1] = __uint_as_float(e.w[i].y); v[4 * i + 2] = __uint_as_float(e.w[i].z); v[4 * i + 3] = __uint_as_float(e.w[i].w); }
}
__device__ __forceinline__ void open8(const Eight<__half> & e, float (&v)[8]) {
    const float2 a = h2f(e.w[0].x), b = h2f(e.w[0].y), c = h2f(e.w[0].z), d = h2f(e.w[0].w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
__device__ __forceinline__ void store8(float * p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half * p, const float (&v)[8]) {
    uint4 u; __half2 * h = reinterpret_cast<__half2 *>(&u);
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<uint4 *>(p) = u;
}

// A unit is 16 values of a head: 8 at d0 and 8 at d1.  KIND 0: pairs (2i, 2i + 1), 16 in a row; 1: pairs (i, i + half), 8 of each half, or 16 in a row of the dimensions
// that pass; 2: the same where a half is no multiple of 8, pair by pair (values still 16 in a row).  In place is fine: a unit is read and written by one thread.
template <typename T, int KIND>
__global__ void __launch_bounds__(AP_THREADS) k_kv_append(const AppendP p) {
    __shared__ float2 cs[AP_TOKENS * 128];
    __shared__ int64_t s_at[AP_TOKENS];                               // a token's row in the pools, without the head; -1: not stored
    const AppendArgs & a = p.a;
    const int group = blockIdx.x / p.parts, part = blockIdx.x - group * p.parts, i = blockIdx.y, half = a.n_rot >> 1, hd = a.c.hd, tid = threadIdx.x, t0 = group * p.tokens;
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(a.b, a.c.n_seq, a.c.n_ctx, i);
    const int nt = min(p.tokens, s.n_new - t0);
    if (nt <= 0) return;
    // ---- this thread's unit, and its values of the first token on their way
    const size_t row = (size_t)(s.first + t0);
    const int turning = (p.heads[0] + p.heads[1]) * p.per_head, units = turning + p.heads[2] * (hd >> 4), n = part * (int)blockDim.x + tid;
    const bool mine = n < units;
    const int m = n < turning ? n : n - turning, h = n < turning ? p.by_unit.of(m) : p.by_value.of(m), at = m - h * (n < turning ? p.per_head : hd >> 4);
    const int which = n >= turning ? 2 : h < p.heads[0] ? 0 : 1, head = which == 1 ? h - p.heads[0] : h;
    const bool pairs = KIND == 2 && which < 2, turns = KIND != 0 && which < 2 && at * (KIND == 2 ? 1 : 8) < half;
    const int step = pairs ? 1 : 8;                                   // values at d0 and at d1
    const int d0 = KIND == 0 || which == 2 ? at * 16 : turns ? at * step : a.n_rot + (at * step - half) * 2, d1 = turns ? d0 + half : d0 + step;
    const int64_t x_stride = mine ? a.x_stride[which] : 0;
    const T * x = mine ? (const T *)a.x[which] + row * x_stride + (size_t)head * hd : nullptr;
    Eight<T> v[2], next[2];
    T pair[2], pair_next[2];
    auto load = [&](Eight<T> (&e)[2], T (&w)[2]) {
        if (pairs) { w[0] = x[d0]; w[1] = x[d1]; }
        else       { load8(x + d0, e[0]); load8(x + d1, e[1]); }
        x += x_stride;
    };
    if (mine) load(v, pair);
    // ---- meanwhile where the tokens go, and their angles
    if (tid < 32) {
        bool later = false;
        if (a.b.seq) {                                                // of entries that name one sequence the last one counts
            for (int j = i + 1 + tid; j < a.b.n; j += 32) {
                const SeqB o = seq_entry(a.b, a.c.n_seq, a.c.n_ctx, j);
                later |= o.sq == s.sq && o.n_new > 0;
            }
            later = __any_sync(0xffffffffu, later);
        }
        if (tid < nt) {
            const int slot = s.pos + t0 + tid, page = s.sq >= 0 && slot < a.c.n_ctx && !later ? page_of(a.c, s.sq, slot >> a.c.shift) : -1;
            s_at[tid] = page < 0 ? -1 : (int64_t)page_at(a.c, page, 0) + (slot & (a.c.page - 1)) * hd;
        }
    }
    for (int j = tid; j < nt * half; j += blockDim.x) {
        const int g = p.by_half.of(j), k = j - g * half;
        cs[g * 128 + k] = rope_angle(a.pos ? a.pos[row + g] : s.pos + t0 + g, a.freqs[k], a.mscale);
    }
    __syncthreads();
    if (!mine) return;
    T * q_out = which == 0 ? (T *)a.q_out + row * a.q_out_stride + (size_t)head * hd : nullptr;
    __half * pool = (which == 1 ? a.c.k : a.c.v) + ((size_t)head << a.c.shift) * hd;
    for (int g = 0; g < nt; g++) {
        if (g + 1 < nt) load(next, pair_next);
        const float2 * c = cs + g * 128;
        const int64_t to = s_at[g];
        if (KIND == 2 && pairs) {
            float y0 = rope_get(&pair[0]), y1 = rope_get(&pair[1]);
            if (turns) {
                const float2 w = c[at];
                const float x0 = y0, x1 = y1;
                y0 = x0 * w.x - x1 * w.y; y1 = x0 * w.y + x1 * w.x;
            }
            if (which == 0)   { rope_put(q_out + d0, y0); rope_put(q_out + d1, y1); }
            else if (to >= 0) { rope_put(pool + to + d0, y0); rope_put(pool + to + d1, y1); }
        } else {
            float x0[8], x1[8];
            open8(v[0], x0);
            open8(v[1], x1);
            if (KIND == 0 && which < 2) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int k = (d0 + j) >> 1;
                    if (k < half) { const float2 w = c[k]; const float a0 = x0[j], a1 = x0[j + 1]; x0[j] = a0 * w.x - a1 * w.y; x0[j + 1] = a0 * w.y + a1 * w.x; }
                    if (k + 4 < half) { const float2 w = c[k + 4]; const float a0 = x1[j], a1 = x1[j + 1]; x1[j] = a0 * w.x - a1 * w.y; x1[j + 1] = a0 * w.y + a1 * w.x; }
                }
            } else if (turns) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float2 w = c[d0 + j];
                    const float a0 = x0[j], a1 = x1[j];
                    x0[j] = a0 * w.x - a1 * w.y; x1[j] = a0 * w.y + a1 * w.x;
                }
            }
            if (which == 0)   { store8(q_out + d0, x0); store8(q_out + d1, x1); }
            else if (to >= 0) { store8(pool + to + d0, x0); store8(pool + to + d1, x1); }
        }
        if (which == 0) q_out += a.q_out_stride;
        v[0] = next[0]; v[1] = next[1]; pair[0] = pair_next[0]; pair[1] = pair_next[1];
    }
}

// Tokens of a CTA: as many as leave AP_LEAST threads an SM, 4 at most, or 8 where the unit is a pair.  Measured with 1, 2, 4 and 8 (us): 3329 FP16 tokens of 128 heads over 8 of 64 38, 27, 24, 24, FP32 52, 41, 40, 45;
// 32 heads over 32 of 128 48, 37, 35, 36; pairs 91, 50, 33, 25; 384 tokens of the first 6.3, 5.0, 6.1, 7.2; 150 of 64 FP32 heads over 8 of 128 6.1, 8.1, 10, 11.
template <typename T>
static int append_go(const AppendArgs & a, cudaStream_t st) {
    AppendP p;
    p.a = a;
    p.heads[0] = a.x[0] ? a.n_head : 0; p.heads[1] = p.heads[2] = a.c.H;
    const int half = a.n_rot / 2, kind = !a.halves || half == 0 ? 0 : half % 8 == 0 ? 1 : 2;
    p.per_head = kind == 2 ? a.c.hd / 2 : a.c.hd / 16;
    p.by_unit = AqDiv::by(p.per_head); p.by_value = AqDiv::by(a.c.hd / 16); p.by_half = AqDiv::by(half > 0 ? half : 1);
    const int64_t units = (int64_t)(p.heads[0] + p.heads[1]) * p.per_head + (int64_t)p.heads[2] * (a.c.hd / 16);
    p.parts = (int)((units + AP_THREADS - 1) / AP_THREADS);
    const int threads = (int)((units + p.parts * 32 - 1) / (p.parts * 32) * 32);
    const int64_t all = (int64_t)a.b.n * a.b.max_new * p.parts * threads;
    p.tokens = 1;
    while (p.tokens < (kind == 2 ? AP_TOKENS : AP_TOKENS / 2) && all / (2 * p.tokens) >= (int64_t)sm_count() * AP_LEAST) p.tokens *= 2;
    const dim3 grid((unsigned)((int64_t)p.parts * ((a.b.max_new + p.tokens - 1) / p.tokens)), a.b.n), block(threads);
    if (kind == 0)      PI_CUDA(launch_k(k_kv_append<T, 0>, grid, block, 0, st, true, p));
    else if (kind == 1) PI_CUDA(launch_k(k_kv_append<T, 1>, grid, block, 0, st, true, p));
    else                PI_CUDA(launch_k(k_kv_append<T, 2>, grid, block, 0, st, true, p));
    return PI_OK;
}

int launch_kv_append_paged(const AppendArgs & a, cudaStream_t st) {
    return a.xtype == PI_TYPE_F16 ? append_go<__half>(a, st) : append_go<float>(a, st);
}

// ------------------------------------------------------------------------------------------------
// A warp takes the path's rows of one layer, of keys or values, of one KV head: KEEP_AT passes of 32 / (row's 16-byte pieces) rows are read before any of them is written.  The
// path rises, so a row is written to a place that is not behind the one it came from, and no later row comes from there.  The rows' places are found once for a CTA's warps.
// Bound by the way from the lengths over the path and the table to the rows (32 layers of 32 heads of 128, a path of 4: 3.8 us), or by rows of 256 bytes apart (80 layers of 8, 8 sequences, 6 rows each: 8 us).
static constexpr int KEEP_WARPS = 8, KEEP_ROWS = 128, KEEP_AT = 4;

__global__ void __launch_bounds__(KEEP_WARPS * 32) k_kv_keep(const KeepArgs p) {
    __shared__ uint32_t s_from[KEEP_ROWS], s_to[KEEP_ROWS];            // page * H * page size + row in it, without the head; 0xffffffff: does not move
    __shared__ int s_last[KEEP_WARPS];
    const int i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
    pdl_launch();
    pdl_wait();
    const int sq = p.seq ? p.seq[i] : i, pos = p.pos0[i];
    int n = min(p.n_path[i], p.max_path);
    if (sq < 0 || sq >= p.c.n_seq || pos < 0 || pos >= p.c.n_ctx || n <= 0) return;
    if (p.seq) {                                                      // of entries that name one sequence the last one counts
        bool later = false;
        for (int j = i + 1 + lane; j < p.n; j += 32) later |= p.seq[j] == sq && p.n_path[j] > 0;
        if (__any_sync(0xffffffffu, later)) return;                   // (the same in every warp)
    }
    const int32_t * path = p.path + (size_t)i * p.max_path;
    const int hd = p.c.hd, nv = hd >> 3, rows_at = 32 / nv, col = lane % nv, sub = lane / nv;
    const int unit = blockIdx.x * KEEP_WARPS + warp, h = unit % p.c.H, lw = unit / p.c.H, layer = lw >> 1;
    const bool mine = layer < p.c.n_layer && sub < rows_at;
    __half * pool = (lw & 1 ? p.c.v : p.c.k) + (size_t)min(layer, p.c.n_layer - 1) * p.c.n_pages * p.c.H * p.c.page * hd + (size_t)h * p.c.page * hd + col * 8;
    for (int r0 = 0; r0 < n; r0 += KEEP_ROWS) {
        // rows of this pass that do not rise end the path
        const int r = r0 + tid;
        int end = n;
        if (tid < KEEP_ROWS && r < n) {
            const int at = path[r];
            if (at < 0 || (r > 0 && at <= path[r - 1])) end = r;
            uint32_t from = 0xffffffffu, to = 0xffffffffu;
            if (at > r && at < p.c.n_ctx - pos) {
                const int a = page_of(p.c, sq, (pos + at) >> p.c.shift), b = page_of(p.c, sq, (pos + r) >> p.c.shift);
                if (a >= 0 && b >= 0) {
                    from = ((uint32_t)a * p.c.H << p.c.shift) + ((pos + at) & (p.c.page - 1));
                    to = ((uint32_t)b * p.c.H << p.c.shift) + ((pos + r) & (p.c.page - 1));
                }
            }
            s_from[tid] = from; s_to[tid] = to;
        }
        end = __reduce_min_sync(0xffffffffu, end);
        if (lane == 0) s_last[warp] = end;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < KEEP_WARPS; w++) n = min(n, s_last[w]);
        const int rows = min(KEEP_ROWS, n - r0);
        for (int k0 = 0; k0 < rows; k0 += KEEP_AT * rows_at) {
            uint4 x[KEEP_AT]; uint32_t to[KEEP_AT];
#pragma unroll
            for (int u = 0; u < KEEP_AT; u++) {
                const int k = k0 + u * rows_at + sub;
                to[u] = 0xffffffffu;
                if (mine && k < rows) {
                    to[u] = s_to[k];
                    if (to[u] != 0xffffffffu) x[u] = *reinterpret_cast<const uint4 *>(pool + (size_t)s_from[k] * hd);
                }
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < KEEP_AT; u++) if (to[u] != 0xffffffffu) *reinterpret_cast<uint4 *>(pool + (size_t)to[u] * hd) = x[u];
            __syncwarp();
        }
        __syncthreads();
    }
}

int launch_kv_keep_paged(const KeepArgs & a, cudaStream_t st) {
    const int64_t units = (int64_t)a.c.n_layer * 2 * a.c.H;
    PI_CUDA(launch_k(k_kv_keep, dim3((unsigned)((units + KEEP_WARPS - 1) / KEEP_WARPS), a.n), dim3(KEEP_WARPS * 32), 0, st, true, a));
    return PI_OK;
}

}  // namespace pi
