// Keys and values into the pages of a cache, keys and queries rotated on the way; and the rows of an accepted path moved up.
//
//     k_cache[slot] = fp16(R(pos) k)     v_cache[slot] = fp16(v)     q_out = R(pos) q     R as in pi_rope.cu
//
// A CTA takes one token and a share of its heads (queries, keys, values): every thread requests its values first, the angles of the token are made while they
// travel (n_rot / 2 of them, once for all heads, in 64 bits).  Bound by the bytes for many tokens (3329 of 128 FP16 heads over 8 of 64: 28 us, 4.4 TB/s; 256 threads of a token, with its angles in 64 bits
// in front of the products), by the launch and the angles for few (150 tokens of 64 FP32 heads over 8 of 128: 6.5 us).
#include "pi_kv_paged.cuh"
#include "pi_rope.cuh"

namespace pi {

static constexpr int AP_THREADS = 256;

struct AppendP {
    AppendArgs a;
    int heads[3];                                                     // queries (0: none), keys, values
    int parts, per_head;                                              // CTAs of a token; units of a head (of queries and keys)
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
template <typename T, int KIND, int U>
__global__ void __launch_bounds__(AP_THREADS) k_kv_append(const AppendP p) {
    __shared__ float2 cs[128];
    const AppendArgs & a = p.a;
    const int t = blockIdx.x / p.parts, part = blockIdx.x - t * p.parts, i = blockIdx.y, half = a.n_rot >> 1, hd = a.c.hd, lane = threadIdx.x & 31;
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(a.b, a.c.n_seq, a.c.n_ctx, i);
    if (t >= s.n_new) return;
    const int slot = s.pos + t;
    const size_t row_in = (size_t)(s.first + t);
    // ---- values on their way
    const int turning = (p.heads[0] + p.heads[1]) * p.per_head, units = turning + p.heads[2] * (hd >> 4);
    Eight<T> v[U][KIND == 2 ? 1 : 2]; T pair[KIND == 2 ? U : 1][2]; int which[U], at[U], head[U];
    (void)pair;
    // first and second 8 of unit `at`: of queries and keys, of values
    auto places = [&](int which, int at, bool & turns, int & d0, int & d1) {
        turns = KIND == 1 && which < 2 && at * 8 < half;
        d0 = KIND != 1 || which == 2 ? at * 16 : turns ? at * 8 : a.n_rot + (at * 8 - half) * 2;
        d1 = turns ? d0 + half : d0 + 8;
    };
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int n = (part * U + u) * (int)blockDim.x + (int)threadIdx.x;
        which[u] = -1;
        if (n >= units) continue;
        const int per = n < turning ? p.per_head : hd >> 4, m = n < turning ? n : n - turning;
        int h = m / per;
        at[u] = m - h * per;
        which[u] = n >= turning ? 2 : h < p.heads[0] ? 0 : 1;
        if (which[u] == 1) h -= p.heads[0];
        head[u] = h;
        const T * x = (const T *)a.x[which[u]] + row_in * a.x_stride[which[u]] + (size_t)h * hd;
        if constexpr (KIND == 2) {
            if (which[u] < 2) {
                const int d0 = at[u] < half ? at[u] : a.n_rot + (at[u] - half) * 2, d1 = at[u] < half ? d0 + half : d0 + 1;
                pair[u][0] = x[d0]; pair[u][1] = x[d1];
            }
        } else {
            bool turns; int d0, d1;
            places(which[u], at[u], turns, d0, d1);
            load8(x + d0, v[u][0]);
            load8(x + d1, v[u][KIND == 2 ? 0 : 1]);
        }
    }
    // ---- meanwhile where they go, and the angles
    int page = -1;
    if (s.sq >= 0 && slot < a.c.n_ctx) page = page_of(a.c, s.sq, slot >> a.c.shift);
    const int pos = a.pos ? a.pos[row_in] : slot;
    for (int j = threadIdx.x; j < half; j += blockDim.x) cs[j] = rope_angle(pos, a.freqs[j], a.mscale);
    if (a.b.seq && page >= 0) {                                       // of entries that name one sequence the last one counts
        bool later = false;
        for (int j = i + 1 + lane; j < a.b.n; j += 32) {
            const SeqB o = seq_entry(a.b, a.c.n_seq, a.c.n_ctx, j);
            later |= o.sq == s.sq && o.n_new > 0;
        }
        if (__any_sync(0xffffffffu, later)) page = -1;                // (the same in every warp)
    }
    __syncthreads();
    auto put = [&](int which, int head, int d, const float (&y)[8]) {
        if (which == 0)     store8((T *)a.q_out + row_in * a.q_out_stride + (size_t)head * hd + d, y);
        else if (page >= 0) store8((which == 1 ? a.c.k : a.c.v) + page_at(a.c, page, head) + (size_t)(slot & (a.c.page - 1)) * hd + d, y);
    };
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (which[u] < 0) continue;
        if constexpr (KIND == 2) {
            if (which[u] < 2) {
                const int d0 = at[u] < half ? at[u] : a.n_rot + (at[u] - half) * 2, d1 = at[u] < half ? d0 + half : d0 + 1;
                float y0 = rope_get(&pair[u][0]), y1 = rope_get(&pair[u][1]);
                if (at[u] < half) {
                    const float2 c = cs[at[u]];
                    const float x0 = y0, x1 = y1;
                    y0 = x0 * c.x - x1 * c.y; y1 = x0 * c.y + x1 * c.x;
                }
                if (which[u] == 0) {
                    T * to = (T *)a.q_out + row_in * a.q_out_stride + (size_t)head[u] * hd;
                    rope_put(to + d0, y0); rope_put(to + d1, y1);
                } else if (page >= 0) {
                    __half * to = a.c.k + page_at(a.c, page, head[u]) + (size_t)(slot & (a.c.page - 1)) * hd;
                    rope_put(to + d0, y0); rope_put(to + d1, y1);
                }
            } else {
                const T * x = (const T *)a.x[2] + row_in * a.x_stride[2] + (size_t)head[u] * hd + at[u] * 16;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    float y[8];
                    load8(x + 8 * w, v[u][0]);
                    open8(v[u][0], y);
                    put(2, head[u], at[u] * 16 + 8 * w, y);
                }
            }
        } else {
            bool turns; int d0, d1;
            places(which[u], at[u], turns, d0, d1);
            float x0[8], x1[8];
            open8(v[u][0], x0);
            open8(v[u][1], x1);
            if (KIND == 0 && which[u] < 2) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int k = (d0 + j) >> 1;
                    if (k < half) { const float2 c = cs[k]; const float a0 = x0[j], a1 = x0[j + 1]; x0[j] = a0 * c.x - a1 * c.y; x0[j + 1] = a0 * c.y + a1 * c.x; }
                    if (k + 4 < half) { const float2 c = cs[k + 4]; const float a0 = x1[j], a1 = x1[j + 1]; x1[j] = a0 * c.x - a1 * c.y; x1[j + 1] = a0 * c.y + a1 * c.x; }
                }
            } else if (turns) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float2 c = cs[d0 + j];
                    const float a0 = x0[j], a1 = x1[j];
                    x0[j] = a0 * c.x - a1 * c.y; x1[j] = a0 * c.y + a1 * c.x;
                }
            }
            put(which[u], head[u], d0, x0);
            put(which[u], head[u], d1, x1);
        }
    }
}

template <typename T, int KIND>
static int append_run(const AppendP & p, int U, int threads, cudaStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.parts * p.a.b.max_new), p.a.b.n), block(threads);
    if (U == 1)      PI_CUDA(launch_k(k_kv_append<T, KIND, 1>, grid, block, 0, st, true, p));
    else if (U == 2 || sizeof(T) == 4) PI_CUDA(launch_k(k_kv_append<T, KIND, 2>, grid, block, 0, st, true, p));
    else if (U == 3) PI_CUDA(launch_k(k_kv_append<T, KIND, 3>, grid, block, 0, st, true, p));
    else             PI_CUDA(launch_k(k_kv_append<T, KIND, 4>, grid, block, 0, st, true, p));
    return PI_OK;
}

// Few tokens: a unit a thread, so that there are threads for all SMs.  Many: two to four units a thread (FP32: one or two, 64 bytes each), the number of units and threads that leaves the fewest without one (of 576 units of the
// falcon shape 2 x 256 and a second CTA of 64 took 40 us for 3329 tokens).
template <typename T>
static int append_go(const AppendArgs & a, cudaStream_t st) {
    AppendP p;
    p.a = a;
    p.heads[0] = a.x[0] ? a.n_head : 0; p.heads[1] = p.heads[2] = a.c.H;
    const int half = a.n_rot / 2, kind = !a.halves || half == 0 ? 0 : half % 8 == 0 ? 1 : 2;
    p.per_head = kind == 2 ? a.c.hd / 2 : a.c.hd / 16;
    const int64_t units = (int64_t)(p.heads[0] + p.heads[1]) * p.per_head + (int64_t)p.heads[2] * (a.c.hd / 16);
    int U = 1; int64_t least = -1;
    for (int u = 1; u <= 4; u++) {
        const bool many = (int64_t)a.b.n * a.b.max_new * units >= (int64_t)sm_count() * 8 * AP_THREADS;
        if (many ? (sizeof(T) == 2 ? u == 1 : u > 2) : u > 1) continue;
        const int64_t parts = (units + (int64_t)u * AP_THREADS - 1) / ((int64_t)u * AP_THREADS), threads = ((units + parts * u - 1) / (parts * u) + 31) / 32 * 32;
        if (least < 0 || parts * threads * u <= least) { least = parts * threads * u; U = u; p.parts = (int)parts; }
    }
    const int threads = (int)(((units + (int64_t)p.parts * U - 1) / ((int64_t)p.parts * U) + 31) / 32 * 32);
    return kind == 0 ? append_run<T, 0>(p, U, threads, st) : kind == 1 ? append_run<T, 1>(p, U, threads, st) : append_run<T, 2>(p, U, threads, st);
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
