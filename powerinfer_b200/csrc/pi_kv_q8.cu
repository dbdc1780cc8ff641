// The KV cache in 8 bits: store, and read back as values.
//
// A block of slots of one sequence and KV head has one scale, for keys and for values.  With a the largest finite magnitude of the
// new rows that fall into a block and s_old its scale where earlier tokens are in it already (0 where none are),
//
//     s = max(a * (1 / 127), s_old)      code = rne(x * (1 / s)) within +-127      earlier codes = rne(code * (s_old / s)) where s > s_old
//
// each step in FP32, so that codes and scales are the same bits wherever they are made.  An infinity is held as +-127, what is not a number as 0,
// and a block whose scale would be no normal number as zeros.  Slots behind the new ones are left as they are.
// Bound by the bytes of the new rows for prompts, by the launch for single tokens.  A unit is one block of keys or values:
// 256 threads, which keep its rows in registers between maximum and codes, or 32 where few tokens come at a time.
// Measured: 4096 FP32 tokens, 8 KV heads of 128 15 us (2.8 TB/s; 72 % of the issue slots: four values a thread go through maximum, product, rounding and packing),
// 32 FP16 tokens of 32 heads 5.4 us.
#include "pi_kv_q8.cuh"

#include <cfloat>

namespace pi {

static constexpr int KV_THREADS = 256;

struct StoreP {
    KvQ8 c; RaggedB b;
    const void * x[2]; int64_t stride[2];
    int n_blocks;                                                     // blocks that max_new tokens can touch
};

template <typename T> __device__ __forceinline__ float4 load4(const T * p);
template <> __device__ __forceinline__ float4 load4<float>(const float * p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
template <> __device__ __forceinline__ float4 load4<__half>(const __half * p) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    const float2 a = h2f(u.x), b = h2f(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float finite_abs(float x) { const float a = fabsf(x); return a <= FLT_MAX ? a : 0.f; }     // (false for NaN)
__device__ __forceinline__ int q8_code(float x, float inv) {
    const float y = x * inv;
    return y != y ? 0 : __float2int_rn(fminf(fmaxf(y, -127.f), 127.f));
}
__device__ __forceinline__ uint32_t q8_codes(const float4 & x, float inv) {
    return (uint32_t)(q8_code(x.x, inv) & 255) | (uint32_t)(q8_code(x.y, inv) & 255) << 8 | (uint32_t)(q8_code(x.z, inv) & 255) << 16 | (uint32_t)q8_code(x.w, inv) << 24;
}
__device__ __forceinline__ uint32_t q8_rescale(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) r |= (uint32_t)(__float2int_rn((float)(int8_t)(w >> (8 * j)) * ratio) & 255) << (8 * j);
    return r;
}

// NT threads per unit, HOLD vectors of four values in registers (others are read again): a block of 32 x 128 or less needs 4, and leaves room for
// more CTAs, which is what hides the way from one's loads to its stores
template <typename T, int NT, int HOLD>
__global__ void __launch_bounds__(KV_THREADS, HOLD <= 4 ? 5 : 3) k_kv_store(const StoreP p) {
    constexpr int UNITS = KV_THREADS / NT;
    __shared__ float s_max[KV_THREADS / 32];
    const int lane = threadIdx.x & 31, tid = NT == 32 ? lane : (int)threadIdx.x;
    const int64_t unit = (int64_t)blockIdx.x * UNITS + (NT == 32 ? threadIdx.x >> 5 : 0);      // (block, keys or values, head), blocks of a head side by side
    const int i = blockIdx.y;
    pdl_launch();
    pdl_wait();
    if (unit >= (int64_t)p.n_blocks * 2 * p.c.H) return;
    const int nb = (int)(unit % p.n_blocks), hv = (int)(unit / p.n_blocks), h = hv >> 1, which = hv & 1;
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, i);
    if (s.sq < 0 || s.n_new == 0) return;
    const int B = p.c.block, b = (s.pos >> p.c.shift) + nb, lo = max(s.pos, b * B), hi = min(min(s.pos + s.n_new, p.c.n_ctx), (b + 1) * B);
    if (lo >= hi) return;
    if (p.b.seq) {                                                    // of entries that name one sequence the last one counts
        bool later = false;
        for (int j = i + 1 + lane; j < p.b.n; j += 32) {
            const SeqB o = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, j);
            later |= o.sq == s.sq && o.n_new > 0;
        }
        if (__any_sync(0xffffffffu, later)) return;                   // (the same in every warp)
    }
    const int hd = p.c.hd, v4 = hd >> 2, n_vec = (hi - lo) * v4;
    const int64_t stride = which ? p.stride[1] : p.stride[0];
    const T * x = (const T *)(which ? p.x[1] : p.x[0]) + (int64_t)(s.first + lo - s.pos) * stride + (int64_t)h * hd;
    const size_t head = (size_t)s.sq * p.c.H + h;
    int8_t * codes = (which ? p.c.v : p.c.k) + (head * p.c.n_ctx + lo) * hd;
    float * scale = (which ? p.c.vs : p.c.ks) + head * (p.c.n_ctx >> p.c.shift) + b;
    const float old = lo > b * B ? *scale : 0.f;
    float4 keep[HOLD];
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < HOLD; u++) {
        const int e = tid + u * NT;
        keep[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (e < n_vec) { const int r = e / v4; keep[u] = load4(x + (int64_t)r * stride + (e - r * v4) * 4); }
    }
#pragma unroll
    for (int u = 0; u < HOLD; u++) m = fmaxf(fmaxf(m, fmaxf(finite_abs(keep[u].x), finite_abs(keep[u].y))), fmaxf(finite_abs(keep[u].z), finite_abs(keep[u].w)));
    for (int e = tid + HOLD * NT; e < n_vec; e += NT) {
        const int r = e / v4;
        const float4 w = load4(x + (int64_t)r * stride + (e - r * v4) * 4);
        m = fmaxf(fmaxf(m, fmaxf(finite_abs(w.x), finite_abs(w.y))), fmaxf(finite_abs(w.z), finite_abs(w.w)));
    }
    m = warp_max(m);
    if (NT > 32) {
        if (lane == 0) s_max[threadIdx.x >> 5] = m;
        __syncthreads();
        m = s_max[0];
#pragma unroll
        for (int w = 1; w < KV_THREADS / 32; w++) m = fmaxf(m, s_max[w]);
    }
    float now = fmaxf(m * (1.0f / 127.0f), old);
    if (!(now >= FLT_MIN)) now = 0.f;
    const float inv = now > 0.f ? 1.0f / now : 0.f;
#pragma unroll
    for (int u = 0; u < HOLD; u++) {
        const int e = tid + u * NT;
        if (e < n_vec) *reinterpret_cast<uint32_t *>(codes + (size_t)e * 4) = q8_codes(keep[u], inv);
    }
    for (int e = tid + HOLD * NT; e < n_vec; e += NT) {
        const int r = e / v4;
        *reinterpret_cast<uint32_t *>(codes + (size_t)e * 4) = q8_codes(load4(x + (int64_t)r * stride + (e - r * v4) * 4), inv);
    }
    if (tid == 0) *scale = now;
    if (lo > b * B && now > old) {                                    // the earlier tokens' codes in the new steps
        const float ratio = old / now;
        uint4 * w = reinterpret_cast<uint4 *>(codes - (size_t)(lo - b * B) * hd);
        const int n16 = (lo - b * B) * hd / 16;
        for (int e0 = tid; e0 < n16; e0 += 4 * NT) {
            uint4 c[4];
#pragma unroll
            for (int u = 0; u < 4; u++) if (e0 + u * NT < n16) c[u] = w[e0 + u * NT];
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (e0 + u * NT < n16)
                    w[e0 + u * NT] = make_uint4(q8_rescale(c[u].x, ratio), q8_rescale(c[u].y, ratio), q8_rescale(c[u].z, ratio), q8_rescale(c[u].w, ratio));
        }
    }
}

// Up to this many tokens at a time a warp takes a unit: its row is four values a lane
static constexpr int STORE_FEW = 4;

template <typename T>
static int store_go(const StoreP & p, cudaStream_t st) {
    const int64_t units = (int64_t)p.n_blocks * 2 * p.c.H;
    if (p.b.max_new <= STORE_FEW)       PI_CUDA(launch_k(k_kv_store<T, 32, 4>, dim3((unsigned)((units + 7) / 8), p.b.n), dim3(KV_THREADS), 0, st, true, p));
    else if (p.c.block * p.c.hd <= 4096) PI_CUDA(launch_k(k_kv_store<T, KV_THREADS, 4>, dim3((unsigned)units, p.b.n), dim3(KV_THREADS), 0, st, true, p));
    else                                PI_CUDA(launch_k(k_kv_store<T, KV_THREADS, 8>, dim3((unsigned)units, p.b.n), dim3(KV_THREADS), 0, st, true, p));
    return PI_OK;
}

int launch_kv_store_q8(const KvQ8 & c, const RaggedB & b, int xtype, const void * k, int64_t k_stride, const void * v, int64_t v_stride, cudaStream_t st) {
    StoreP p;
    p.c = c; p.b = b; p.x[0] = k; p.x[1] = v; p.stride[0] = k_stride; p.stride[1] = v_stride;
    p.b.max_new = (int)imin64(b.max_new, c.n_ctx);                    // (no sequence holds more)
    p.n_blocks = (p.b.max_new + 2 * c.block - 2) >> c.shift;
    p.b.max_new = b.max_new;
    return xtype == PI_TYPE_F16 ? store_go<__half>(p, st) : store_go<float>(p, st);
}

// ------------------------------------------------------------------------------------------------
struct LoadP { KvQ8 c; RaggedB b; void * y[2]; int64_t stride[2]; int groups; };

// x = code * scale.  A warp takes LOAD_ROWS slots of a head, contiguous in the cache: all of its loads, four codes each, are on their way at once.
// Bound by the bytes of the values: 614 MB in 104 us (5.9 TB/s).
static constexpr int LOAD_ROWS = 16;

template <typename T, int HD>
__global__ void __launch_bounds__(KV_THREADS) k_kv_load(const LoadP p) {
    constexpr int V4 = HD / 4, N = LOAD_ROWS * V4 / 32;
    const int i = blockIdx.y, which = blockIdx.z, lane = threadIdx.x & 31;
    const int unit = blockIdx.x * (KV_THREADS / 32) + (threadIdx.x >> 5), h = unit / p.groups, t0 = (unit - h * p.groups) * LOAD_ROWS;
    pdl_launch();
    pdl_wait();
    const SeqB s = seq_entry(p.b, p.c.n_seq, p.c.n_ctx, i);
    if (h >= p.c.H || t0 >= s.n_new) return;
    const size_t head = (size_t)max(s.sq, 0) * p.c.H + h;
    const int8_t * codes = (which ? p.c.v : p.c.k) + (head * p.c.n_ctx + s.pos + t0) * HD;
    const float * scale = (which ? p.c.vs : p.c.ks) + head * (p.c.n_ctx >> p.c.shift);
    const int there = s.sq < 0 ? 0 : p.c.n_ctx - s.pos - t0, rows = min(LOAD_ROWS, s.n_new - t0);     // (slots that the cache lacks: zeros)
    uint32_t w[N]; float sc[N];
#pragma unroll
    for (int u = 0; u < N; u++) {
        const int e = u * 32 + lane, t = e / V4;
        w[u] = 0u; sc[u] = 0.f;
        if (t < rows && t < there) {
            w[u] = __ldg(reinterpret_cast<const uint32_t *>(codes + (size_t)e * 4));
            sc[u] = __ldg(scale + ((s.pos + t0 + t) >> p.c.shift));
        }
    }
    const int64_t stride = which ? p.stride[1] : p.stride[0];
    T * y = (T *)(which ? p.y[1] : p.y[0]) + (int64_t)(s.first + t0) * stride + h * HD;
#pragma unroll
    for (int u = 0; u < N; u++) {
        const int e = u * 32 + lane, t = e / V4;
        if (t >= rows) continue;
        T * at = y + t * stride + (e - t * V4) * 4;
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = (float)(int8_t)(w[u] >> (8 * j)) * sc[u];
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(at) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            __half2 hh[2] = {__floats2half2_rn(f[0], f[1]), __floats2half2_rn(f[2], f[3])};
            *reinterpret_cast<uint2 *>(at) = *reinterpret_cast<uint2 *>(hh);
        }
    }
}

template <typename T>
static int load_go(const LoadP & p, dim3 grid, cudaStream_t st) {
    switch (p.c.hd) {
        case 64:  PI_CUDA(launch_k(k_kv_load<T, 64>, grid, dim3(KV_THREADS), 0, st, true, p)); break;
        case 96:  PI_CUDA(launch_k(k_kv_load<T, 96>, grid, dim3(KV_THREADS), 0, st, true, p)); break;
        case 128: PI_CUDA(launch_k(k_kv_load<T, 128>, grid, dim3(KV_THREADS), 0, st, true, p)); break;
        case 192: PI_CUDA(launch_k(k_kv_load<T, 192>, grid, dim3(KV_THREADS), 0, st, true, p)); break;
        default:  PI_CUDA(launch_k(k_kv_load<T, 256>, grid, dim3(KV_THREADS), 0, st, true, p));
    }
    return PI_OK;
}

int launch_kv_load_q8(const KvQ8 & c, const RaggedB & b, int xtype, void * k, int64_t k_stride, void * v, int64_t v_stride, cudaStream_t st) {
    LoadP p;
    p.c = c; p.b = b; p.y[0] = k; p.y[1] = v; p.stride[0] = k_stride; p.stride[1] = v_stride;
    p.groups = (b.max_new + LOAD_ROWS - 1) / LOAD_ROWS;
    const dim3 grid((unsigned)(((int64_t)p.groups * c.H + KV_THREADS / 32 - 1) / (KV_THREADS / 32)), b.n, 2);
    return xtype == PI_TYPE_F16 ? load_go<__half>(p, grid, st) : load_go<float>(p, grid, st);
}

}  // namespace pi
