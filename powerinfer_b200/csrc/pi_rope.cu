// Rotary positions of queries and keys: interleaved pairs (2i, 2i + 1) or halves (i, i + n_rot / 2), the first n_rot dimensions of each head,
// any frequency per pair (ggml_rope_custom with freq_scale / ext_factor / attn_factor, ggml.c:11163-11325).
//
//     a = pos * f_i     (y0, y1) = mscale * (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
//
// At position 10^6 an angle in 32 bits is off by 0.03, so the product is taken in 64 bits and reduced there to [-pi/4, pi/4]
// and a quarter turn (pi / 2 as the sum of two numbers, after Cody and Waite); sine and cosine of what is left are FP32 functions.  A CTA takes one token and a share of its heads: every
// thread requests its vectors first, the angles of the token are made while they travel (n_rot / 2 of them, once for all heads).
// Bound by the bytes of x and y for many tokens, by the launch for one.  Measured: 1901 tokens of 128 + 8 FP16 heads of 64 15 us (66 MB, 4.3 TB/s), one token 4 us.
#include "pi_kv_q8.cuh"
#include "pi_rope.cuh"

namespace pi {

static constexpr int ROPE_THREADS = 256;

template <typename T> struct RopeVec;                                 // 16 bytes of a row
template <> struct RopeVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void open(const uint4 & u, float (&v)[4]) { v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w); }
    static __device__ __forceinline__ uint4 close(const float (&v)[4]) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
};
template <> struct RopeVec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void open(const uint4 & u, float (&v)[8]) {
        const float2 a = h2f(u.x), b = h2f(u.y), c = h2f(u.z), d = h2f(u.w);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
    }
    static __device__ __forceinline__ uint4 close(const float (&v)[8]) {
        uint4 u; __half2 * h = reinterpret_cast<__half2 *>(&u);
        for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        return u;
    }
};
// UNIT: what a thread takes at once.  0: 32 bytes of a row (whole pairs); 1: 16 bytes of the first half and those of the second, or 32 of
// the dimensions that pass; 2: one pair, where a half is no multiple of 16 bytes.
template <typename T, int UNIT>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_ext(const RopeExtArgs p, int parts, int per_head) {
    constexpr int N = RopeVec<T>::N, U = UNIT == 2 ? 4 : 2;
    __shared__ float2 cs[128];
    const int t = blockIdx.x / parts, part = blockIdx.x - t * parts, half = p.n_rot >> 1;
    const int units = (p.heads[0] + p.heads[1]) * per_head;
    pdl_launch();
    pdl_wait();
    const T * src[U]; T * dst[U];
    int at[U];                                                        // unit's number in its head, -1: none
    uint4 v[U][2]; float e[U][2];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = (part * U + u) * ROPE_THREADS + threadIdx.x;
        at[u] = -1;
        if (i < units) {
            int h = i / per_head;
            at[u] = i - h * per_head;
            const int which = h >= p.heads[0];
            if (which) h -= p.heads[0];
            src[u] = (const T *)(which ? p.x[1] : p.x[0]) + (size_t)t * (which ? p.x_stride[1] : p.x_stride[0]) + (size_t)h * p.hd;
            dst[u] = (T *)(which ? p.y[1] : p.y[0]) + (size_t)t * (which ? p.y_stride[1] : p.y_stride[0]) + (size_t)h * p.hd;
            if constexpr (UNIT == 0) {
                const int d = at[u] * 2 * N;
                v[u][0] = *reinterpret_cast<const uint4 *>(src[u] + d);
                if (d + N < p.hd) v[u][1] = *reinterpret_cast<const uint4 *>(src[u] + d + N);
            } else if constexpr (UNIT == 1) {
                const bool turns = at[u] * N < half;
                const int d0 = turns ? at[u] * N : p.n_rot + (at[u] - half / N) * 2 * N, d1 = turns ? d0 + half : d0 + N;
                v[u][0] = *reinterpret_cast<const uint4 *>(src[u] + d0);
                if (d1 < p.hd) v[u][1] = *reinterpret_cast<const uint4 *>(src[u] + d1);
            } else {
                const bool turns = at[u] < half;
                const int d0 = turns ? at[u] : p.n_rot + (at[u] - half) * 2, d1 = turns ? d0 + half : d0 + 1;
                e[u][0] = rope_get(src[u] + d0);
                e[u][1] = rope_get(src[u] + d1);
            }
        }
    }
    const int pos = p.pos[t];
    for (int i = threadIdx.x; i < half; i += ROPE_THREADS) cs[i] = rope_angle(pos, p.freqs[i], p.mscale);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (at[u] < 0) continue;
        if constexpr (UNIT == 0) {
            const int d = at[u] * 2 * N;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int dw = d + w * N;
                if (dw >= p.hd) break;
                float x[N];
                RopeVec<T>::open(v[u][w], x);
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const int i = (dw + j) >> 1;
                    if (i < half) {
                        const float2 a = cs[i];
                        const float y0 = x[j] * a.x - x[j + 1] * a.y, y1 = x[j] * a.y + x[j + 1] * a.x;
                        x[j] = y0; x[j + 1] = y1;
                    }
                }
                *reinterpret_cast<uint4 *>(dst[u] + dw) = RopeVec<T>::close(x);
            }
        } else if constexpr (UNIT == 1) {
            const bool turns = at[u] * N < half;
            const int d0 = turns ? at[u] * N : p.n_rot + (at[u] - half / N) * 2 * N, d1 = turns ? d0 + half : d0 + N;
            if (turns) {
                float x0[N], x1[N];
                RopeVec<T>::open(v[u][0], x0);
                RopeVec<T>::open(v[u][1], x1);
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const float2 a = cs[d0 + j];
                    const float y0 = x0[j] * a.x - x1[j] * a.y, y1 = x0[j] * a.y + x1[j] * a.x;
                    x0[j] = y0; x1[j] = y1;
                }
                v[u][0] = RopeVec<T>::close(x0);
                v[u][1] = RopeVec<T>::close(x1);
            }
            *reinterpret_cast<uint4 *>(dst[u] + d0) = v[u][0];
            if (d1 < p.hd) *reinterpret_cast<uint4 *>(dst[u] + d1) = v[u][1];
        } else {
            const bool turns = at[u] < half;
            const int d0 = turns ? at[u] : p.n_rot + (at[u] - half) * 2, d1 = turns ? d0 + half : d0 + 1;
            if (turns) {
                const float2 a = cs[at[u]];
                const float y0 = e[u][0] * a.x - e[u][1] * a.y, y1 = e[u][0] * a.y + e[u][1] * a.x;
                e[u][0] = y0; e[u][1] = y1;
            }
            rope_put(dst[u] + d0, e[u][0]);
            rope_put(dst[u] + d1, e[u][1]);
        }
    }
}

template <typename T>
static int rope_ext_go(const RopeExtArgs & a, cudaStream_t st) {
    constexpr int N = RopeVec<T>::N;
    const int half = a.n_rot / 2, heads = a.heads[0] + a.heads[1];
    const int unit = !a.halves ? 0 : half % N == 0 ? 1 : 2;
    const int per_head = unit == 0 ? (a.hd / N + 1) / 2 : unit == 1 ? half / N + ((a.hd - a.n_rot) / N + 1) / 2 : a.hd / 2;
    const int64_t units = (int64_t)heads * per_head, of_cta = (int64_t)ROPE_THREADS * (unit == 2 ? 4 : 2);
    const int64_t parts = (units + of_cta - 1) / of_cta;
    const dim3 grid((unsigned)(parts * a.T));
    if (unit == 0)      PI_CUDA(launch_k(k_rope_ext<T, 0>, grid, dim3(ROPE_THREADS), 0, st, true, a, (int)parts, per_head));
    else if (unit == 1) PI_CUDA(launch_k(k_rope_ext<T, 1>, grid, dim3(ROPE_THREADS), 0, st, true, a, (int)parts, per_head));
    else                PI_CUDA(launch_k(k_rope_ext<T, 2>, grid, dim3(ROPE_THREADS), 0, st, true, a, (int)parts, per_head));
    return PI_OK;
}

int launch_rope_ext(const RopeExtArgs & a, cudaStream_t st) {
    return a.xtype == PI_TYPE_F16 ? rope_ext_go<__half>(a, st) : rope_ext_go<float>(a, st);
}

}  // namespace pi
