// The rotation's angles, and single values of rows.
#pragma once
#include "pi_common.cuh"

namespace pi {

__device__ __forceinline__ float rope_get(const float * p) { return *p; }
__device__ __forceinline__ float rope_get(const __half * p) { return __half2float(*p); }
__device__ __forceinline__ void rope_put(float * p, float v) { *p = v; }
__device__ __forceinline__ void rope_put(__half * p, float v) { *p = __float2half_rn(v); }

// cosine and sine of pos * f
__device__ __forceinline__ float2 rope_angle(int pos, double f, float mscale) {
    const double a = (double)pos * f, n = rint(a * 0.63661977236758134308);               // quarter turns
    double r = fma(n, -1.57079632679489655800, a);                                        // pi / 2 in two parts
    r = fma(n, -6.12323399573676603587e-17, r);
    const float s0 = sinf((float)r), c0 = cosf((float)r);
    const int k = (int)((long long)n & 3);
    const float c = k & 1 ? s0 : c0, s = k & 1 ? c0 : s0;
    return make_float2((k == 1 || k == 2 ? -c : c) * mscale, (k >= 2 ? -s : s) * mscale);
}

}  // namespace pi
