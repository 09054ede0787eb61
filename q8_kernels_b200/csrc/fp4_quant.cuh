// The arithmetic of the 4-bit quantizer, one unit of 16 values at a time: the quantizer's kernels (fp4.cu) and the product that quantises
// its few rows itself (gemm_fp4.cu) give the same bits.
#pragma once

#include "fp4.cuh"

namespace q8k {

constexpr int kFp4Unit = 16;                                   // values of a thread at a time: 32 bytes

// |max| of two 16-bit values or of one fp32 value; NaN wins.
template <typename T> struct Fp4In;
template <> struct Fp4In<__nv_bfloat16> {
    static __device__ __forceinline__ float absmax(const uint4 (&r)[2]) {
        __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&r[0].x));
        const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
        const float2 f = __bfloat1622float2(m);
        return max_nan(f.x, f.y);
    }
    static __device__ __forceinline__ void widen(const uint4& r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <> struct Fp4In<__half> {
    static __device__ __forceinline__ float absmax(const uint4 (&r)[2]) {
        __half2 m = __habs2(*reinterpret_cast<const __half2*>(&r[0].x));
        const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
        const float2 f = __half22float2(m);
        return max_nan(f.x, f.y);
    }
    static __device__ __forceinline__ void widen(const uint4& r, float (&v)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};

__device__ __forceinline__ float fp4_finite(float factor) { return fminf(factor, 3.402823466e38f); }

// A unit's values times `factor`, as 8 bytes.
template <typename T> __device__ __forceinline__ uint2 fp4_pack(const uint4 (&r)[2], float factor) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[8];
        Fp4In<T>::widen(r[h], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], factor);
        w[h] = float8_to_e2m1(v);
    }
    return make_uint2(w[0], w[1]);
}

// A row's scale and the factor on its blocks' absmax (nvfp4), from the row's absmax.
__device__ __forceinline__ void fp4_row_factors(float top, float& g, float& rs) {
    g = top > 0.f ? fp4_finite(__fdiv_rn(448.0f, top)) : top;  // 0 and NaN stay what they are
    rs = __fdiv_rn(top, 2688.0f);
}
// The scale byte of a unit's block and the factor on its values.  mxfp4: a block of 32 is the units of two neighbouring lanes.
template <bool NV> __device__ __forceinline__ uint8_t fp4_block_scale(float a, float g, float rs, float& factor) {
    if constexpr (NV) {
        const uint8_t scale = float_to_e4m3_sat(__fmul_rn(a, g));
        const float s = e4m3_to_float(scale);
        factor = s == 0.f ? 0.f : fp4_finite(__fdiv_rn(1.0f, __fmul_rn(s, rs)));
        return scale;
    } else {
        const float both = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
        const int field = (int)(__float_as_uint(both) >> 23);  // (no sign)
        const int e = field == 255 ? 255 : field > 2 ? field - 2 : 0;
        factor = __uint_as_float((uint32_t)(254 - (e == 255 ? 254 : e)) << 23);     // 2^-e; any for NaN
        return (uint8_t)e;
    }
}
template <typename Tin, int UNITS>
__device__ __forceinline__ void fp4_load(const Tin* __restrict__ row, int t, int threads, int units, bool here, uint4 (&r)[UNITS][2]) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int u = t + i * threads;
        const uint4* p = reinterpret_cast<const uint4*>(row + u * kFp4Unit);
        const bool in = here && u < units;
        r[i][0] = in ? p[0] : make_uint4(0, 0, 0, 0);
        r[i][1] = in ? p[1] : make_uint4(0, 0, 0, 0);
    }
}

}  // namespace q8k
