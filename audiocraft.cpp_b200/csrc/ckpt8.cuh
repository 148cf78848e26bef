// ckpt8.cuh -- 8-bit tensors (codes and power-of-two block scales) and typed element access for
// the kernels that write or read them: ckpt8.cu, layernorm.cu, rank_ckpt8.cu, gemm_f8.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "train_ops.h"

namespace act {
namespace c8 {

constexpr int BLOCK = 128;  // columns of a block
constexpr uint32_t FULL = 0xffffffffu;

// ---------------------------------------------------------------------------------------
// Four elements of a row per lane, one block of 128 columns per warp.  With VEC the lane owns the
// columns 4 lane .. 4 lane + 3 and moves them as one word when all four exist (bases and strides
// are multiples of four elements); without, it owns lane, lane + 32, .. so that a warp's scalar
// accesses still cover whole sectors.
template <bool VEC>
__device__ __forceinline__ int lane_col(int lane, int i) {
    return VEC ? 4 * lane + i : lane + 32 * i;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES>
struct Word4;
template <>
struct Word4<4> { typedef uint4 type; };
template <>
struct Word4<2> { typedef uint2 type; };
template <>
struct Word4<1> { typedef uint32_t type; };

// p: the block's first element; n: columns of the row from there (may exceed 128); missing
// columns read as 0
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, int n, int lane, float v[4]) {
    if (VEC && 4 * lane + 3 < n) {
        typedef typename Word4<sizeof(T)>::type W;
        const W w = *reinterpret_cast<const W*>(p + 4 * lane);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane_col<VEC>(lane, i);
        v[i] = c < n ? to_f32(p[c]) : 0.f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* p, int n, int lane, const float v[4]) {
    if (VEC && 4 * lane + 3 < n) {
        typedef typename Word4<sizeof(T)>::type W;
        W w;
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<W*>(p + 4 * lane) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane_col<VEC>(lane, i);
        if (c < n) p[c] = from_f32<T>(v[i]);
    }
}

// the same with the element type known at run time only (one uniform branch per four elements)
template <bool VEC>
__device__ __forceinline__ void store4_as(void* base, int type, long off, int n, int lane, const float v[4]) {
    if (type == OP_F16) store4<f16, VEC>(static_cast<f16*>(base) + off, n, lane, v);
    else if (type == OP_BF16) store4<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(base) + off, n, lane, v);
    else store4<float, VEC>(static_cast<float*>(base) + off, n, lane, v);
}
template <bool VEC>
__device__ __forceinline__ void load4_as(const void* base, int type, long off, int n, int lane, float v[4]) {
    if (type == OP_F16) load4<f16, VEC>(static_cast<const f16*>(base) + off, n, lane, v);
    else if (type == OP_BF16) load4<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(base) + off, n, lane, v);
    else load4<float, VEC>(static_cast<const float*>(base) + off, n, lane, v);
}

// ---------------------------------------------------------------------------------------
// Block scale.  top = m 2^k (1 <= m < 2) and amax = a 2^j: the smallest power of two s with
// amax <= top s is 2^(j - k), or 2^(j - k + 1) where a > m: one comparison of mantissa bits.
// 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.  s >= 2^-126 keeps s and 1 / s normal, which is what
// an all-zero block (and a subnormal amax) gets.
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax_bits, bool e4m3) {
    const uint32_t k = e4m3 ? 8u : 6u, m = e4m3 ? 0x600000u : 0x7e0000u;
    const uint32_t e = (amax_bits >> 23) + ((amax_bits & 0x7fffffu) > m ? 1u : 0u);
    return max(e, k + 1) - k << 23;
}
// 1 / s of a power of two: exponent 254 - e
__device__ __forceinline__ float inverse_pow2(uint32_t s_bits) { return __uint_as_float((254u << 23) - s_bits); }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest finite |x| of a block as float bits, and whether the block holds anything that is not
// finite (which is rare and costs its own pass).  Non-negative floats order like their bits, and
// bits >= 0x7f800000 are infinities and NaN.
struct Top {
    uint32_t bits;
    bool bad;
};
__device__ __forceinline__ uint32_t largest(const float v[4]) {
    return max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
}
__device__ __forceinline__ uint32_t largest_finite(const float v[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, abs_bits(v[i]) < 0x7f800000u ? abs_bits(v[i]) : 0u);
    return m;
}
__device__ __forceinline__ Top warp_top(const float v[4]) {
    Top t;
    t.bits = __reduce_max_sync(FULL, largest(v));
    t.bad = t.bits >= 0x7f800000u;
    if (t.bad) t.bits = __reduce_max_sync(FULL, largest_finite(v));
    return t;
}

// Four values times 1 / s (exact) -> four codes; with `bad`, what is not finite becomes NaN first.
// I8: adding 1.5 * 2^23 rounds to nearest even and leaves the whole number in the low byte.
__device__ __forceinline__ uint32_t encode4(const float v[4], float inv, bool e4m3, bool bad) {
    if (e4m3) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i] * inv;
        if (bad)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (abs_bits(v[i]) >= 0x7f800000u) x[i] = __int_as_float(0x7fc00000);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(fmaf(v[i], inv, 12582912.0f));
    if (bad)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (abs_bits(v[i]) >= 0x7f800000u) r[i] = 0x80u;
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

// four codes -> the whole numbers / floats they stand for before scaling (I8 -128: NaN)
__device__ __forceinline__ void decode4(uint32_t w, bool e4m3, float v[4]) {
    if (e4m3) {
        const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
        const __half2 b = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
        const float2 fa = __half22float2(a), fb = __half22float2(b);
        v[0] = fa.x; v[1] = fa.y; v[2] = fb.x; v[3] = fb.y;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = (int)(int8_t)(w >> (8 * i));
        v[i] = q == -128 ? __int_as_float(0x7fc00000) : (float)q;
    }
}

// codes of one block of a row
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, int lane, uint32_t w) {
    if (VEC && 4 * lane + 3 < n) {
        *reinterpret_cast<uint32_t*>(p + 4 * lane) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane_col<VEC>(lane, i);
        if (c < n) p[c] = (uint8_t)(w >> (8 * i));
    }
}
template <bool VEC>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int n, int lane) {
    if (VEC && 4 * lane + 3 < n) return *reinterpret_cast<const uint32_t*>(p + 4 * lane);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane_col<VEC>(lane, i);
        if (c < n) w |= (uint32_t)p[c] << (8 * i);
    }
    return w;
}

// quantise and store one block held by a warp; returns the scale's bits (the caller stores it)
template <bool VEC>
__device__ __forceinline__ uint32_t store_block(uint8_t* p, int n, int lane, const float v[4], bool e4m3) {
    const Top t = warp_top(v);
    const uint32_t s = scale_bits(t.bits, e4m3);
    store_codes<VEC>(p, n, lane, encode4(v, inverse_pow2(s), e4m3, t.bad));
    return s;
}

template <bool VEC>
__device__ __forceinline__ void load_block(const uint8_t* p, int n, int lane, float scale, bool e4m3, float v[4]) {
    decode4(load_codes<VEC>(p, n, lane), e4m3, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= scale;
}

// ---------------------------------------------------------------------------------------
// Normal distribution: Q = 1 - Phi(|z|) = P(t) exp(-z^2 / 2), t = 1 / (1 + 0.3 |z|), where P is
// the polynomial of degree 8 fitted (iteratively reweighted least squares, relative error
// 5.8e-8 for |z| <= 14.5, where Q leaves fp32's range) to exp(z^2 / 2) (1 - Phi(|z|)).  The form
// keeps relative accuracy in the tail, where 1 - erf would cancel.  With the hardware's
// reciprocal and exponential the results are within about 1e-6 of gelu and gelu'.
__device__ __forceinline__ float normal_tail(float a, float e) {
    const float t = __fdividef(1.0f, fmaf(0.3f, a, 1.0f));
    float r = 0.03840748965740204f;
    r = fmaf(r, t, -0.1693079173564911f);
    r = fmaf(r, t, 0.22895267605781555f);
    r = fmaf(r, t, -0.07684063166379929f);
    r = fmaf(r, t, 0.14276590943336487f);
    r = fmaf(r, t, 0.0945856124162674f);
    r = fmaf(r, t, 0.121945321559906f);
    r = fmaf(r, t, 0.11948420107364655f);
    r = fmaf(r, t, 7.372795153059997e-06f);
    return r * e;
}
__device__ __forceinline__ float gelu(float z) {
    const float a = fabsf(z), q = normal_tail(a, __expf(-0.5f * a * a));
    return z * (z > 0.f ? 1.0f - q : q);
}
__device__ __forceinline__ float gelu_grad(float z) {
    const float a = fabsf(z), e = __expf(-0.5f * a * a), q = normal_tail(a, e);
    return fmaf(z * 0.3989422804014327f, e, z > 0.f ? 1.0f - q : q);
}

}  // namespace c8
}  // namespace act
