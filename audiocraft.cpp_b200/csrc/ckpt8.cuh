// ckpt8.cuh -- 8-bit tensors (codes and power-of-two block scales) and typed element access for
// the kernels that write or read them: ckpt8.cu, layernorm_fwd.cu, layernorm_bwd.cu, rank_ckpt8.cu, gemm_f8.cu.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "train_ops.h"

namespace act {
namespace c8 {

constexpr int BLOCK = 128;  // columns of a block
constexpr uint32_t FULL_WARP = 0xffffffffu;

// ---------------------------------------------------------------------------------------
// Four elements of a row per lane, one block of 128 columns per warp.  With VEC (bases, strides and
// columns are multiples of four elements) the lane owns the columns 4 lane .. 4 lane + 3, which
// exist all or not at all, and moves them as one word; without, it owns lane, lane + 32, .. so
// that a warp's scalar accesses still cover whole sectors.  Pointers are the lane's own (block's
// first element plus first_col) and `n` counts the columns of the row from the lane's first one.
template <bool VEC>
__device__ __forceinline__ int first_col(int lane) {
    return VEC ? 4 * lane : lane;
}
template <bool VEC>
__device__ __forceinline__ constexpr int elem(int i) {
    return VEC ? i : 32 * i;
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

// four neighbouring elements as one word
__device__ __forceinline__ void unpack4(const float4& w, float v[4], float) {
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void unpack4(const uint2& w, float v[4], f16) {
    const float2 a = unpack_f16(w.x), b = unpack_f16(w.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void unpack4(const uint2& w, float v[4], __nv_bfloat16) {
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
    v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float4 pack4(const float v[4], float) { return make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ uint2 pack4(const float v[4], f16) {
    return make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]));
}
__device__ __forceinline__ uint2 pack4(const float v[4], __nv_bfloat16) {
    return make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}

// what a lane holds of a block as it lies in memory, for loads issued well before their use;
// missing columns read as 0
template <typename T, bool VEC>
struct Raw4 {
    typedef decltype(pack4((const float*)nullptr, T())) Word;
    Word w;
    __device__ __forceinline__ void load(const T* p, int n) {
        w = Word();
        if (n > 0) w = *reinterpret_cast<const Word*>(p);
    }
    __device__ __forceinline__ void values(float v[4]) const { unpack4(w, v, T()); }
};
template <typename T>
struct Raw4<T, false> {
    T e[4];
    __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = 32 * i < n ? p[32 * i] : T(0.f);
    }
    __device__ __forceinline__ void values(float v[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
    }
};
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, int n, float v[4]) {
    Raw4<T, VEC> r;
    r.load(p, n);
    r.values(v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* p, int n, const float v[4]) {
    typedef decltype(pack4(v, T())) Word;
    if (VEC) {
        if (n > 0) *reinterpret_cast<Word*>(p) = pack4(v, T());
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (32 * i < n) p[32 * i] = from_f32<T>(v[i]);
}
// parameters that no kernel here writes: loads that may move across its stores
template <bool VEC>
__device__ __forceinline__ void load4_const(const float* p, int n, float v[4]) {
    if (VEC) {
        float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n > 0) w = __ldg(reinterpret_cast<const float4*>(p));
        unpack4(w, v, float());
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 32 * i < n ? __ldg(p + 32 * i) : 0.f;
}
// elements of B bytes: fp32, or f16 / bf16 told apart at run time
template <int B, bool VEC>
__device__ __forceinline__ void store4_bytes(char* p, bool half, int n, const float v[4]) {
    if (B == 4) return store4<float, VEC>(reinterpret_cast<float*>(p), n, v);
    if (VEC) {
        const uint2 a = pack4(v, f16()), b = pack4(v, __nv_bfloat16());
        if (n > 0) *reinterpret_cast<uint2*>(p) = half ? a : b;
        return;
    }
    if (half) store4<f16, VEC>(reinterpret_cast<f16*>(p), n, v);
    else store4<__nv_bfloat16, VEC>(reinterpret_cast<__nv_bfloat16*>(p), n, v);
}
template <int B, bool VEC>
__device__ __forceinline__ void load4_bytes(const char* p, bool half, int n, float v[4]) {
    if (B == 4) return load4<float, VEC>(reinterpret_cast<const float*>(p), n, v);
    if (half) load4<f16, VEC>(reinterpret_cast<const f16*>(p), n, v);
    else load4<__nv_bfloat16, VEC>(reinterpret_cast<const __nv_bfloat16*>(p), n, v);
}

// ---------------------------------------------------------------------------------------
// Two fp32 in a 64-bit register: one instruction works on both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(lo)), "r"(__float_as_uint(hi)));
    return r;
}
__device__ __forceinline__ uint64_t pair(float v) { return pair(v, v); }
__device__ __forceinline__ float2 unpair(uint64_t v) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void pairs(const float v[4], uint64_t o[2]) {
    o[0] = pair(v[0], v[1]);
    o[1] = pair(v[2], v[3]);
}
__device__ __forceinline__ void unpairs(const uint64_t v[2], float o[4]) {
    const float2 a = unpair(v[0]), b = unpair(v[1]);
    o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}

// ---------------------------------------------------------------------------------------
// Block scale.  top = m 2^k (1 <= m < 2) and amax = a 2^j: the smallest power of two s with
// amax <= top s is 2^(j - k), or 2^(j - k + 1) where a > m: adding the mantissa's distance from m
// to its end carries into the exponent just then.  448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
// s >= 2^-126 keeps s and 1 / s normal, which is what an all-zero block (and a subnormal amax) gets.
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax_bits, bool e4m3) {
    const uint32_t k = e4m3 ? 8u : 6u, room = e4m3 ? 0x1fffffu : 0x1ffffu;
    return max((amax_bits + room) & 0x7f800000u, (k + 1) << 23) - (k << 23);
}
// 1 / s of a power of two: exponent 254 - e
__device__ __forceinline__ float inverse_pow2(uint32_t s_bits) { return __uint_as_float((254u << 23) - s_bits); }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest value a code and a scale stand for in fp32, 240 * 2^120 or 127 * 2^121, as float bits: the
// next code stands for 2^128.  Values beyond it are stored as it.
__device__ __forceinline__ constexpr uint32_t limit_bits(bool e4m3) { return e4m3 ? 0x7f700000u : 0x7f7e0000u; }
__device__ __forceinline__ float limited(float v, bool e4m3) {  // infinities and NaN stay
    return abs_bits(v) > limit_bits(e4m3) && abs_bits(v) < 0x7f800000u
               ? copysignf(__uint_as_float(limit_bits(e4m3)), v)
               : v;
}
__device__ __forceinline__ void limit4(float v[4], bool e4m3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = limited(v[i], e4m3);
}

// The largest finite |x| of a block as float bits, and whether the block holds anything beyond the limit or
// not finite (which is rare and costs its own pass).  Non-negative floats order like their bits, and
// bits >= 0x7f800000 are infinities and NaN.
struct Top {
    uint32_t bits;
    bool bad;
};
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t largest(const float v[4]) {
    return abs_bits(max_nan(max_nan(fabsf(v[0]), fabsf(v[1])), max_nan(fabsf(v[2]), fabsf(v[3]))));
}
__device__ __forceinline__ uint32_t largest_finite(const float v[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, abs_bits(v[i]) < 0x7f800000u ? abs_bits(v[i]) : 0u);
    return m;
}
__device__ __forceinline__ Top warp_top(float v[4], bool e4m3) {  // and limits the values
    Top t;
    t.bits = __reduce_max_sync(FULL_WARP, largest(v));
    t.bad = t.bits > limit_bits(e4m3);
    if (t.bad) {
        limit4(v, e4m3);
        t.bits = __reduce_max_sync(FULL_WARP, largest_finite(v));
    }
    return t;
}

// Four values within the limit times 1 / s (exact) -> four codes; with `bad`, what is not finite becomes NaN
// first.
// I8: adding 1.5 * 2^23 rounds to nearest even and leaves the whole number in the low byte.
__device__ __forceinline__ uint32_t encode4(const float v[4], float inv, bool e4m3, bool bad) {
    const uint64_t i2 = pair(inv);
    if (e4m3) {
        float x[4];
        const uint64_t m[2] = {mul2(pair(v[0], v[1]), i2), mul2(pair(v[2], v[3]), i2)};
        unpairs(m, x);
        if (bad)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (abs_bits(v[i]) >= 0x7f800000u) x[i] = __int_as_float(0x7fc00000);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
    uint32_t r[4];
    float x[4];
    const uint64_t m[2] = {fma2(pair(v[0], v[1]), i2, pair(12582912.0f)), fma2(pair(v[2], v[3]), i2, pair(12582912.0f))};
    unpairs(m, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
    if (bad)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (abs_bits(v[i]) >= 0x7f800000u) r[i] = 0x80u;
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

// Four codes -> the whole numbers / floats they stand for before scaling (I8 -128: NaN).  I8: the
// code plus 128 goes into the low byte of the float 2^23, from which 2^23 + 128 is taken (exact).
__device__ __forceinline__ void decode4(uint32_t w, bool e4m3, float v[4]) {
    if (e4m3) {
        const __half2 a = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
        const __half2 b = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
        const float2 fa = __half22float2(a), fb = __half22float2(b);
        v[0] = fa.x; v[1] = fa.y; v[2] = fb.x; v[3] = fb.y;
        return;
    }
    const uint32_t x = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7650 + i)) - 8388736.0f;
    if ((x - 0x01010101u) & ~x & 0x80808080u)  // a zero byte of x (a borrow may flag the one above too)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (((x >> (8 * i)) & 0xffu) == 0) v[i] = __int_as_float(0x7fc00000);
}

// a lane's codes of one block of a row
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, uint32_t w) {
    if (VEC) {
        if (n > 0) *reinterpret_cast<uint32_t*>(p) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (32 * i < n) p[32 * i] = (uint8_t)(w >> (8 * i));
}
template <bool VEC>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int n) {
    uint32_t w = 0;
    if (VEC) {
        if (n > 0) w = *reinterpret_cast<const uint32_t*>(p);
        return w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (32 * i < n) w |= (uint32_t)p[32 * i] << (8 * i);
    return w;
}

// quantise and store one block held by a warp, whose values are limited on the way; returns the scale's
// bits (the caller stores it)
template <bool VEC>
__device__ __forceinline__ uint32_t store_block(uint8_t* p, int n, float v[4], bool e4m3) {
    const Top t = warp_top(v, e4m3);
    const uint32_t s = scale_bits(t.bits, e4m3);
    store_codes<VEC>(p, n, encode4(v, inverse_pow2(s), e4m3, t.bad));
    return s;
}

// ---------------------------------------------------------------------------------------
// Normal distribution: Q = 1 - Phi(|z|) = P(t) exp(-z^2 / 2), t = 1 / (1 + 0.3 |z|), where P is
// the polynomial of degree 8 fitted (iteratively reweighted least squares, relative error
// 6.8e-8 for |z| <= 14.5, where Q leaves fp32's range; evaluated in fp32 5.6e-7 with a reciprocal
// one step off) to exp(z^2 / 2) (1 - Phi(|z|)).  The form keeps relative accuracy in the tail,
// where 1 - erf would cancel.  With the hardware's exponential (2^-22; it flushes below 2^-126) and
// its argument's roundings (6.7e-8 z^2) the tail is within 2^-20 + 6.7e-8 z^2 of the true one.  Two
// values at a time: half the instructions.
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// a = -min(|z|, 16): beyond 16 Q and exp(-z^2 / 2) are 0
__device__ __forceinline__ uint64_t minus_abs(float z0, float z1) {
    return pair(fmaxf(-fabsf(z0), -16.f), fmaxf(-fabsf(z1), -16.f));
}
// Q and exp(-z^2 / 2)
__device__ __forceinline__ void normal_tail(uint64_t a, uint64_t& q, uint64_t& e) {
    const float2 x = unpair(mul2(mul2(a, a), pair(-0.72134752044448170f)));  // -z^2 / 2 in powers of two
    const float2 d = unpair(fma2(a, pair(-0.3f), pair(1.0f)));
    const uint64_t t = pair(rcp(d.x), rcp(d.y));
    e = pair(ex2(x.x), ex2(x.y));
    uint64_t r = pair(0.03840748965740204f);
    r = fma2(r, t, pair(-0.1693079173564911f));
    r = fma2(r, t, pair(0.22895267605781555f));
    r = fma2(r, t, pair(-0.07684063166379929f));
    r = fma2(r, t, pair(0.14276590943336487f));
    r = fma2(r, t, pair(0.0945856124162674f));
    r = fma2(r, t, pair(0.121945321559906f));
    r = fma2(r, t, pair(0.11948420107364655f));
    r = fma2(r, t, pair(7.372795153059997e-06f));
    q = mul2(r, e);
}
// z Phi(z) = max(z, 0) - |z| Q
__device__ __forceinline__ uint64_t gelu2(float z0, float z1) {
    const uint64_t a = minus_abs(z0, z1);
    uint64_t q, e;
    normal_tail(a, q, e);
    return fma2(a, q, pair(max_nan(z0, 0.f), max_nan(z1, 0.f)));
}
// Phi(z) + z phi(z), Phi(z) = [z > 0] - sign(z) Q
__device__ __forceinline__ uint64_t gelu_grad2(uint64_t z) {
    const float2 f = unpair(z);
    uint64_t q, e;
    normal_tail(minus_abs(f.x, f.y), q, e);
    const float2 u = unpair(q);
    const uint64_t sq = pair(f.x > 0.f ? -u.x : u.x, f.y > 0.f ? -u.y : u.y);
    const uint64_t step = pair(f.x > 0.f ? 1.f : 0.f, f.y > 0.f ? 1.f : 0.f);
    return fma2(mul2(z, pair(0.3989422804014327f)), e, add2(step, sq));
}

}  // namespace c8
}  // namespace act
