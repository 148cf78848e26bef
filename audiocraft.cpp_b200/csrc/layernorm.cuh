// layernorm.cuh -- sums over a row that several warps share, for the layer norm's two passes
// (layernorm_fwd.cu, layernorm_bwd.cu).
#pragma once
#include "ckpt8.cuh"

namespace act {
namespace ln {

using namespace c8;

// The sum of one value, and of two, over the W warps of a row.  slot: W (2 W) floats of shared memory
// that nobody else uses between two calls (the caller alternates between two); bar: the row's
// own named barrier.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* slot, int wid, int lane, int bar) {
    v = warp_sum(v);
    if (W == 1) return v;
    if (lane == 0) slot[wid] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(W * 32) : "memory");
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += slot[w];
    return s;
}
template <int W>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* slot, int wid, int lane, int bar) {
    // after the first exchange the lower half-warp holds a's pairs and the upper one b's
    const bool up = lane & 16;
    float v = (up ? b : a) + __shfl_xor_sync(FULL_WARP, up ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_WARP, v, o);
    if (W == 1) return make_float2(__shfl_sync(FULL_WARP, v, 0), __shfl_sync(FULL_WARP, v, 16));
    if ((lane & 15) == 0) reinterpret_cast<float*>(slot + wid)[lane >> 4] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(W * 32) : "memory");
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        s.x += slot[w].x;
        s.y += slot[w].y;
    }
    return s;
}

}  // namespace ln
}  // namespace act
