// rank_ckpt8.cu -- the rank product that reads an 8-bit checkpoint: C[j][c] (+)= alpha * sum over
// rows t of U[t][j] * X[t][c], the lora_A gradient from a kept input.
//
// A CTA owns 64 columns of C and all nb <= 64 of its rows; X is decoded on its way into shared
// memory, sums are fp32 in registers.
#include "ckpt8.cuh"

namespace act {

namespace {

using namespace c8;

__global__ void __launch_bounds__(256) rank_kernel(const RankCkpt8 p) {
    __shared__ float us[32][65], xs[32][65];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const long c0 = (long)blockIdx.x * 64;
    float acc[4][4] = {};
    for (long t0 = 0; t0 < p.rows; t0 += 32) {
        for (int i = threadIdx.x; i < 32 * 64; i += 256) {
            const int r = i / 64, c = i % 64;
            const long t = t0 + r;
            float u = 0.f, x = 0.f;
            if (t < p.rows && c < p.nb) {
                const long at = t * p.u.ld + c;
                u = p.u.type == OP_F32 ? static_cast<const float*>(p.u.p)[at]
                    : p.u.type == OP_F16 ? to_f32(static_cast<const f16*>(p.u.p)[at])
                                         : to_f32(static_cast<const __nv_bfloat16*>(p.u.p)[at]);
            }
            if (t < p.rows && c0 + c < p.cols) {
                float v[4];
                decode4(p.x.q[t * p.x.ldq + c0 + c], p.x.e4m3, v);
                x = v[0] * p.x.scale[((c0 + c) / BLOCK) * p.x.lds + t];
            }
            us[r][c] = u;
            xs[r][c] = x;
        }
        __syncthreads();
        for (int r = 0; r < 32; ++r)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(us[r][ty + 16 * i], xs[r][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = ty + 16 * i;
            const long c = c0 + tx + 16 * j;
            if (r >= p.nb || c >= p.cols) continue;
            float* o = p.c + r * p.ldc + c;
            *o = p.accumulate ? *o + p.alpha * acc[i][j] : p.alpha * acc[i][j];
        }
}

}  // namespace

void rank_ckpt8(const RankCkpt8& a, cudaStream_t s) {
    rank_kernel<<<(unsigned)((a.cols + 63) / 64), 256, 0, s>>>(a);
}

}  // namespace act
