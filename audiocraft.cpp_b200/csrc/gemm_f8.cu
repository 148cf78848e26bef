// gemm_f8.cu -- product of two E4M3 tensors with a scale for each block of 128:
//   Y[m][n] = sum over k-blocks b of sx[b][m] * sw[b][n / 128] * (sum over the block's k of X[m][k] W[n][k])
//
// A CTA owns 64 x 64 of Y; both operands are decoded on their way into shared memory, sums are
// fp32 in registers.
#include "ckpt8.cuh"

namespace act {

namespace {

using namespace c8;

__global__ void __launch_bounds__(256) gemm_f8_kernel(const GemmF8 p) {
    __shared__ float xs[32][65], ws[32][65];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const long n0 = (long)blockIdx.x * 64;
    for (long m0 = (long)blockIdx.y * 64; m0 < p.M; m0 += (long)gridDim.y * 64) {
        float acc[4][4] = {};
        for (long k0 = 0; k0 < p.K; k0 += 32) {
            for (int i = threadIdx.x; i < 32 * 64; i += 256) {
                const int k = i % 32, r = i / 32, wk = p.w_mn ? i / 64 : k, wr = p.w_mn ? i % 64 : r;
                float v[4], x = 0.f, w = 0.f;
                if (k0 + k < p.K && m0 + r < p.M) {
                    decode4(p.x.q[(m0 + r) * p.x.ldq + k0 + k], true, v);
                    x = v[0] * p.x.scale[((k0 + k) / BLOCK) * p.x.lds + m0 + r];
                }
                if (k0 + wk < p.K && n0 + wr < p.N) {
                    const long n = n0 + wr, kk = k0 + wk;
                    decode4(p.w.q[p.w_mn ? kk * p.w.ldq + n : n * p.w.ldq + kk], true, v);
                    w = v[0] * p.w.scale[p.w_mn ? (n / BLOCK) * p.w.lds + kk / BLOCK
                                                : (kk / BLOCK) * p.w.lds + n / BLOCK];
                }
                xs[k][r] = x;
                ws[wk][wr] = w;
            }
            __syncthreads();
            for (int k = 0; k < 32; ++k)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty + 16 * i], ws[k][tx + 16 * j], acc[i][j]);
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (m >= p.M || n >= p.N) continue;
                const long at = m * p.y.ld + n;
                const float v = acc[i][j] + (p.bias ? p.bias[n] : 0.f);
                void* y = const_cast<void*>(p.y.p);
                if (p.y.type == OP_F32) {
                    float* o = static_cast<float*>(y) + at;
                    *o = p.accumulate ? *o + v : v;
                } else if (p.y.type == OP_F16) {
                    f16* o = static_cast<f16*>(y) + at;
                    *o = from_f32<f16>(p.accumulate ? to_f32(*o) + v : v);
                } else {
                    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(y) + at;
                    *o = from_f32<__nv_bfloat16>(p.accumulate ? to_f32(*o) + v : v);
                }
            }
    }
}

}  // namespace

void gemm_f8(const GemmF8& a, cudaStream_t s) {
    const long mt = (a.M + 63) / 64;
    gemm_f8_kernel<<<dim3((unsigned)((a.N + 63) / 64), (unsigned)(mt < 65535 ? mt : 65535)), 256, 0, s>>>(a);
}

}  // namespace act
