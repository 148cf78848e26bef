// layernorm.cu -- layer norm whose weight and bias learn: forward with the 8-bit checkpoint of its
// input and the 8-bit form of its result, backward from either form of the input, with the sums
// over the rows that are the weight's and the bias's gradients.
//
// Both passes read every element once and are bound by HBM.  A row is held in registers, four
// columns a lane and NCH blocks of 128 columns a warp, by W warps; variance is the mean square of
// the differences from the mean, taken from those registers (no cancellation as in E[x^2] -
// E[x]^2, and no second read).  All statistics and sums are fp32.
#include "ckpt8.cuh"

namespace act {

namespace {

using namespace c8;

// ---------------------------------------------------------------------------------------
// sums of N values over the W warps of a row; slot: W * N floats of shared memory that nobody
// else uses between two calls (the caller alternates between two)
template <int W, int N>
__device__ __forceinline__ void row_sum(float* v, float* slot, int wid, int lane, int bar) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (W == 1) return;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) slot[wid * N + i] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(W * 32) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += slot[w * N + i];
        v[i] = s;
    }
}

struct FwdParams {
    long rows, ldx, ldy;
    const void* x;
    void* y;
    int y_type, dim;
    const float *w, *b;
    float eps, inv_dim;
    Q8 y8, x8;
    float *mean, *rstd;
};

// G rows per CTA, W warps a row
template <typename T, int W, int NCH, int G, bool VEC>
__global__ void __launch_bounds__(W * G * 32) ln_fwd_kernel(const FwdParams p) {
    __shared__ float slots[2][G][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W, wid = warp % W;
    const long row = (long)blockIdx.x * G + grp;
    if (row >= p.rows) return;  // whole groups: the barriers below are the group's own
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    float v[NCH][4];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c0 = (k * W + wid) * BLOCK;
        load4<T, VEC>(x + c0, p.dim - c0, lane, v[k]);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) sum += (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
    row_sum<W, 1>(&sum, slots[0][grp], wid, lane, 1 + grp);
    const float mean = sum * p.inv_dim;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int n = p.dim - (k * W + wid) * BLOCK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float d = lane_col<VEC>(lane, i) < n ? v[k][i] - mean : 0.f;
            sq = fmaf(d, d, sq);
        }
    }
    row_sum<W, 1>(&sq, slots[1][grp], wid, lane, 1 + grp);
    const float rstd = rsqrtf(sq * p.inv_dim + p.eps);
    if (wid == 0 && lane == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int chunk = k * W + wid, c0 = chunk * BLOCK, n = p.dim - c0;
        if (n <= 0) break;
        if (p.x8.q) {
            const uint32_t s = store_block<VEC>(p.x8.q + row * p.x8.ldq + c0, n, lane, v[k], p.x8.e4m3);
            if (lane == 0) p.x8.scale[(long)chunk * p.x8.lds + row] = __uint_as_float(s);
        }
        float w[4] = {1.f, 1.f, 1.f, 1.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.w) load4<float, VEC>(p.w + c0, n, lane, w);
        if (p.b) load4<float, VEC>(p.b + c0, n, lane, b);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[k][i] = lane_col<VEC>(lane, i) < n ? fmaf((v[k][i] - mean) * rstd, w[i], b[i]) : 0.f;
        if (p.y) store4_as<VEC>(p.y, p.y_type, row * p.ldy + c0, n, lane, v[k]);
        if (p.y8.q) {
            const uint32_t s = store_block<VEC>(p.y8.q + row * p.y8.ldq + c0, n, lane, v[k], p.y8.e4m3);
            if (lane == 0) p.y8.scale[(long)chunk * p.y8.lds + row] = __uint_as_float(s);
        }
    }
}

// ---------------------------------------------------------------------------------------
// Backward.  A CTA's G row groups of W warps walk over rows; each lane keeps the sums dw and db of
// its own columns in registers over all rows of its group, the groups add theirs in order in
// shared memory, and each CTA leaves one row of partial sums that a second kernel adds in CTA
// order.  RPI rows of a group are in flight together and share one exchange of the row sums.
constexpr int BWD_WARPS = 16;
constexpr int BWD_NCH = 4;
constexpr int BWD_RPI = 2;

struct BwdParams {
    long rows, ldy, ldx, lddx;
    const void *dy, *x, *add;
    void* dx;
    int x_type, dx_type, dim;
    Q8 x8;
    const float *w, *mean, *rstd;
    float inv_dim;
    float* part;  // [CTAs][2][dim]
};

template <typename TY, bool X8, int W, bool VEC>
__global__ void __launch_bounds__(BWD_WARPS * 32) ln_bwd_kernel(const BwdParams p) {
    constexpr int G = BWD_WARPS / W, NCH = BWD_NCH, R = BWD_RPI;
    __shared__ float slots[2][G][W * 2 * R];
    extern __shared__ float sums[];  // [2][dim]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W, wid = warp % W;
    float dw[NCH][4] = {}, db[NCH][4] = {};
    int turn = 0;
    const long step = (long)gridDim.x * G * R;
    for (long row = ((long)blockIdx.x * G + grp) * R; row < p.rows; row += step) {
        const int nr = p.rows - row < R ? (int)(p.rows - row) : R;
        float h[R][NCH][4], g[R][NCH][4], red[2 * R];
        float rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long at = row + r;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                const int chunk = k * W + wid, c0 = chunk * BLOCK, n = r < nr ? p.dim - c0 : 0;
                load4<TY, VEC>(static_cast<const TY*>(p.dy) + at * p.ldy + c0, n, lane, g[r][k]);
                if (X8)
                    load_block<VEC>(p.x8.q + at * p.x8.ldq + c0, n, lane,
                                    n > 0 ? p.x8.scale[(long)chunk * p.x8.lds + at] : 0.f, p.x8.e4m3, h[r][k]);
                else load4_as<VEC>(p.x, p.x_type, at * p.ldx + c0, n, lane, h[r][k]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float mean = r < nr ? p.mean[row + r] : 0.f;
            rstd[r] = r < nr ? p.rstd[row + r] : 0.f;
            red[2 * r] = red[2 * r + 1] = 0.f;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                const int c0 = (k * W + wid) * BLOCK, n = r < nr ? p.dim - c0 : 0;
                float w[4] = {1.f, 1.f, 1.f, 1.f};
                if (p.w) load4<float, VEC>(p.w + c0, p.dim - c0, lane, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[r][k][i] = lane_col<VEC>(lane, i) < n ? (h[r][k][i] - mean) * rstd[r] : 0.f;
                    dw[k][i] = fmaf(g[r][k][i], h[r][k][i], dw[k][i]);
                    db[k][i] += g[r][k][i];
                    g[r][k][i] *= w[i];
                    red[2 * r] += g[r][k][i];
                    red[2 * r + 1] = fmaf(g[r][k][i], h[r][k][i], red[2 * r + 1]);
                }
            }
        }
        row_sum<W, 2 * R>(red, slots[turn][grp], wid, lane, 1 + grp);
        turn ^= 1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float c1 = red[2 * r] * p.inv_dim, c2 = red[2 * r + 1] * p.inv_dim;
            const long at = row + r;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                const int c0 = (k * W + wid) * BLOCK, n = r < nr ? p.dim - c0 : 0;
                float a[4] = {0.f, 0.f, 0.f, 0.f};
                if (p.add) load4_as<VEC>(p.add, p.dx_type, at * p.lddx + c0, n, lane, a);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a[i] = fmaf(rstd[r], fmaf(-h[r][k][i], c2, g[r][k][i] - c1), a[i]);
                store4_as<VEC>(p.dx, p.dx_type, at * p.lddx + c0, n, lane, a);
            }
        }
    }
    // the groups' sums, one group after the other
    for (int q = 0; q < G; ++q) {
        if (grp == q)
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                const int c0 = (k * W + wid) * BLOCK, n = p.dim - c0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = lane_col<VEC>(lane, i);
                    if (c < n) {
                        sums[c0 + c] = q == 0 ? dw[k][i] : sums[c0 + c] + dw[k][i];
                        sums[p.dim + c0 + c] = q == 0 ? db[k][i] : sums[p.dim + c0 + c] + db[k][i];
                    }
                }
            }
        __syncthreads();
    }
    float* out = p.part + (long)blockIdx.x * 2 * p.dim;
    for (int c = threadIdx.x; c < 2 * p.dim; c += BWD_WARPS * 32) out[c] = sums[c];
}

// dw / db from nparts rows of partial sums: 32 columns a CTA, 8 lanes of parts each, added in a
// fixed order
__global__ void __launch_bounds__(256) ln_sums_kernel(const float* part, int nparts, int dim, float* dw, float* db,
                                                      int accumulate) {
    __shared__ float s[8][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float a = 0.f;
    if (c < 2 * dim)
        for (int q = slice; q < nparts; q += 8) a += part[(long)q * 2 * dim + c];
    s[slice][lane] = a;
    __syncthreads();
    if (slice || c >= 2 * dim) return;
#pragma unroll
    for (int q = 1; q < 8; ++q) a += s[q][lane];
    float* out = c < dim ? dw : db;
    if (!out) return;
    out += c < dim ? c : c - dim;
    *out = accumulate ? *out + a : a;
}

int bwd_warps(long dim) {
    int w = 1;
    while (w < BWD_WARPS && (long)w * BWD_NCH * BLOCK < dim) w *= 2;
    return w;
}
int bwd_ctas(long rows, long dim) {
    const long per = (long)(BWD_WARPS / bwd_warps(dim)) * BWD_RPI, need = (rows + per - 1) / per;
    const long sms = current_sm_count();
    return (int)(need < sms ? need : sms);
}

template <typename T, int W, int NCH, int G>
void launch_fwd(const FwdParams& p, bool vec, cudaStream_t s) {
    const long ctas = (p.rows + G - 1) / G;
    if (vec) ln_fwd_kernel<T, W, NCH, G, true><<<(unsigned)ctas, W * G * 32, 0, s>>>(p);
    else ln_fwd_kernel<T, W, NCH, G, false><<<(unsigned)ctas, W * G * 32, 0, s>>>(p);
}

template <typename T>
void fwd_by_dim(const FwdParams& p, bool vec, cudaStream_t s) {
    if (p.dim <= 256) launch_fwd<T, 1, 2, 8>(p, vec, s);
    else if (p.dim <= 512) launch_fwd<T, 1, 4, 8>(p, vec, s);
    else if (p.dim <= 1024) launch_fwd<T, 1, 8, 8>(p, vec, s);
    else if (p.dim <= 2048) launch_fwd<T, 4, 4, 2>(p, vec, s);
    else if (p.dim <= 4096) launch_fwd<T, 4, 8, 2>(p, vec, s);
    else launch_fwd<T, 16, 4, 1>(p, vec, s);
}

template <typename TY, bool X8, int W, bool VEC>
void launch_bwd(const BwdParams& p, int ctas, cudaStream_t s) {
    static DeviceOnce once;
    once([] {
        cudaFuncSetAttribute(ln_bwd_kernel<TY, X8, W, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(2 * LN_MAX_DIM * sizeof(float)));
    });
    ln_bwd_kernel<TY, X8, W, VEC><<<ctas, BWD_WARPS * 32, 2 * p.dim * sizeof(float), s>>>(p);
}

template <typename TY, bool X8, int W>
void launch_bwd(const BwdParams& p, bool vec, int ctas, cudaStream_t s) {
    if (vec) launch_bwd<TY, X8, W, true>(p, ctas, s);
    else launch_bwd<TY, X8, W, false>(p, ctas, s);
}

template <typename TY, bool X8>
void bwd_by_dim(const BwdParams& p, bool vec, int ctas, cudaStream_t s) {
    switch (bwd_warps(p.dim)) {
        case 1: return launch_bwd<TY, X8, 1>(p, vec, ctas, s);
        case 2: return launch_bwd<TY, X8, 2>(p, vec, ctas, s);
        case 4: return launch_bwd<TY, X8, 4>(p, vec, ctas, s);
        case 8: return launch_bwd<TY, X8, 8>(p, vec, ctas, s);
        default: return launch_bwd<TY, X8, 16>(p, vec, ctas, s);
    }
}

}  // namespace

void layernorm_train_fwd(const LnFwd& a, cudaStream_t s) {
    FwdParams p;
    p.rows = a.rows; p.ldx = a.x.ld; p.ldy = a.y.ld; p.x = a.x.p; p.y = const_cast<void*>(a.y.p);
    p.y_type = a.y.type; p.dim = a.dim; p.w = a.w; p.b = a.b; p.eps = a.eps; p.inv_dim = 1.0f / (float)a.dim;
    p.y8 = a.y8; p.x8 = a.x8; p.mean = a.mean; p.rstd = a.rstd;
    const bool vec = vec4(a.x) && vec4(a.y) && vec4(a.y8) && vec4(a.x8) && vec4(a.w) && vec4(a.b);
    if (a.x.type == OP_F16) fwd_by_dim<f16>(p, vec, s);
    else if (a.x.type == OP_BF16) fwd_by_dim<__nv_bfloat16>(p, vec, s);
    else fwd_by_dim<float>(p, vec, s);
}

size_t layernorm_train_bwd_space(long rows, long dim) {
    return (size_t)bwd_ctas(rows > 0 ? rows : 1, dim) * 2 * dim * sizeof(float);
}

void layernorm_train_bwd(const LnBwd& a, cudaStream_t s) {
    BwdParams p;
    p.rows = a.rows; p.ldy = a.dy.ld; p.ldx = a.x.ld; p.lddx = a.dx.ld;
    p.dy = a.dy.p; p.x = a.x.p; p.add = a.add.p; p.dx = const_cast<void*>(a.dx.p);
    p.x_type = a.x.type; p.dx_type = a.dx.type; p.dim = a.dim; p.x8 = a.x8;
    p.w = a.w; p.mean = a.mean; p.rstd = a.rstd; p.inv_dim = 1.0f / (float)a.dim; p.part = a.space;
    const bool vec = vec4(a.dy) && vec4(a.x) && vec4(a.add) && vec4(a.dx) && vec4(a.x8) && vec4(a.w);
    const int ctas = a.rows > 0 ? bwd_ctas(a.rows, a.dim) : 0;
    auto go = [&](auto t) {
        typedef decltype(t) T;
        if (a.x8.q) bwd_by_dim<T, true>(p, vec, ctas, s);
        else bwd_by_dim<T, false>(p, vec, ctas, s);
    };
    if (ctas) {
        if (a.dy.type == OP_F16) go(f16{});
        else if (a.dy.type == OP_BF16) go(__nv_bfloat16{});
        else go(float{});
    }
    if (a.dw || a.db)
        ln_sums_kernel<<<(2 * a.dim + 31) / 32, 256, 0, s>>>(a.space, ctas, a.dim, a.dw, a.db, a.accumulate ? 1 : 0);
}

}  // namespace act
