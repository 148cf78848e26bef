// layernorm_fwd.cu -- layer norm whose weight and bias learn, forward: row statistics, the result in
// 16 or 32 bits and in 8 bits, and the 8-bit checkpoint of the input, in one pass.
//
// Every element is read once into registers, four columns a lane and up to NCH blocks of 128 columns a
// warp, by W warps a row.
// All statistics and sums are fp32.
// The variance is the mean square of the differences from the mean, taken from the registers that
// hold the row (no cancellation as in E[x^2] - E[x]^2, and no second read).  24000 x 1536 bf16 with an
// I8 checkpoint: 44 us in a captured loop, 4.2 TB/s (65% of HBM's rate), at 2.7 of 4 issues a cycle and 44%
// of the warps: what waits is the chain from a row's sums to its writing.
#include <atomic>

#include "layernorm.cuh"

namespace act {

namespace {

using namespace ln;

struct FwdParams {
    long rows, ldx, ldy;  // strides in bytes
    const char* x;
    char* y;
    int y_wide, y_half, dim;  // y in fp32, or f16 (else bf16)
    const float *w, *b;
    float eps, inv_dim;
    Q8 y8, x8;
    float *mean, *rstd;
};

// G groups of W warps a CTA, NCH blocks of 128 columns a warp.  A group walks over rows and has the
// next row's words under way while it works on this one's.
// KEEP: checkpoint of x, 0 none, 1 I8, 2 E4M3
template <typename T, int W, int NCH, int G, bool VEC, int KEEP>
__global__ void __launch_bounds__(W * G * 32) ln_fwd_kernel(const FwdParams p) {
    __shared__ float slots[2][G][W];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W, wid = warp % W;
    const int first = wid * BLOCK + first_col<VEC>(lane);  // the lane's first column; the next block's is W * 128 on
    const int left = p.dim - first;                        // columns from there
    const bool ragged = p.dim != NCH * W * BLOCK;          // some of the lane's columns are missing
    const long step = (long)gridDim.x * G;
    long row = (long)blockIdx.x * G + grp;
    Raw4<T, VEC> raw[NCH];
    const char* x = p.x + row * p.ldx + first * (int)sizeof(T);
    auto fetch = [&]() {
#pragma unroll
        for (int k = 0; k < NCH; ++k)
            raw[k].load(reinterpret_cast<const T*>(x) + k * W * BLOCK, left - k * W * BLOCK);
        x += step * p.ldx;
    };
    // where this lane's columns of the row go, and (lane k) its warp's k-th block's scale
    const bool mine = lane < NCH && (lane * W + wid) * BLOCK < p.dim;
    char* y = p.y + row * p.ldy + first * (p.y_wide ? 4 : 2);
    uint8_t *x8 = p.x8.q + row * p.x8.ldq + first, *y8 = p.y8.q + row * p.y8.ldq + first;
    float* xs = p.x8.scale + (mine ? (long)(lane * W + wid) * p.x8.lds : 0);
    float* ys = p.y8.scale + (mine ? (long)(lane * W + wid) * p.y8.lds : 0);
    if (row < p.rows) fetch();
    for (; row < p.rows; row += step) {  // whole groups: the barriers are the group's own
        uint64_t v[NCH][2], sum2 = 0;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            float f[4];
            raw[k].values(f);
            pairs(f, v[k]);
            sum2 = add2(sum2, add2(v[k][0], v[k][1]));
        }
        if (row + step < p.rows) fetch();
        const float mean =
            row_sum<W>(unpair(sum2).x + unpair(sum2).y, slots[0][grp], wid, lane, 1 + grp) * p.inv_dim;
        const uint64_t minus = pair(-mean);
        uint64_t sq2 = 0;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            uint64_t d[2] = {add2(v[k][0], minus), add2(v[k][1], minus)};
            if (ragged) {  // missing columns hold 0, not the mean
                float f[4];
                unpairs(d, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = elem<VEC>(i) < left - k * W * BLOCK ? f[i] : 0.f;
                pairs(f, d);
            }
            sq2 = fma2(d[0], d[0], fma2(d[1], d[1], sq2));
        }
        const float sq = row_sum<W>(unpair(sq2).x + unpair(sq2).y, slots[1][grp], wid, lane, 1 + grp);
        const float rstd = rsqrtf(sq * p.inv_dim + p.eps);
        if (wid == 0 && lane == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        if (KEEP) {
            // one test a row: a value that is not finite or beyond the limit makes the sum of squares infinite or
            // NaN, unless it is the mean (one column)
            const bool bad = !(fmaf(mean, mean, sq) < __int_as_float(0x7f800000));
            uint32_t scale = 0;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                float f[4];
                unpairs(v[k], f);
                if (bad) limit4(f, KEEP == 2);
                const uint32_t s =
                    scale_bits(__reduce_max_sync(FULL_WARP, bad ? largest_finite(f) : largest(f)), KEEP == 2);
                store_codes<VEC>(x8 + k * W * BLOCK, left - k * W * BLOCK, encode4(f, inverse_pow2(s), KEEP == 2, bad));
                scale = lane == k ? s : scale;
            }
            if (mine) xs[row] = __uint_as_float(scale);
            x8 += step * p.x8.ldq;
        }
        const uint64_t r2 = pair(rstd);
        uint32_t scale = 0;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int at = k * W * BLOCK, n = left - at;
            uint64_t h[2] = {mul2(add2(v[k][0], minus), r2), mul2(add2(v[k][1], minus), r2)}, w2[2], b2[2];
            float f[4];
            if (p.w) {
                load4_const<VEC>(p.w + first + at, n, f);
                pairs(f, w2);
                h[0] = mul2(h[0], w2[0]);
                h[1] = mul2(h[1], w2[1]);
            }
            if (p.b) {
                load4_const<VEC>(p.b + first + at, n, f);
                pairs(f, b2);
                h[0] = add2(h[0], b2[0]);
                h[1] = add2(h[1], b2[1]);
            }
            unpairs(h, f);
            if (p.y) {
                if (p.y_wide) store4_bytes<4, VEC>(y + at * 4, false, n, f);
                else store4_bytes<2, VEC>(y + at * 2, p.y_half, n, f);
            }
            if (p.y8.q) {
                if (ragged)
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[i] = elem<VEC>(i) < n ? f[i] : 0.f;
                const uint32_t s = store_block<VEC>(y8 + at, n, f, p.y8.e4m3);
                scale = lane == k ? s : scale;
            }
        }
        y += step * p.ldy;
        if (p.y8.q) {
            if (mine) ys[row] = __uint_as_float(scale);
            y8 += step * p.y8.ldq;
        }
    }
}

template <typename T, int W, int NCH, int G, bool VEC, int KEEP>
void launch_fwd(const FwdParams& p, cudaStream_t s) {
    // as many CTAs as run at once, each walking over rows
    static std::atomic<int> known[64];
    int dev = 0, per_sm = 0;
    const bool cached = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    if (cached) per_sm = known[dev].load(std::memory_order_relaxed);
    if (per_sm < 1) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, ln_fwd_kernel<T, W, NCH, G, VEC, KEEP>, W * G * 32, 0) !=
                cudaSuccess || per_sm < 1) {
            cudaGetLastError();
            per_sm = 1;
        } else if (cached) {
            known[dev].store(per_sm, std::memory_order_relaxed);
        }
    }
    const long need = (p.rows + G - 1) / G, most = (long)per_sm * current_sm_count();
    ln_fwd_kernel<T, W, NCH, G, VEC, KEEP><<<(unsigned)(need < most ? need : most), W * G * 32, 0, s>>>(p);
}

template <typename T, int W, int NCH, int G, bool VEC>
void launch_fwd(const FwdParams& p, cudaStream_t s) {
    if (!p.x8.q) launch_fwd<T, W, NCH, G, VEC, 0>(p, s);
    else if (p.x8.e4m3) launch_fwd<T, W, NCH, G, VEC, 2>(p, s);
    else launch_fwd<T, W, NCH, G, VEC, 1>(p, s);
}

template <typename T, int W, int NCH, int G>
void launch_fwd(const FwdParams& p, bool vec, cudaStream_t s) {
    if (vec) launch_fwd<T, W, NCH, G, true>(p, s);
    else launch_fwd<T, W, NCH, G, false>(p, s);
}

// Up to four blocks of 128 columns a warp: at 24000 x 1536 bf16 with an I8 checkpoint one warp a row takes
// 169 us (128 registers, few rows in flight), two 56 us, four 49 us (single launches, cold)
template <typename T>
void fwd_by_dim(const FwdParams& p, bool vec, cudaStream_t s) {
    if (p.dim <= 256) launch_fwd<T, 1, 2, 8>(p, vec, s);
    else if (p.dim <= 512) launch_fwd<T, 1, 4, 8>(p, vec, s);
    else if (p.dim <= 1024) launch_fwd<T, 2, 4, 4>(p, vec, s);
    else if (p.dim <= 1536) launch_fwd<T, 4, 3, 2>(p, vec, s);
    else if (p.dim <= 2048) launch_fwd<T, 4, 4, 2>(p, vec, s);
    else if (p.dim <= 4096) launch_fwd<T, 8, 4, 1>(p, vec, s);
    else launch_fwd<T, 16, 4, 1>(p, vec, s);
}

}  // namespace

void layernorm_train_fwd(const LnFwd& a, cudaStream_t s) {
    FwdParams p;
    p.rows = a.rows; p.ldx = a.x.ld * op_bytes(a.x.type); p.ldy = a.y.ld * op_bytes(a.y.type);
    p.x = static_cast<const char*>(a.x.p); p.y = static_cast<char*>(const_cast<void*>(a.y.p));
    p.y_wide = a.y.type == OP_F32; p.y_half = a.y.type == OP_F16;
    p.dim = a.dim; p.w = a.w; p.b = a.b; p.eps = a.eps; p.inv_dim = 1.0f / (float)a.dim;
    p.y8 = a.y8; p.x8 = a.x8; p.mean = a.mean; p.rstd = a.rstd;
    const bool vec = a.dim % 4 == 0 && vec4(a.x) && vec4(a.y) && vec4(a.y8) && vec4(a.x8) && vec4(a.w) && vec4(a.b);
    if (a.x.type == OP_F16) fwd_by_dim<f16>(p, vec, s);
    else if (a.x.type == OP_BF16) fwd_by_dim<__nv_bfloat16>(p, vec, s);
    else fwd_by_dim<float>(p, vec, s);
}

}  // namespace act
